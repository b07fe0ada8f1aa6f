"""Query-aware block selection on the GPU: the Quest bound and top-K, fused in one kernel.

Mirrors lazykv/selection.py's module functions (:35-74) with the same names, arguments and
results, computed by the `lkv_bound_topk` HIP kernel instead of two batched GEMMs, an add, an
amax and torch.topk. The selected ids stay on the device.

One deliberate difference: `dtype=None` in the reference computes the bound in the model dtype
through cuBLAS, whose bits depend on the GEMM backend. Here `dtype=None` reproduces that
precision's rounding points (each of the two products and their sum rounded to the model dtype,
accumulation in float32); `dtype=torch.float32` ranks on the float32 bound, which is what the
tier uses (ties at the K-th place are far rarer there).
"""

from __future__ import annotations

import math
import time
from dataclasses import dataclass

import torch
from transformers.cache_utils import Cache

from lazykv_amd import _lib, kernels
from lazykv_amd.cache import CacheStats, Decoded, FullGPUCache, MXFP8Layer

QUEST_DENSE_LAYERS = 2  # lazykv/selection.py:35 -- Quest's first two layers stay dense


def _rank_mode(dtype: torch.dtype | None, model_dtype: torch.dtype) -> int:
    if dtype is None or dtype == model_dtype:
        return _lib.RANK_MODEL
    if dtype == torch.float32:
        return _lib.RANK_F32
    raise ValueError(f"bound dtype {dtype} unsupported: None (model dtype) or torch.float32")


def quest_bound(query: torch.Tensor, kmin: torch.Tensor, kmax: torch.Tensor, dtype: torch.dtype | None = None) -> torch.Tensor:
    """Quest's upper bound [1, kv, n] on each candidate block's score (lazykv/selection.py:38-53).

    `query` is [1, n_q, 1, d]; `kmin`/`kmax` are [1, kv, n, d] over the candidate blocks. Each block
    is scored by the maximum over the head's query group of q+ . kmax + q- . kmin. Returned in
    `dtype` (float32), or in the metadata dtype when `dtype` is None.
    """
    mode = _rank_mode(dtype, kmin.dtype)
    n_kv, n = kmin.shape[1], kmin.shape[2]
    out = torch.empty((n_kv, n), dtype=torch.float32, device=kmin.device)
    kernels.bound_topk(query, kmin, kmax, 0, rank_mode=mode, out_bound=out)
    out = out.unsqueeze(0)
    return out if mode == _lib.RANK_F32 else out.to(kmin.dtype)


def top_blocks(query: torch.Tensor, kmin: torch.Tensor, kmax: torch.Tensor, k: int, dtype: torch.dtype | None = None) -> torch.Tensor:
    """Indices [1, kv, k] of the k candidate blocks with the highest bound (lazykv/selection.py:56-62).

    In descending bound order, like `topk`; equal bounds are ordered by the lower index. Indices
    are candidate-relative (callers add 1 for the sink, lazykv/tiered.py:386,500), int64.
    """
    if k > kmin.shape[2]:
        raise ValueError(f"selected k={k} exceeds the {kmin.shape[2]} candidate blocks")
    idx = kernels.bound_topk(query, kmin, kmax, k, rank_mode=_rank_mode(dtype, kmin.dtype), sorted_=True)
    assert idx is not None
    return idx.to(torch.int64).unsqueeze(0)


def current_block_mask(total: int, block_size: int, fill: int, dtype: torch.dtype, device: torch.device, reuse: torch.Tensor | None = None) -> torch.Tensor:
    """Additive mask [1, 1, 1, total] hiding the unfilled part of the current block (lazykv/selection.py:65-69).

    The decode kernel takes `fill` as a scalar and needs no mask; this is kept for callers that
    build one.
    """
    mask = torch.zeros((1, 1, 1, total), dtype=dtype, device=device) if reuse is None else reuse.zero_()
    mask[..., total - block_size + fill :] = float("-inf")
    return mask


def lazy_extent(length: int, block_size: int) -> tuple[int, int]:
    """(n_full, fill) for `length` tokens under lazy sealing (lazykv/selection.py:153-155,
    lazykv/tiered.py:306-314): block n_full is the current block with `fill` live tokens, 1..block_size.
    A block that has just filled stays current until the next token arrives."""
    n_full, fill = divmod(length, block_size)
    if fill == 0 and n_full > 0:
        n_full, fill = n_full - 1, block_size
    return n_full, fill


def _policy_name(bound_dtype: torch.dtype | None) -> str:
    """"quest" ranks in the model dtype; "quest_float32" (and so on) names the ranking dtype."""
    if bound_dtype is None:
        return "quest"
    return "quest_" + str(bound_dtype).split(".")[-1]


def blocks_for_budget(fraction: float, total_tokens: int, block_size: int) -> int:
    """Selected blocks K such that sink + K blocks + the current block stay within the budget (:72-74)."""
    return max(1, math.floor(fraction * total_tokens / block_size) - 2)


# -- rung 5: selection over a dense cache resident in HBM -----------------------------------------


@dataclass
class SelectorCounters:
    """Host time spent in `select` and the number of selections (lazykv/selection.py:77-80)."""

    host_select_s: float = 0.0
    selections: int = 0


class QuestView(Cache):
    """A decode-time view over a prefilled FullGPUCache that attends only to selected blocks
    (lazykv/selection.py:90-183): the sink, the top-K blocks by Quest bound and the current block.

    Shares the full cache's layers, so decode appends to them. Per selecting layer it keeps key
    min/max metadata [1, kv, cap, d], extended on the device as blocks complete. `select` runs the
    fused bound + top-K and the block-sparse decode over the dense cache in place and returns a
    Decoded (the finished attention of the step) where the reference gathers (k_sel, v_sel, mask)
    for SDPA; nothing is gathered and nothing returns to the host. It returns None (attend densely)
    for the dense layers, for multi-token queries and when the budget covers every block.
    """

    def __init__(self, full: FullGPUCache, k_blocks: int, block_size: int, dense_layers: int = QUEST_DENSE_LAYERS,
                 bound_dtype: torch.dtype | None = None) -> None:
        if any(isinstance(layer, MXFP8Layer) for layer in full.layers[dense_layers:]):
            raise ValueError("the selecting layers' rows are read in the model dtype; an 8-bit cache has none")
        super().__init__(layers=full.layers)
        self.full = full  # decode writes into the full cache's own layers; this view holds no KV
        self.k_blocks = k_blocks
        self.block_size = block_size
        self.dense_layers = dense_layers
        self.bound_dtype = bound_dtype
        self.counters = SelectorCounters()
        self.policy_name = _policy_name(bound_dtype)
        self._meta: dict[int, tuple[torch.Tensor, torch.Tensor]] = {}
        self._n_meta: dict[int, int] = {}
        self._idx: torch.Tensor | None = None
        self._ws: kernels.Workspace | None = None
        for i in range(dense_layers, len(full.layers)):
            if full.layers[i].is_initialized:
                self._refresh_metadata(i, full.layers[i].get_seq_length() // block_size)

    def _dense(self, layer_idx: int):  # noqa: ANN202
        return self.full.layers[layer_idx]

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int, *args: object, **kwargs: object) -> tuple[torch.Tensor, torch.Tensor]:
        """New tokens go to the full cache's layer; the view selects over what it holds."""
        return self._dense(layer_idx).update(key_states, value_states)

    def get_seq_length(self, layer_idx: int = 0) -> int:
        return self._dense(layer_idx).get_seq_length()

    def model_kwargs(self) -> dict[str, object]:
        """The forward's extra keyword: this view, as the attention function's selector."""
        return {"lazykv_selector": self}

    def stats(self) -> CacheStats:
        """The full cache's bytes: under this view every block stays in HBM; only what a step attends shrinks."""
        return self.full.stats()

    def attended_tokens(self) -> int:
        """Tokens a selecting layer attends per step: the sink, K selected blocks and the current block."""
        return self.block_size * (self.k_blocks + 2)

    # -- selection --------------------------------------------------------------------------------

    def _refresh_metadata(self, layer_idx: int, n_full: int) -> None:
        """Key min/max of full blocks [n_meta, n_full) of the layer's cache, written on the device."""
        layer = self.full.layers[layer_idx]
        bs = self.block_size
        h, d = layer.keys.shape[1], layer.keys.shape[3]
        if layer_idx not in self._meta:
            cap = -(-layer.keys.shape[2] // bs)
            kmin = torch.zeros((1, h, cap, d), dtype=layer.keys.dtype, device=layer.keys.device)
            self._meta[layer_idx] = (kmin, torch.zeros_like(kmin))
            self._n_meta[layer_idx] = 0
        n0 = self._n_meta[layer_idx]
        if n_full > n0:
            kmin, kmax = self._meta[layer_idx]
            src = kernels.dense_source(layer.keys, layer.values, bs)
            kernels.store_blocks(src, n_kv=h, head_dim=d, block_size=bs, first_block=n0, n_blocks=n_full - n0, kmin=kmin, kmax=kmax)
            self._n_meta[layer_idx] = n_full

    def select(self, layer_idx: int, query: torch.Tensor, key: torch.Tensor | None = None, value: torch.Tensor | None = None,
               scaling: float | None = None) -> Decoded | None:
        """The attention of this decode step over sink + top-K + current, or None to attend densely."""
        if query.shape[-2] != 1 or layer_idx < self.dense_layers:
            return None  # prefill chunks and Quest's dense layers attend everything
        bs = self.block_size
        layer = self._dense(layer_idx)
        n_full, fill = lazy_extent(layer.get_seq_length(), bs)
        if n_full - 1 <= self.k_blocks:
            # Blocks 1..n_full-1 are the candidates; a selection of K would name all of them, so the
            # dense decode attends the same set in one pass.
            return None
        t0 = time.perf_counter()
        self._refresh_metadata(layer_idx, n_full)
        kmin, kmax = self._meta[layer_idx]
        h, d = layer.keys.shape[1], layer.keys.shape[3]
        dev = layer.keys.device
        if self._idx is None or self._idx.shape[0] != h or self._idx.device != dev:
            self._idx = torch.empty((h, self.k_blocks), dtype=torch.int32, device=dev)
            self._ws = kernels.Workspace(dev)
        mode = _rank_mode(self.bound_dtype, kmin.dtype)
        src = kernels.dense_source(layer.keys, layer.values, bs)
        # The current block may end past the last whole block of the storage; only its rows below
        # `fill` are read.
        src.n_blocks = -(-layer.keys.shape[2] // bs)
        scale = scaling if scaling is not None else d**-0.5
        q = query.reshape(-1, d)
        # Bound, top-K and attention in one call; the selected ids are kept for inspection.
        out, lse = kernels.select_decode(q, kmin, kmax, self.k_blocks, cand_offset=1, n_cand=n_full - 1, block_size=bs, scale=scale,
                                         sel=src, sink=src, sink_block=0, cur=src, cur_block=n_full, fill=fill, rank_mode=mode,
                                         out_idx=self._idx, ws=self._ws)
        self.counters.host_select_s += time.perf_counter() - t0
        self.counters.selections += 1
        n_q = out.shape[0]
        return Decoded(out.view(1, n_q, 1, d), lse.view(1, n_q))
