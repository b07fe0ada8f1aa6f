"""Dense KV stores on the GPU: the layers that attend densely, and the prefill's one-layer scratch.

The transformers `Cache` surface of the reference's dense store (`FullGPUCache`, its per-layer
`PreallocatedLayer` and `CacheStats`, lazykv/cache.py:20-115) is kept, because `TieredCache`,
`QuestView` and the snapshot reader take one. The storage is laid out for this library:

* A layer's keys and values share one slab `[2, 1, h, capacity, d]` in HBM (`keys` is slab[0],
  `values` slab[1]): one allocation per layer, made the first time the layer sees KV, so a layer
  that never stores anything here (a tiered layer built by the layer-major prefill) holds no VRAM.
* `update` appends along the token axis and returns views of the filled prefix `[1, h, n, d]`,
  rows `d` elements apart: exactly the dense layout `kernels.dense_source` describes, so the decode
  kernel reads this store in place.
* The slab is zero-filled once. The HIP kernels never read rows past the live length, but a
  consumer that masks unused rows by adding -inf would turn uninitialised NaN into NaN.

Batch size 1, as in the reference. Two stores go beyond it: `MXFP8Cache` holds every layer in 8 bits
(E4M3 codes, a power-of-two scale for every 32 channels of a row), written as tokens arrive and read in
place by the decode, and `SharedPrefixCache` is a batch of sequences over one prefilled cache, each with
rows of its own behind it.
"""

from __future__ import annotations

from bisect import bisect_left
from dataclasses import dataclass

import torch
from transformers.cache_utils import Cache, CacheLayerMixin

from lazykv_amd import kernels


@dataclass
class Decoded:
    """What a selector's `select` returns here (TieredCache, QuestView): the finished attention of
    the step, not a key set. out [1, n_q, 1, d] in the model dtype, lse [1, n_q] float32 (natural log)."""

    out: torch.Tensor
    lse: torch.Tensor


@dataclass(frozen=True)
class CacheStats:
    """Where a cache's KV sits (the reference's `CacheStats`, lazykv/cache.py:105-115): bytes held
    in VRAM, bytes held only in host memory, and the VRAM reserved for KV."""

    seq_len: int
    gpu_resident_kv_bytes: int
    host_kv_bytes: int
    gpu_allocated_kv_bytes: int

    @property
    def gpu_residency_fraction(self) -> float:
        held = self.gpu_resident_kv_bytes + self.host_kv_bytes
        return self.gpu_resident_kv_bytes / held if held else 1.0


class DenseLayer(CacheLayerMixin):
    """One layer's KV in a single preallocated slab (the reference's `PreallocatedLayer`)."""

    def __init__(self, max_len: int, **kwargs: object) -> None:
        super().__init__()
        if max_len <= 0:
            raise ValueError(f"a dense layer needs a positive capacity, got {max_len}")
        self.max_len = max_len
        self.length = 0
        self.slab: torch.Tensor | None = None
        self.cuts = 0  # how often tokens were forgotten
        self._least: list[tuple[int, int]] = []  # (number of the cut, tokens left) of those that no later one went below

    # -- storage ----------------------------------------------------------------------------------

    def lazy_initialization(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        if key_states.shape[0] != 1 or key_states.shape != value_states.shape:
            raise ValueError(f"dense layers hold batch-1 KV with matching key/value shapes, got {tuple(key_states.shape)} / {tuple(value_states.shape)}")
        _, h, _, d = key_states.shape
        self.slab = torch.zeros((2, 1, h, self.max_len, d), dtype=key_states.dtype, device=key_states.device)
        self.keys, self.values = self.slab[0], self.slab[1]
        self.dtype, self.device = key_states.dtype, key_states.device
        self.is_initialized = True

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args: object, **kwargs: object) -> tuple[torch.Tensor, torch.Tensor]:
        self.store(key_states, value_states)
        return self.dense()

    def store(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        """Append the tokens' keys and values [1, h, T, d]."""
        if not self.is_initialized:
            self.lazy_initialization(key_states, value_states)
        a = self.length
        b = a + key_states.shape[-2]
        if b > self.max_len:
            raise RuntimeError(f"dense layer full: appending {b - a} tokens to {a} exceeds its {self.max_len}-token capacity")
        self._write(key_states, value_states, a, b)
        self.length = b

    def _write(self, key_states: torch.Tensor, value_states: torch.Tensor, a: int, b: int) -> None:
        self.keys[:, :, a:b].copy_(key_states)
        self.values[:, :, a:b].copy_(value_states)

    def dense(self) -> tuple[torch.Tensor, torch.Tensor]:
        """The live tokens' keys and values [1, h, n, d] in the model dtype."""
        return self.keys[:, :, : self.length], self.values[:, :, : self.length]

    def rows(self) -> kernels.Rows:
        """The layer's rows as the batch decode reads them."""
        return kernels.dense_rows(self.keys, self.values)

    def _set_length(self, n: int) -> None:
        if n < 0 or n > self.length:
            raise ValueError(f"a dense layer of {self.length} tokens cannot be cut to {n}")
        self.length = n
        while self._least and self._least[-1][1] >= n:
            self._least.pop()
        self._least.append((self.cuts, n))
        self.cuts += 1

    def reset(self) -> None:
        """Forget every token; the slab is kept (only the live prefix is ever read)."""
        self._set_length(0)

    def least_since(self, cuts: int) -> int:
        """The fewest tokens that a cut has left since `cuts` was this many (what there is now, without one): of the rows there were then, those
        below are the same, those from there on may have been filled again."""
        i = bisect_left(self._least, (cuts, -1))
        return self._least[i][1] if i < len(self._least) else self.length

    def truncate(self, length: int) -> None:
        """Forget the tokens past `length`, so one prefill can be decoded from more than once."""
        self._set_length(length)

    # -- transformers plumbing --------------------------------------------------------------------

    def get_mask_sizes(self, query_length: int) -> tuple[int, int]:
        return self.length + query_length, 0

    def get_seq_length(self) -> int:
        return self.length

    def get_max_length(self) -> int:
        return self.max_len

    # -- accounting -------------------------------------------------------------------------------

    def _token_bytes(self) -> int:
        if self.slab is None:
            return 0
        _, _, h, _, d = self.slab.shape
        return 2 * h * d * self.slab.element_size()

    def resident_bytes(self) -> int:
        """VRAM bytes of the live tokens' keys and values."""
        return self._token_bytes() * self.length

    def allocated_bytes(self) -> int:
        return self._token_bytes() * self.max_len


PreallocatedLayer = DenseLayer  # the reference's name for the per-layer store (lazykv/cache.py:20)


class MXFP8Layer(DenseLayer):
    """A dense layer in 8 bits: E4M3 codes under a power-of-two scale for every 32 channels of a row (`kernels.mx_rows`), 33/64 of
    the model dtype's bytes. Tokens are quantised as they are stored, each on its own, so what the layer holds does not depend on
    how they came. Every query attends what the layer holds: a forward of several tokens gets all rows read back in the model
    dtype (exact, but for the code's own rounding), a decode token's attention reads the codes in place (`attention.attend`
    finds them by the `lazykv_rows` that the returned keys carry)."""

    def lazy_initialization(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        if key_states.shape[0] != 1 or key_states.shape != value_states.shape:
            raise ValueError(f"dense layers hold batch-1 KV with matching key/value shapes, got {tuple(key_states.shape)} / {tuple(value_states.shape)}")
        _, h, _, d = key_states.shape
        if d not in (64, 128):
            raise ValueError(f"8-bit layers take head_dim 64 or 128, got {d}")
        self.codes, self.scales = kernels.mx_empty(1, h, self.max_len, d, key_states.device)
        self._rows = kernels.mx_rows(self.codes, self.scales, key_states.dtype)
        self.slab = self.codes
        self.keys, self.values = self.codes[0], self.codes[1]
        self.dtype, self.device = key_states.dtype, key_states.device
        self.is_initialized = True

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args: object, **kwargs: object) -> tuple[torch.Tensor, torch.Tensor]:
        self.store(key_states, value_states)
        if key_states.shape[-2] != 1:
            return self.dense()
        k, v = self.keys[:, :, : self.length], self.values[:, :, : self.length]
        k.lazykv_rows = self._rows
        return k, v

    def _write(self, key_states: torch.Tensor, value_states: torch.Tensor, a: int, b: int) -> None:
        kernels.append_rows(self._rows, key_states, value_states, start=a)

    def dense(self) -> tuple[torch.Tensor, torch.Tensor]:
        return kernels.read_rows(self._rows, 0, self.length)

    def rows(self) -> kernels.Rows:
        return self._rows

    def _token_bytes(self) -> int:
        if self.slab is None:
            return 0
        _, _, h, _, d = self.slab.shape
        return 2 * h * (d + d // kernels.MX_GROUP)


class FullGPUCache(Cache):
    """Every layer's KV held densely in VRAM (the reference's rung 1, lazykv/cache.py:80-102)."""

    layer_type: type[DenseLayer] = DenseLayer

    def __init__(self, num_layers: int, max_len: int) -> None:
        super().__init__(layers=[self.layer_type(max_len) for _ in range(num_layers)])
        self.max_len = max_len

    def truncate(self, length: int) -> None:
        for layer in self.layers:
            layer.truncate(length)

    def stats(self) -> CacheStats:
        dense = [layer for layer in self.layers if isinstance(layer, DenseLayer)]
        return CacheStats(
            seq_len=dense[0].get_seq_length() if dense else 0,
            gpu_resident_kv_bytes=sum(layer.resident_bytes() for layer in dense),
            host_kv_bytes=0,
            gpu_allocated_kv_bytes=sum(layer.allocated_bytes() for layer in dense),
        )

    @classmethod
    def from_kv(cls, layers: list[tuple[torch.Tensor, torch.Tensor]], max_len: int) -> FullGPUCache:
        """A cache holding copies of per-layer prompt KV [1, h, L, d]."""
        cache = cls(len(layers), max_len)
        for dense, (k, v) in zip(cache.layers, layers):
            dense.store(k, v)
        return cache


class MXFP8Cache(FullGPUCache):
    """Every layer's KV held in VRAM in 8 bits (`MXFP8Layer`). It takes a FullGPUCache's place: as a model's cache, under a
    TieredCache (whose dense layers then stay in 8 bits), as a SharedPrefixCache's prefix."""

    layer_type = MXFP8Layer


QUANTS = (None, "mxfp8")


class SharedLayer(CacheLayerMixin):
    """One layer of a SharedPrefixCache: the prefix's layer, read only, and the sequences' own rows behind it."""

    def __init__(self, prefix: DenseLayer, n_seqs: int, max_new: int, quant: str | None) -> None:
        super().__init__()
        self.prefix = prefix
        self.prefix_tokens = prefix.get_seq_length()
        self.prefix_rows = prefix.rows()
        self.prefix_cuts = prefix.cuts
        self.n_seqs, self.max_new, self.quant = n_seqs, max_new, quant
        self.base = 0  # the longest sequence's own tokens when lengths were last set
        self.added = 0  # tokens of every sequence since then
        self.attended = 0  # of these, the ones whose attention was taken: those of whole forwards, once all layers have as many
        self.own: tuple[torch.Tensor, ...] = ()  # keys, values, or codes and scales
        self.own_rows: kernels.Rows | None = None

    def lazy_initialization(self, key_states: torch.Tensor, value_states: torch.Tensor) -> None:
        p = self.prefix_rows
        h, d, dtype = p.n_kv, p.head_dim, p.model_dtype
        if tuple(key_states.shape[:2]) != (self.n_seqs, h) or key_states.shape[3] != d or key_states.dtype != dtype or key_states.device != p.device:
            raise ValueError(f"expected {dtype} KV of {self.n_seqs} sequences [{self.n_seqs}, {h}, T, {d}] on {p.device}, got {key_states.dtype} "
                             f"{tuple(key_states.shape)} on {key_states.device}")
        if self.quant is None:
            self._hold(torch.zeros((2, self.n_seqs, h, self.max_new, d), dtype=dtype, device=p.device))
        else:
            self._hold(*kernels.mx_empty(self.n_seqs, h, self.max_new, d, p.device))
        self.dtype, self.device = dtype, key_states.device
        self.is_initialized = True

    def _hold(self, *own: torch.Tensor) -> None:
        self.own = own
        self.keys, self.values = own[0][0], own[0][1]
        self.own_rows = kernels.dense_rows(self.keys, self.values) if self.quant is None else kernels.mx_rows(*own, self.prefix_rows.model_dtype)

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, *args: object, **kwargs: object) -> tuple[torch.Tensor, torch.Tensor]:
        raise RuntimeError("a shared layer is written through its SharedPrefixCache")

    def own_dense(self, b: int, n: int) -> tuple[torch.Tensor, torch.Tensor]:
        """Sequence b's first n own rows [1, h, n, d] in the model dtype."""
        if self.quant is None:
            return self.keys[b : b + 1, :, :n], self.values[b : b + 1, :, :n]
        codes, scales = self.own
        return kernels.read_rows(kernels.mx_rows(codes[:, b : b + 1], scales[:, b : b + 1], self.prefix_rows.model_dtype), 0, n)

    def keep(self, indices: torch.Tensor) -> None:
        self.n_seqs = indices.numel()
        if self.is_initialized:
            self._hold(*(x.index_select(1, indices) for x in self.own))

    def reset(self) -> None:
        raise RuntimeError("a shared layer is reset through its SharedPrefixCache")

    def reorder_cache(self, beam_idx: torch.Tensor) -> None:
        raise RuntimeError("a shared layer is reordered through its SharedPrefixCache")

    def get_mask_sizes(self, query_length: int) -> tuple[int, int]:
        return self.get_seq_length() + query_length, 0

    def get_seq_length(self) -> int:
        return self.prefix_tokens + self.base + self.added

    def get_max_length(self) -> int:
        return self.prefix_tokens + self.max_new

    def own_bytes(self) -> int:
        """VRAM of the sequences' own rows."""
        return sum(x.numel() * x.element_size() for x in self.own)


class SharedPrefixCache(Cache):
    """A batch of `n_seqs` sequences that continue one prefilled cache, the prefix: samples of one prompt, questions about one
    document. The prefix is held once, however many sequences there are, and is not written to; each sequence has up to `max_new`
    rows of its own behind it, in the model dtype or, with `quant="mxfp8"`, in 8 bits (what the prefix is held in is its own
    matter: a FullGPUCache or an MXFP8Cache). It may grow and be cut back, but once it was cut below the length it had here the
    batch goes no further (RuntimeError), whatever it was filled with again.

    A decode forward (input_ids [n_seqs, 1], `**cache.model_kwargs()`) writes each sequence's token and attends in one call, the
    prefix's keys and values read once for all sequences (`kernels.shared_decode`). A forward of several tokens gives every
    sequence that many; its attention goes sequence by sequence, over the prefix and the sequence's rows, with the causal attention
    of `attention.attend`. Sequences of different lengths: write them padded on the right and `truncate` to the lengths they have;
    later tokens are written and attended behind each one's own end (the model needs position_ids then, [n_seqs, T] from
    `positions`). An attention_mask is not looked at: padding on the left is attended."""

    batched = True  # the attention function takes a batch from this selector
    policy_name = "shared_prefix"

    def __init__(self, prefix: FullGPUCache, n_seqs: int, max_new: int, quant: str | None = None) -> None:
        if quant not in QUANTS:
            raise ValueError(f"unknown precision {quant!r}; expected one of {QUANTS}")
        if n_seqs <= 0 or max_new <= 0:
            raise ValueError(f"a batch needs sequences and room for their tokens, got n_seqs={n_seqs}, max_new={max_new}")
        if not isinstance(prefix, FullGPUCache):
            raise ValueError(f"the prefix must hold every layer densely (FullGPUCache, MXFP8Cache), got {type(prefix).__name__}")
        lengths = {layer.get_seq_length() if layer.is_initialized else 0 for layer in prefix.layers}
        if len(lengths) != 1 or 0 in lengths:
            raise ValueError(f"the prefix must be prefilled, every layer with as many tokens; they hold {sorted(lengths)}")
        super().__init__(layers=[SharedLayer(layer, n_seqs, max_new, quant) for layer in prefix.layers])
        self.full = prefix
        self.n_seqs, self.max_new, self.quant = n_seqs, max_new, quant
        self.prefix_tokens = lengths.pop()
        self._base = [0] * n_seqs  # own lengths as last set; a layer has `added` more
        self._starts: torch.Tensor | None = None  # those on the device, where they differ
        self._scratch: tuple[torch.Tensor, torch.Tensor] | None = None
        self._unattended: int | None = None  # the layer whose new tokens `select` has not seen yet
        self._ended, self._written = 0, 0  # tokens that every layer has since lengths were set, layers that have the current forward's

    # -- lengths ----------------------------------------------------------------------------------

    def _room(self, layer: SharedLayer) -> tuple[int, int]:
        """(what a call adds to `_starts`, tokens of its own that a sequence has at the most) in a layer."""
        most = layer.base + layer.added
        return (most if self._starts is None else layer.added), most

    def lengths(self, layer_idx: int = 0) -> list[int]:
        """Own tokens of each sequence."""
        return [n + self.layers[layer_idx].added for n in self._base]

    def positions(self, n_new: int = 1) -> torch.Tensor:
        """position_ids [n_seqs, n_new] of each sequence's next tokens, made on the device: nothing is waited for."""
        first = self.prefix_tokens + self._room(self.layers[0])[0]
        new = torch.arange(first, first + n_new, device=self.layers[0].prefix_rows.device)
        return new.repeat(self.n_seqs, 1) if self._starts is None else self._starts[:, None] + new

    def truncate(self, lengths: int | list[int]) -> None:
        """Forget each sequence's own tokens past its length (one for all, or one each), between forwards."""
        new = [lengths] * self.n_seqs if isinstance(lengths, int) else [int(n) for n in lengths]
        now = self._whole()
        if len(new) != self.n_seqs or any(n < 0 or n > m for n, m in zip(new, now)):
            raise ValueError(f"sequences of {now} own tokens cannot be cut to {new}")
        self._set(new)

    def keep(self, indices: list[int] | torch.Tensor) -> None:
        """Go on with these sequences, in this order: finished ones left out, one more than once (a beam's branches, each with a
        copy of its rows)."""
        chosen = [int(i) for i in indices]
        if not chosen or any(i < 0 or i >= self.n_seqs for i in chosen):
            raise ValueError(f"sequences {chosen} of {self.n_seqs}")
        now = self._whole()
        at = torch.tensor(chosen, dtype=torch.int64, device=self.layers[0].prefix_rows.device)
        for layer in self.layers:
            layer.keep(at)
        self.n_seqs = len(chosen)
        self._set([now[i] for i in chosen])

    def reorder_cache(self, beam_idx: torch.Tensor) -> None:
        self.keep(beam_idx)

    def batch_select_indices(self, indices: torch.Tensor) -> None:
        self.keep(indices)

    def rollback(self) -> None:
        """Forget the tokens of a forward that raised before its last layer's attention: every sequence has what it had before it. (A forward
        that got further has ended here; `truncate` takes it back.)"""
        whole = min(layer.attended for layer in self.layers)
        self._set([n + whole for n in self._base])

    def reset(self) -> None:
        """Forget every sequence's own tokens; the prefix stays."""
        self._set([0] * self.n_seqs)

    def _whole(self) -> list[int]:
        if len({layer.added for layer in self.layers}) != 1:
            raise RuntimeError("lengths are set between forwards: the layers hold different numbers of tokens; rollback() forgets those of a forward that "
                               "did not end")
        return self.lengths()

    def _set(self, lengths: list[int]) -> None:
        self._base = lengths
        for layer in self.layers:
            layer.base, layer.added, layer.attended = max(lengths), 0, 0
        self._ended, self._written, self._unattended, self._scratch = 0, 0, None, None
        same = len(set(lengths)) == 1
        self._starts = None if same else torch.tensor(lengths, dtype=torch.int32, device=self.layers[0].prefix_rows.device)

    # -- transformers plumbing --------------------------------------------------------------------

    def update(self, key_states: torch.Tensor, value_states: torch.Tensor, layer_idx: int, *args: object, **kwargs: object) -> tuple[torch.Tensor, torch.Tensor]:
        """The tokens' keys and values [n_seqs, h, T, d] behind each sequence's own. What is returned is the new tokens' alone:
        the attention is `select`'s."""
        layer = self.layers[layer_idx]
        if self._unattended is not None:
            raise RuntimeError(f"layer {self._unattended}'s attention did not come from this cache: the forward needs **cache.model_kwargs() and this "
                               "library's attention function (rollback() forgets the token it wrote)")
        if layer.added != self._ended:
            raise RuntimeError(f"layer {layer_idx} holds tokens of a forward that did not end; rollback() forgets them")
        if not layer.is_initialized:
            layer.lazy_initialization(key_states, value_states)
        self._prefix_whole(layer)
        n_new = key_states.shape[-2]
        start, most = self._room(layer)
        if most + n_new > self.max_new:
            raise RuntimeError(f"sequences full: appending {n_new} tokens to {most} exceeds their {self.max_new}-token capacity")
        kernels.append_rows(layer.own_rows, key_states, value_states, start=start, starts=self._starts)
        layer.added += n_new
        self._unattended = layer_idx
        self._written += 1
        if self._written == len(self.layers):
            self._ended, self._written = layer.added, 0
        return key_states, value_states

    def _prefix_whole(self, layer: SharedLayer) -> None:
        if layer.prefix.cuts == layer.prefix_cuts:
            return
        least = layer.prefix.least_since(layer.prefix_cuts)
        if least < self.prefix_tokens:
            raise RuntimeError(f"the prefix was cut to {least} tokens; the batch was made over {self.prefix_tokens}")

    def get_seq_length(self, layer_idx: int = 0) -> int:
        """The longest sequence's tokens, the prefix's among them."""
        return self.prefix_tokens + self._room(self.layers[layer_idx])[1]

    def model_kwargs(self) -> dict[str, object]:
        """The forward's extra keyword: this cache, as the attention function's selector."""
        return {"lazykv_selector": self}

    def select(self, layer_idx: int, query: torch.Tensor, key: torch.Tensor | None = None, value: torch.Tensor | None = None,
               scaling: float | None = None) -> Decoded:
        """The attention of the forward's tokens, whose keys and values `update` has taken: query [n_seqs, n_q, T, d]. The lse is that
        of a decode step; of a forward of several tokens it is empty."""
        layer = self.layers[layer_idx]
        if query.shape[0] != self.n_seqs:
            raise ValueError(f"queries of {query.shape[0]} sequences, the cache holds {self.n_seqs}")
        self._prefix_whole(layer)
        self._unattended = None
        _, n_q, n_new, d = query.shape
        scale = scaling if scaling is not None else d**-0.5
        if n_new > 1:
            got = self._select_many(layer, query, scale)
            layer.attended = layer.added
            if self._written == 0:  # the last layer of this forward
                self._scratch = None
            return got
        start, most = self._room(layer)
        out, lse = kernels.shared_decode(query, scale=scale, prefix=layer.prefix_rows, prefix_tokens=self.prefix_tokens, own=layer.own_rows,
                                         own_tokens=start, lengths=self._starts, max_own=most)
        layer.attended = layer.added
        return Decoded(out.view(self.n_seqs, n_q, 1, d), lse)

    def _select_many(self, layer: SharedLayer, query: torch.Tensor, scale: float) -> Decoded:
        """Several tokens of each sequence: the prefix into one dense buffer in the model dtype, which the layers of a forward share, then each
        sequence's rows behind it in turn. The buffer goes with the forward."""
        from lazykv_amd.attention import attend

        p, r = self.prefix_tokens, layer.prefix_rows
        lengths = [n + layer.added for n in self._base]
        total = p + max(lengths)
        kept = self._scratch[0] if self._scratch is not None else None
        if kept is None or kept.shape[1] != r.n_kv or kept.shape[2] < total or kept.shape[3] != r.head_dim or kept.dtype != r.model_dtype or kept.device != r.device:
            shape = (1, r.n_kv, -(-total // 256) * 256, r.head_dim)
            self._scratch = (torch.empty(shape, dtype=r.model_dtype, device=r.device), torch.empty(shape, dtype=r.model_dtype, device=r.device))
        k, v = self._scratch
        if isinstance(layer.prefix, MXFP8Layer):
            kernels.read_rows(r, 0, p, out=(k[:, :, :p], v[:, :, :p]))
        else:
            k[:, :, :p].copy_(layer.prefix.keys[:, :, :p])
            v[:, :, :p].copy_(layer.prefix.values[:, :, :p])
        outs = []
        for b, n in enumerate(lengths):
            own_k, own_v = layer.own_dense(b, n)
            k[:, :, p : p + n].copy_(own_k)
            v[:, :, p : p + n].copy_(own_v)
            outs.append(attend(query[b : b + 1], k[:, :, : p + n], v[:, :, : p + n], scale))
        return Decoded(torch.cat(outs), torch.empty(0, device=r.device))

    def stats(self) -> CacheStats:
        """The prefix's bytes, once, and the sequences' own; allocated, also a buffer that a forward of several tokens holds until it ends."""
        p = self.full.stats()
        own = sum(layer.own_bytes() for layer in self.layers)
        used = own * sum(self.lengths()) // (self.n_seqs * self.max_new)
        own += sum(x.numel() * x.element_size() for x in self._scratch or ())
        return CacheStats(seq_len=self.get_seq_length(), gpu_resident_kv_bytes=p.gpu_resident_kv_bytes + used, host_kv_bytes=0,
                          gpu_allocated_kv_bytes=p.gpu_allocated_kv_bytes + own)
