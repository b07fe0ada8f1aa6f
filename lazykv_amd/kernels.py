"""Tensor-level calls into the HIP kernels: validation, layout descriptors, workspaces.

Every function here enqueues work on the current HIP stream of its tensors' device and returns
without synchronising. Shapes are checked on the host before any launch (the kernels assume
them). The reference-facing modules (`selection`, `quant`, `exact`, `attention`, `tiered`) are
built on these.
"""

from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from lazykv_amd import _lib
from lazykv_amd.pinned import device_address, is_mapped


# -- workspaces -----------------------------------------------------------------------------------


class Workspace:
    """A device scratch buffer (partials, bounds), grown on demand.

    Its contents need no initialisation, so one workspace serves any number of calls issued in
    order on one stream. Growing it allocates a fresh buffer; calls already prepared against the
    old one keep it alive.
    """

    def __init__(self, device: torch.device | str | None = None, nbytes: int = 0) -> None:
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.buf = torch.zeros(max(nbytes, 256), dtype=torch.uint8, device=self.device)

    def get(self, nbytes: int) -> tuple[int, int]:
        if nbytes > self.buf.numel():
            self.buf = torch.zeros(int(nbytes * 1.25) + 256, dtype=torch.uint8, device=self.device)
        return self.buf.data_ptr(), self.buf.numel()


_DEFAULT_WS: dict[tuple[int, int], Workspace] = {}


def default_workspace(device: torch.device) -> Workspace:
    """One workspace per (device, stream), for callers that do not bring their own."""
    dev = torch.device(device)
    idx = dev.index if dev.index is not None else torch.cuda.current_device()
    key = (idx, torch.cuda.current_stream(idx).cuda_stream)
    ws = _DEFAULT_WS.get(key)
    if ws is None:
        ws = _DEFAULT_WS[key] = Workspace(torch.device("cuda", idx))
    return ws


# -- layout descriptors ---------------------------------------------------------------------------


def address(t: torch.Tensor) -> int:
    """Device-visible address of a tensor: its own pointer on the GPU, the mapped alias for a pool."""
    if t.is_cuda:
        return t.data_ptr()
    if is_mapped(t):
        return device_address(t)
    raise RuntimeError("tensor is neither on the GPU nor in mapped pinned memory (there is no CPU path)")


@dataclass
class Source:
    """A `lkv_kv_source`: base addresses and strides of one set of KV blocks, plus its keep-alives."""

    k: int
    v: int
    block_stride: int
    head_stride: int
    dtype: int
    deq_dtype: int
    n_blocks: int
    owners: tuple = ()
    flags: int = 0  # _lib.SRC_HOST for blocks in mapped host memory

    def c(self) -> _lib.KVSource:
        return _lib.KVSource(self.k, self.v, self.block_stride, self.head_stride, self.n_blocks, self.dtype, self.deq_dtype, self.flags)


def _location(t: torch.Tensor) -> int:
    return 0 if t.is_cuda else _lib.SRC_HOST


def pool_source(pool: torch.Tensor) -> Source:
    """Blocks of a `[blocks, h, 2, bs, d]` pool (host pool or GPU slot pool, lazykv/tiered.py:261,265)."""
    if pool.ndim != 5 or pool.shape[2] != 2 or not pool.is_contiguous():
        raise ValueError(f"expected a contiguous [blocks, h, 2, bs, d] pool, got {tuple(pool.shape)}")
    _, h, _, bs, d = pool.shape
    base = address(pool)
    es = pool.element_size()
    code = _lib.dtype_code(pool.dtype)
    return Source(base, base + bs * d * es, h * 2 * bs * d, 2 * bs * d, code, code, pool.shape[0], (pool,), _location(pool))


def record_source(records: torch.Tensor, deq_dtype: torch.dtype) -> Source:
    """Blocks of an int8 record pool `[blocks, h, P]` (lazykv/tiered.py:265, quant.py:46-56)."""
    if records.ndim != 3 or records.dtype != torch.uint8 or not records.is_contiguous():
        raise ValueError(f"expected contiguous uint8 records [blocks, h, P], got {tuple(records.shape)} {records.dtype}")
    _, h, p = records.shape
    base = address(records)
    return Source(base, 0, h * p, p, _lib.INT8_RECORD, _lib.dtype_code(deq_dtype), records.shape[0], (records,), _location(records))


def dense_source(keys: torch.Tensor, values: torch.Tensor, block_size: int) -> Source:
    """Blocks of dense per-head KV `[1, h, T, d]` or `[h, T, d]` (a full cache, lazykv/cache.py:35-36;
    the exact tier's float32 mirror, lazykv/exact.py:131-140). Rows must be contiguous and the token
    stride must be head_dim."""
    # Shapes and strides of the last three dimensions: a view of each tensor's first entry costs microseconds.
    ks, vs = tuple(keys.shape), tuple(values.shape)
    if len(ks) not in (3, 4) or len(vs) not in (3, 4) or ks[-3:] != vs[-3:] or keys.dtype != values.dtype or 0 in (ks[0], vs[0]):
        raise ValueError(f"expected matching [h, T, d] keys/values, got {ks} / {vs}")
    d = ks[-1]
    kst, vst = keys.stride(), values.stride()
    if kst[-1] != 1 or kst[-2] != d or vst[-1] != 1 or vst[-2] != d:
        raise ValueError("dense KV rows must be contiguous with a token stride of head_dim")
    if kst[-3] != vst[-3]:
        raise ValueError("keys and values must share their head stride")
    code = _lib.dtype_code(keys.dtype)
    return Source(address(keys), address(values), block_size * d, kst[-3], code, code, ks[-2] // block_size, (keys, values), _location(keys))


# -- a1 + a2: bound and top-K -----------------------------------------------------------------------


def _meta_layout(kmin: torch.Tensor, kmax: torch.Tensor) -> tuple[int, int, int, int]:
    """(n_kv, n_blocks, head_dim, head_stride) of `[1, h, n, d]` or `[h, n, d]` metadata views."""
    # Shapes and strides of the last three dimensions, as in dense_source.
    a, b = tuple(kmin.shape), tuple(kmax.shape)
    if len(a) not in (3, 4) or len(b) not in (3, 4) or a[-3:] != b[-3:] or kmin.dtype != kmax.dtype or 0 in (a[0], b[0]):
        raise ValueError(f"kmin/kmax must be matching [1, h, n, d] tensors, got {a} / {b}")
    sa, sb = kmin.stride()[-3:], kmax.stride()[-3:]
    if sa != sb or sa[2] != 1 or sa[1] != a[-1]:
        raise ValueError("kmin/kmax rows must be contiguous, with equal strides")
    return a[-3], a[-2], a[-1], sa[0]


def bound_topk(
    q: torch.Tensor,
    kmin: torch.Tensor,
    kmax: torch.Tensor,
    k: int,
    *,
    cand_offset: int = 0,
    n_cand: int | None = None,
    rank_mode: int = _lib.RANK_F32,
    sorted_: bool = False,
    out_idx: torch.Tensor | None = None,
    out_bound: torch.Tensor | None = None,
    ws: Workspace | None = None,
) -> torch.Tensor | None:
    """Quest bound + top-k over block metadata `[1, h, cap, d]`; candidates are blocks
    cand_offset .. cand_offset + n_cand - 1 (default: all of them).

    Returns int32 block ids `[h, k]` (cand_offset included), ascending, or in descending bound
    order when `sorted_`. `out_bound` `[h, n_cand]` float32 receives the bounds when given.
    """
    _lib.require_cuda(q, kmin, kmax)
    n_kv, cap, d, hs = _meta_layout(kmin, kmax)
    if n_cand is None:
        n_cand = cap - cand_offset
    if cand_offset < 0 or n_cand <= 0 or cand_offset + n_cand > cap:
        raise ValueError(f"candidates {cand_offset}..{cand_offset + (n_cand or 0)} outside {cap} metadata blocks")
    qq = q.reshape(-1, q.shape[-1])
    if qq.shape[-1] != d or qq.shape[0] % n_kv:
        raise ValueError(f"query {tuple(q.shape)} does not match metadata with {n_kv} heads of dim {d}")
    qq = qq.contiguous()
    if k > 0 and out_idx is None:
        out_idx = torch.empty((n_kv, k), dtype=torch.int32, device=q.device)
    if out_idx is not None and (out_idx.dtype != torch.int32 or out_idx.shape[-1] < k or out_idx.stride(-1) != 1):
        raise ValueError("out_idx must be int32 [h, >=k] with contiguous rows")
    if out_bound is not None and (out_bound.dtype != torch.float32 or tuple(out_bound.shape) != (n_kv, n_cand) or not out_bound.is_contiguous()):
        raise ValueError(f"out_bound must be contiguous float32 [{n_kv}, {n_cand}]")
    meta_base = address(kmin)
    meta_max = address(kmax)
    ws = ws or default_workspace(q.device)
    ws_ptr, ws_n = ws.get(_lib.lib().lkv_bound_topk_workspace_bytes(n_kv, n_cand, k))
    rc = _lib.lib().lkv_bound_topk(
        _lib.stream_of(q), qq.data_ptr(), _lib.dtype_code(qq.dtype), meta_base, meta_max, _lib.dtype_code(kmin.dtype), hs,
        qq.shape[0], n_kv, d, cand_offset, n_cand, k, rank_mode, _lib.SORTED if sorted_ else 0,
        out_idx.data_ptr() if out_idx is not None else None, out_idx.stride(0) if out_idx is not None else 0,
        out_bound.data_ptr() if out_bound is not None else None, ws_ptr, ws_n,
    )
    _lib.check(rc, "bound_topk")
    return out_idx


# -- a5..a9, a11: sparse decode ---------------------------------------------------------------------


def sparse_decode(
    q: torch.Tensor,
    *,
    n_kv: int,
    block_size: int,
    scale: float,
    sel: Source | None = None,
    idx: torch.Tensor | None = None,
    attend_selected: bool = True,
    sink: Source | None = None,
    sink_block: int = -1,
    cur: Source | None = None,
    cur_block: int = -1,
    fill: int = 0,
    rem: Source | None = None,
    rem_range: tuple[int, int] = (0, 0),
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
    lse: torch.Tensor | None = None,
    ws: Workspace | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Block-sparse GQA decode attention with LSE; see lkv_sparse_decode in include/lazykv_hip.h.

    q `[n_q, d]`; idx int32 `[n_kv, k]` block ids (device). Returns (out `[n_q, d]`, lse `[n_q]` float32).
    """
    _lib.require_cuda(q)
    qq = q.reshape(-1, q.shape[-1]).contiguous()
    n_q, d = qq.shape
    k = 0
    if idx is not None:
        _lib.require_cuda(idx)
        if idx.dtype != torch.int32 or idx.ndim != 2 or idx.shape[0] != n_kv or idx.stride(-1) != 1:
            raise ValueError(f"idx must be int32 [{n_kv}, k] with contiguous rows, got {tuple(idx.shape)} {idx.dtype}")
        k = idx.shape[1]
    out_dtype = out_dtype or (out.dtype if out is not None else qq.dtype)
    if out is None:
        out = torch.empty((n_q, d), dtype=out_dtype, device=q.device)
    if lse is None:
        lse = torch.empty((n_q,), dtype=torch.float32, device=q.device)
    if not out.is_contiguous() or out.numel() != n_q * d or not lse.is_contiguous() or lse.numel() != n_q or lse.dtype != torch.float32:
        raise ValueError("out must be contiguous [n_q, d] and lse contiguous float32 [n_q]")
    desc = _lib.DecodeDesc(n_q, n_kv, d, block_size, float(scale), k, 1 if attend_selected else 0, sink_block, cur_block, fill, rem_range[0], rem_range[1])
    ws = ws or default_workspace(q.device)
    ws_ptr, ws_n = ws.get(_lib.lib().lkv_sparse_decode_workspace_bytes(ctypes.byref(desc)))
    cs = [s.c() if s is not None else None for s in (sel, sink, cur, rem)]
    refs = [ctypes.byref(c) if c is not None else None for c in cs]
    rc = _lib.lib().lkv_sparse_decode(
        _lib.stream_of(qq), ctypes.byref(desc), qq.data_ptr(), _lib.dtype_code(qq.dtype), refs[0],
        idx.data_ptr() if idx is not None else None, idx.stride(0) if idx is not None else 0, refs[1], refs[2], refs[3],
        out.data_ptr(), _lib.dtype_code(out.dtype), lse.data_ptr(), ws_ptr, ws_n,
    )
    _lib.check(rc, "sparse_decode")
    return out, lse


# -- a1 + a2 + a5 + a6: bound, top-K and decode of one layer in one call ----------------------------


def _select_desc(q: torch.Tensor, n_kv: int, block_size: int, scale: float, k: int, sink_block: int, cur_block: int, fill: int) -> _lib.DecodeDesc:
    n_q, d = q.reshape(-1, q.shape[-1]).shape
    return _lib.DecodeDesc(n_q, n_kv, d, block_size, float(scale), k, 1, sink_block, cur_block, fill, 0, 0)


class PreparedSelectDecode:
    """`lkv_select_decode` with its arguments converted once: the Quest bound of candidates
    cand_offset .. cand_offset + n_cand - 1 from metadata `[1, h, cap, d]`, the top k per head, and
    the block-sparse decode over sink + selected (from `sel`) + current. `desc.fill` /
    `desc.cur_block` and `n_cand` (`set_candidates`, up to the count the workspace was sized for) may
    change between calls."""

    def __init__(self, q: torch.Tensor, kmin: torch.Tensor, kmax: torch.Tensor, k: int, *, cand_offset: int, n_cand: int, block_size: int,
                 scale: float, sel: Source, sink: Source | None, sink_block: int, cur: Source | None, cur_block: int, fill: int,
                 out: torch.Tensor, lse: torch.Tensor, rank_mode: int = _lib.RANK_F32, out_idx: torch.Tensor | None = None,
                 ws: Workspace | None = None, max_cand: int | None = None) -> None:
        _lib.require_cuda(q, kmin, kmax, out, lse)
        n_kv, cap, d, hs = _meta_layout(kmin, kmax)
        qq = q.reshape(-1, d)
        if not qq.is_contiguous() or qq.shape[0] % n_kv:
            raise ValueError("query must be contiguous [n_q, d] with n_q a multiple of the KV heads")
        if cand_offset < 0 or n_cand <= 0 or cand_offset + n_cand > cap or not 0 < k <= n_cand:
            raise ValueError(f"candidates {cand_offset}..{cand_offset + n_cand} of {cap} metadata blocks, k={k}")
        if not out.is_contiguous() or out.numel() != qq.numel() or not lse.is_contiguous() or lse.numel() != qq.shape[0] or lse.dtype != torch.float32:
            raise ValueError("out must be contiguous [n_q, d] and lse contiguous float32 [n_q]")
        if out_idx is not None and (out_idx.dtype != torch.int32 or tuple(out_idx.shape) != (n_kv, k) or not out_idx.is_contiguous()):
            raise ValueError(f"out_idx must be contiguous int32 [{n_kv}, {k}]")
        self.desc = _select_desc(qq, n_kv, block_size, scale, k, sink_block, cur_block, fill)
        ws = ws or default_workspace(q.device)
        sizing = max(n_cand, max_cand or 0)
        ws_ptr, ws_n = ws.get(_lib.lib().lkv_select_decode_workspace_bytes(ctypes.byref(self.desc), sizing))
        self._c = [s.c() if s is not None else None for s in (sel, sink, cur)]
        refs = [ctypes.byref(c) if c is not None else None for c in self._c]
        self._keep = (q, kmin, kmax, out, lse, out_idx, ws.buf, sel, sink, cur)
        self._fn = _lib.lib().lkv_select_decode
        self._head = (ctypes.byref(self.desc), qq.data_ptr(), _lib.dtype_code(qq.dtype), address(kmin),
                      address(kmax), _lib.dtype_code(kmin.dtype), hs, cand_offset)
        self._tail = (rank_mode, refs[0], refs[1], refs[2], out.data_ptr(), _lib.dtype_code(out.dtype), lse.data_ptr(),
                      out_idx.data_ptr() if out_idx is not None else None, k, ws_ptr, ws_n)
        self.n_cand = n_cand
        self._sized = sizing
        self._cap = min(cap - cand_offset, sizing)
        self.device = q.device

    def set_candidates(self, n_cand: int) -> None:
        """A new candidate count, up to the one the workspace was sized for (the constructor's
        n_cand, or max_cand). The count decides where the top K is chosen and which kernel instance
        runs, so a HIP graph captured before the change must be captured again after it."""
        if not self.desc.k <= n_cand <= self._cap:
            raise ValueError(f"{n_cand} candidates for k={self.desc.k}: at most {self._cap} (the workspace was sized for {self._sized})")
        self.n_cand = n_cand

    def __call__(self) -> None:
        rc = self._fn(torch.cuda.current_stream(self.device).cuda_stream, *self._head, self.n_cand, *self._tail)
        if rc:
            _lib.check(rc, "select_decode")


def select_decode(q: torch.Tensor, kmin: torch.Tensor, kmax: torch.Tensor, k: int, *, cand_offset: int, n_cand: int, block_size: int, scale: float,
                  sel: Source, sink: Source | None = None, sink_block: int = -1, cur: Source | None = None, cur_block: int = -1, fill: int = 0,
                  rank_mode: int = _lib.RANK_F32, out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None, lse: torch.Tensor | None = None,
                  out_idx: torch.Tensor | None = None, ws: Workspace | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Bound + top-k + block-sparse decode of one layer (lkv_select_decode). Returns (out [n_q, d], lse [n_q])."""
    qq = q.reshape(-1, q.shape[-1]).contiguous()
    n_q, d = qq.shape
    out_dtype = out_dtype or (out.dtype if out is not None else qq.dtype)
    out = out if out is not None else torch.empty((n_q, d), dtype=out_dtype, device=q.device)
    lse = lse if lse is not None else torch.empty((n_q,), dtype=torch.float32, device=q.device)
    PreparedSelectDecode(qq, kmin, kmax, k, cand_offset=cand_offset, n_cand=n_cand, block_size=block_size, scale=scale, sel=sel, sink=sink,
                         sink_block=sink_block, cur=cur, cur_block=cur_block, fill=fill, out=out, lse=lse, rank_mode=rank_mode, out_idx=out_idx, ws=ws)()
    return out, lse


# -- hybrid residency: hits from HBM slots, misses read in place and admitted -------------------------


@dataclass
class Residency:
    """HBM slots of one layer (`slots` [n_slots, h, 2, bs, d]) and the tables that say what they hold:
    block_slot [h, cap] (slot or -1), slot_block [h, n_slots] (block or -1), and `order` [h, n_slots]:
    each head's slots from least to most recently used, ties to the lower slot. All int32 on the GPU.
    With n_slots == k the order decides only which unhit slot a missed block lands in (every unhit
    slot is evicted), and the library accepts None there; `allocate` always keeps it, so the tables
    follow the reference's least-recently-used rule slot for slot."""

    slots: torch.Tensor
    block_slot: torch.Tensor
    slot_block: torch.Tensor
    order: torch.Tensor | None = None

    @classmethod
    def allocate(cls, k: int, h: int, cap_blocks: int, block_size: int, head_dim: int, dtype: torch.dtype, device: torch.device,
                 n_slots: int | None = None) -> Residency:
        n = k if n_slots is None else n_slots
        if n < k:
            raise ValueError(f"{n} slots cannot hold a selection of {k} blocks")
        order = torch.arange(n, dtype=torch.int32, device=device).repeat(h, 1)
        return cls(torch.zeros((n, h, 2, block_size, head_dim), dtype=dtype, device=device),
                   torch.full((h, cap_blocks), -1, dtype=torch.int32, device=device),
                   torch.full((h, n), -1, dtype=torch.int32, device=device), order)

    @property
    def n_slots(self) -> int:
        return self.slots.shape[0]

    def seed(self, first: int, n: int) -> None:
        """Record that slots 0..n-1 of every head hold blocks first..first+n-1 (the caller has written
        them), with the empty slots least recently used: the reference's seeded residency
        (lazykv/tiered.py:274-287). Device-side fills only."""
        dev = self.slot_block.device
        blocks = torch.arange(first, first + n, dtype=torch.int32, device=dev)
        self.slot_block[:, :n] = blocks
        self.block_slot[:, first : first + n] = torch.arange(n, dtype=torch.int32, device=dev)
        if self.order is not None:
            used = torch.cat([torch.arange(n, self.n_slots, device=dev), torch.arange(0, n, device=dev)]).to(torch.int32)
            self.order.copy_(used.expand_as(self.order))

    def tables(self) -> _lib.ResidencyTables:
        order = self.order
        return _lib.ResidencyTables(self.block_slot.data_ptr(), self.block_slot.stride(0), self.slot_block.data_ptr(), self.slot_block.stride(0),
                                    order.data_ptr() if order is not None else None, order.stride(0) if order is not None else 0)

    def check(self, n_kv: int, n_blocks: int, k: int) -> None:
        """Shapes the residency launch relies on: tables with contiguous rows covering the pool's
        blocks and the slots, and n_slots >= k."""
        n = self.n_slots
        for t, want in ((self.block_slot, n_blocks), (self.slot_block, n)) + (((self.order, n),) if self.order is not None else ()):
            if t.dtype != torch.int32 or t.ndim != 2 or t.shape[0] != n_kv or t.shape[1] < want or t.stride(1) != 1:
                raise ValueError(f"residency table must be int32 [{n_kv}, >= {want}] with contiguous rows, got {tuple(t.shape)} {t.dtype}")
        if n < k:
            raise ValueError(f"the slot pool holds {n} slots per head, fewer than k={k}")
        if n > k and self.order is None:
            raise ValueError(f"{n} slots for k={k} need the slots' use order")


def hybrid_decode(
    q: torch.Tensor,
    *,
    n_kv: int,
    block_size: int,
    scale: float,
    host: Source,
    res: Residency,
    idx: torch.Tensor,
    sink: Source | None = None,
    sink_block: int = -1,
    cur: Source | None = None,
    cur_block: int = -1,
    fill: int = 0,
    rem: Source | None = None,
    rem_range: tuple[int, int] = (0, 0),
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
    lse: torch.Tensor | None = None,
    ws: Workspace | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """lkv_hybrid_decode: `sparse_decode` over `host` with the selected pairs in `res`'s slots read
    from HBM, the others read in place and admitted; with `rem`, also every block of `rem_range` the
    selection does not name (the exact tier's remainder). Updates `res`'s tables."""
    p = PreparedHybridDecode(q, n_kv=n_kv, block_size=block_size, scale=scale, host=host, res=res, idx=idx, sink=sink, sink_block=sink_block,
                             cur=cur, cur_block=cur_block, fill=fill, rem=rem, rem_range=rem_range, out=out, out_dtype=out_dtype, lse=lse, ws=ws)
    p()
    return p.out, p.lse


class PreparedHybridDecode:
    """`hybrid_decode` with its arguments converted once; `desc.fill` / `desc.cur_block` may change between calls."""

    def __init__(self, q: torch.Tensor, *, n_kv: int, block_size: int, scale: float, host: Source, res: Residency, idx: torch.Tensor, sink: Source | None,
                 sink_block: int, cur: Source | None, cur_block: int, fill: int, rem: Source | None = None, rem_range: tuple[int, int] = (0, 0),
                 out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None, lse: torch.Tensor | None = None, ws: Workspace | None = None) -> None:
        _lib.require_cuda(q, idx, res.slots, res.block_slot, res.slot_block)
        qq = q.reshape(-1, q.shape[-1]).contiguous()
        n_q, d = qq.shape
        if idx.dtype != torch.int32 or idx.ndim != 2 or idx.shape[0] != n_kv or not idx.is_contiguous():
            raise ValueError(f"idx must be contiguous int32 [{n_kv}, k], got {tuple(idx.shape)} {idx.dtype}")
        k = idx.shape[1]
        res.check(n_kv, host.n_blocks, k)
        out_dtype = out_dtype or (out.dtype if out is not None else qq.dtype)
        self.out = out if out is not None else torch.empty((n_q, d), dtype=out_dtype, device=q.device)
        self.lse = lse if lse is not None else torch.empty((n_q,), dtype=torch.float32, device=q.device)
        r0, r1 = rem_range if rem is not None else (0, 0)
        self.desc = _lib.DecodeDesc(n_q, n_kv, d, block_size, float(scale), k, 1, sink_block, cur_block, fill, r0, r1)
        ws = ws or default_workspace(q.device)
        ws_ptr, ws_n = ws.get(_lib.lib().lkv_hybrid_decode_workspace_bytes(ctypes.byref(self.desc)))
        slot_src = pool_source(res.slots)
        self._c = [s.c() if s is not None else None for s in (host, slot_src, sink, cur, rem)]
        self._tables = res.tables()
        refs = [ctypes.byref(c) if c is not None else None for c in self._c]
        self._keep = (qq, idx, self.out, self.lse, ws.buf, host, res, sink, cur, rem)
        self._fn = _lib.lib().lkv_hybrid_decode
        self._args = (ctypes.byref(self.desc), qq.data_ptr(), _lib.dtype_code(qq.dtype), refs[0], refs[1], idx.data_ptr(), idx.stride(0),
                      ctypes.byref(self._tables), refs[2], refs[3], refs[4], self.out.data_ptr(), _lib.dtype_code(self.out.dtype),
                      self.lse.data_ptr(), ws_ptr, ws_n)
        self.device = q.device

    def __call__(self) -> None:
        rc = self._fn(torch.cuda.current_stream(self.device).cuda_stream, *self._args)
        if rc:
            _lib.check(rc, "hybrid_decode")


class PreparedSelectHybridDecode:
    """`lkv_select_hybrid_decode` with its arguments converted once: the Quest bound of candidates
    cand_offset .. cand_offset + n_cand - 1 from metadata `[1, h, cap, d]`, the top k per head chosen
    by the launch that updates `res`'s tables, and the hybrid decode over sink + selected (hits from
    `res`'s slots, misses from `host`) + current, plus, with `rem`, the exact tier's remainder.
    Equals `PreparedBoundTopk` followed by `PreparedHybridDecode`, bit for bit. `desc.fill` /
    `desc.cur_block` and `n_cand` (`set_candidates`, up to the count the workspace was sized for)
    may change between calls."""

    def __init__(self, q: torch.Tensor, kmin: torch.Tensor, kmax: torch.Tensor, k: int, *, cand_offset: int, n_cand: int, block_size: int,
                 scale: float, host: Source, res: Residency, sink: Source | None, sink_block: int, cur: Source | None, cur_block: int, fill: int,
                 out: torch.Tensor, lse: torch.Tensor, rem: Source | None = None, rem_range: tuple[int, int] = (0, 0), rank_mode: int = _lib.RANK_F32,
                 out_idx: torch.Tensor | None = None, ws: Workspace | None = None, max_cand: int | None = None) -> None:
        _lib.require_cuda(q, kmin, kmax, out, lse, res.slots, res.block_slot, res.slot_block)
        n_kv, cap, d, hs = _meta_layout(kmin, kmax)
        qq = q.reshape(-1, d)
        if not qq.is_contiguous() or qq.shape[0] % n_kv:
            raise ValueError("query must be contiguous [n_q, d] with n_q a multiple of the KV heads")
        if cand_offset < 0 or n_cand <= 0 or cand_offset + n_cand > cap or not 0 < k <= n_cand:
            raise ValueError(f"candidates {cand_offset}..{cand_offset + n_cand} of {cap} metadata blocks, k={k}")
        if not out.is_contiguous() or out.numel() != qq.numel() or not lse.is_contiguous() or lse.numel() != qq.shape[0] or lse.dtype != torch.float32:
            raise ValueError("out must be contiguous [n_q, d] and lse contiguous float32 [n_q]")
        if out_idx is not None and (out_idx.dtype != torch.int32 or tuple(out_idx.shape) != (n_kv, k) or not out_idx.is_contiguous()):
            raise ValueError(f"out_idx must be contiguous int32 [{n_kv}, {k}]")
        res.check(n_kv, host.n_blocks, k)
        self.desc = _select_desc(qq, n_kv, block_size, scale, k, sink_block, cur_block, fill)
        if rem is not None:
            self.desc.rem_first, self.desc.rem_last = rem_range
        ws = ws or default_workspace(q.device)
        sizing = max(n_cand, max_cand or 0)
        ws_ptr, ws_n = ws.get(_lib.lib().lkv_select_hybrid_decode_workspace_bytes(ctypes.byref(self.desc), sizing))
        self._c = [s.c() if s is not None else None for s in (host, pool_source(res.slots), sink, cur, rem)]
        self._tables = res.tables()
        refs = [ctypes.byref(c) if c is not None else None for c in self._c]
        self._keep = (q, kmin, kmax, out, lse, out_idx, ws.buf, host, res, sink, cur, rem)
        self._fn = _lib.lib().lkv_select_hybrid_decode
        self._head = (ctypes.byref(self.desc), qq.data_ptr(), _lib.dtype_code(qq.dtype), address(kmin),
                      address(kmax), _lib.dtype_code(kmin.dtype), hs, cand_offset)
        self._tail = (rank_mode, refs[0], refs[1], ctypes.byref(self._tables), refs[2], refs[3], refs[4], out.data_ptr(), _lib.dtype_code(out.dtype),
                      lse.data_ptr(), out_idx.data_ptr() if out_idx is not None else None, k, ws_ptr, ws_n)
        self.n_cand = n_cand
        self._sized = sizing
        self._cap = min(cap - cand_offset, sizing)
        self.device = q.device

    def set_candidates(self, n_cand: int) -> None:
        """A new candidate count, up to the one the workspace was sized for (the constructor's
        n_cand, or max_cand). A HIP graph captured before the change keeps the old count: capture
        again after it."""
        if not self.desc.k <= n_cand <= self._cap:
            raise ValueError(f"{n_cand} candidates for k={self.desc.k}: at most {self._cap} (the workspace was sized for {self._sized})")
        self.n_cand = n_cand

    def __call__(self) -> None:
        rc = self._fn(torch.cuda.current_stream(self.device).cuda_stream, *self._head, self.n_cand, *self._tail)
        if rc:
            _lib.check(rc, "select_hybrid_decode")


def select_hybrid_decode(q: torch.Tensor, kmin: torch.Tensor, kmax: torch.Tensor, k: int, *, cand_offset: int, n_cand: int, block_size: int,
                         scale: float, host: Source, res: Residency, sink: Source | None = None, sink_block: int = -1, cur: Source | None = None,
                         cur_block: int = -1, fill: int = 0, rem: Source | None = None, rem_range: tuple[int, int] = (0, 0),
                         rank_mode: int = _lib.RANK_F32, out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None,
                         lse: torch.Tensor | None = None, out_idx: torch.Tensor | None = None, ws: Workspace | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Bound + top-k + hybrid decode of one layer (lkv_select_hybrid_decode), with the exact tier's
    remainder when `rem` is given. Returns (out [n_q, d], lse [n_q])."""
    qq = q.reshape(-1, q.shape[-1]).contiguous()
    n_q, d = qq.shape
    out_dtype = out_dtype or (out.dtype if out is not None else qq.dtype)
    out = out if out is not None else torch.empty((n_q, d), dtype=out_dtype, device=q.device)
    lse = lse if lse is not None else torch.empty((n_q,), dtype=torch.float32, device=q.device)
    PreparedSelectHybridDecode(qq, kmin, kmax, k, cand_offset=cand_offset, n_cand=n_cand, block_size=block_size, scale=scale, host=host, res=res,
                               sink=sink, sink_block=sink_block, cur=cur, cur_block=cur_block, fill=fill, out=out, lse=lse, rem=rem, rem_range=rem_range,
                               rank_mode=rank_mode, out_idx=out_idx, ws=ws)()
    return out, lse


# -- a8: merge --------------------------------------------------------------------------------------


def merge_lse(out_a: torch.Tensor, lse_a: torch.Tensor, out_b: torch.Tensor, lse_b: torch.Tensor, out_dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    _lib.require_cuda(out_a, lse_a, out_b, lse_b)
    if out_a.shape != out_b.shape or lse_a.shape != lse_b.shape or out_a.shape[:-1] != lse_a.shape:
        raise ValueError(f"partials must match: {tuple(out_a.shape)}/{tuple(lse_a.shape)} vs {tuple(out_b.shape)}/{tuple(lse_b.shape)}")
    dt = torch.promote_types(out_a.dtype, out_b.dtype)
    a = out_a.to(dt).contiguous()
    b = out_b.to(dt).contiguous()
    la = lse_a.float().contiguous()
    lb = lse_b.float().contiguous()
    d = a.shape[-1]
    rows = a.numel() // d if d else 0
    out = torch.empty(a.shape, dtype=out_dtype or dt, device=a.device)
    lse = torch.empty(la.shape, dtype=torch.float32, device=a.device)
    rc = _lib.lib().lkv_merge_lse(_lib.stream_of(a), a.data_ptr(), la.data_ptr(), b.data_ptr(), lb.data_ptr(), _lib.dtype_code(dt), rows, d, out.data_ptr(), _lib.dtype_code(out.dtype), lse.data_ptr())
    _lib.check(rc, "merge_lse")
    return out, lse


# -- a4, a10, a11: stores ---------------------------------------------------------------------------


def store_blocks(
    src: Source,
    *,
    n_kv: int,
    head_dim: int,
    block_size: int,
    first_block: int,
    n_blocks: int,
    dst: Source | None = None,
    kmin: torch.Tensor | None = None,
    kmax: torch.Tensor | None = None,
    stream: int | None = None,
) -> None:
    """Copy / int8-pack blocks and write their key min/max metadata (lkv_store_blocks).

    kmin/kmax are the full `[1, h, cap, d]` metadata tensors; block b of head h lands at [0, h, b].
    """
    mh, mdt, kmin_p, kmax_p = 0, _lib.F16, None, None
    if kmin is not None:
        _lib.require_cuda(kmin, kmax)
        n, cap, d, mh = _meta_layout(kmin, kmax)
        if n != n_kv or d != head_dim or first_block + n_blocks > cap:
            raise ValueError(f"metadata {tuple(kmin.shape)} cannot hold blocks {first_block}..{first_block + n_blocks} of {n_kv} heads")
        mdt = _lib.dtype_code(kmin.dtype)
        kmin_p, kmax_p = address(kmin), address(kmax)
    if first_block + n_blocks > src.n_blocks or (dst is not None and first_block + n_blocks > dst.n_blocks):
        raise ValueError("block range exceeds the source or destination")
    s = src.c()
    dd = dst.c() if dst is not None else None
    if stream is None:
        stream = torch.cuda.current_stream().cuda_stream
    rc = _lib.lib().lkv_store_blocks(stream, ctypes.byref(s), ctypes.byref(dd) if dd is not None else None, n_kv, head_dim, block_size, first_block, n_blocks, kmin_p, kmax_p, mdt, mh)
    _lib.check(rc, "store_blocks")


def copy_rows(copies: list[tuple[torch.Tensor, torch.Tensor]]) -> None:
    """`dst.copy_(src)` for each (dst, src) of `[h, rows, d]` views, up to 8 of them in one launch (lkv_copy_rows) on
    the current stream. A copy the launch does not cover -- another shape, dtype or device, rows that are not contiguous or
    not of whole 2-byte words, tensors that autograd follows in either mode -- is torch's."""
    first = copies[0][0]
    here = first.is_cuda and first.device.index == torch.cuda.current_device() and 0 < first.shape[0] <= 65535 and _forward_level() < 0
    descs, written = [], []
    for dst, src in copies:
        ds, ss = dst.stride(), src.stride()
        es = dst.element_size()
        if (not here or dst.shape != src.shape or src.dtype != dst.dtype or src.device != first.device or dst.device != first.device
                or ds[-1] != 1 or ss[-1] != 1 or dst.shape[0] != first.shape[0] or src.requires_grad or dst.requires_grad
                or type(src) not in _PLAIN or type(dst) not in _PLAIN
                or (es == 1 and (ds[0] | ds[1] | ss[0] | ss[1] | dst.shape[2] | dst.data_ptr() | src.data_ptr()) & 1)):
            dst.copy_(src)
            continue
        _, rows, d = dst.shape
        descs.append(_lib.RowCopy(src.data_ptr(), dst.data_ptr(), ss[0] * es, ss[1] * es, ds[0] * es, ds[1] * es, rows, d * es))
        written.append(dst)
    if not descs:
        return
    torch.autograd.graph.increment_version(written)  # a graph that saved one of them sees the write, as after copy_
    for i in range(0, len(descs), MAX_ROW_COPIES):
        part = descs[i : i + MAX_ROW_COPIES]
        _lib.check(_lib.lib().lkv_copy_rows(_lib.stream_of(first), (_lib.RowCopy * len(part))(*part), len(part), first.shape[0]), "copy_rows")


MAX_ROW_COPIES = 8  # LKV_MAX_ROW_COPIES
_PLAIN = (torch.Tensor, torch.nn.Parameter)


def _forward_level() -> int:
    """The level of forward-mode differentiation, whose tangents a launch would leave behind; negative outside of any."""
    return getattr(_FORWARD_AD, "_current_level", 0)


_FORWARD_AD = torch.autograd.forward_ad


# -- rows of dense caches: 8 bits as tokens arrive, and a batch over a shared prefix ---------------------


MX_GROUP = 32  # channels of a row that share a scale (LKV_MXFP8)


class Rows:
    """A `lkv_kv_rows`: the keys' and values' rows of `seqs` sequences, one per token, in the model dtype or in 8 bits
    (`dense_rows`, `mx_rows`). It describes the tensors it was made of and keeps them; a program may keep it."""

    __slots__ = ("seqs", "n_kv", "tokens", "head_dim", "dtype", "model_dtype", "model_code", "device_index", "owners", "spans", "struct", "ref")

    def __init__(self, k: int, v: int, k_scale: int | None, v_scale: int | None, strides: tuple, seqs: int, n_kv: int, tokens: int, head_dim: int,
                 dtype: int, model_dtype: torch.dtype, model_code: int, device_index: int, owners: tuple) -> None:
        self.seqs, self.n_kv, self.tokens, self.head_dim = seqs, n_kv, tokens, head_dim
        self.dtype = dtype  # _lib.F16, _lib.BF16 or _lib.MXFP8
        self.model_dtype, self.model_code, self.device_index, self.owners = model_dtype, model_code, device_index, owners
        # The addresses between which keys, values and their scales lie.
        n = (seqs - 1) * strides[0] + (n_kv - 1) * strides[1] + tokens * head_dim
        if k_scale is None:
            self.spans = (k, k + 2 * n), (v, v + 2 * n)
        else:
            self.spans = (k, k + n), (v, v + n), (k_scale, k_scale + n // MX_GROUP), (v_scale, v_scale + n // MX_GROUP)
        self.struct = _lib.KVRows(k, v, k_scale, v_scale, *strides, tokens, seqs, dtype, model_code)
        self.ref = ctypes.byref(self.struct)

    @property
    def device(self) -> torch.device:
        return self.owners[0].device


_ROW_DTYPES = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_CODE_DTYPES = (torch.float8_e4m3fn, torch.uint8)


def _row_dtype(dtype: torch.dtype) -> int:
    code = _ROW_DTYPES.get(dtype)
    if code is None:
        raise ValueError(f"rows are float16 or bfloat16, got {dtype}")
    return code


def dense_rows(keys: torch.Tensor, values: torch.Tensor) -> Rows:
    """Rows in the model dtype: keys and values `[seqs, h, T, d]`, contiguous rows d elements apart, any strides above
    that are multiples of 32 elements and the same for both."""
    _lib.require_cuda(keys, values)
    shape, st, device, dtype = keys.shape, keys.stride(), keys.get_device(), keys.dtype
    if len(shape) != 4 or values.shape != shape or values.dtype != dtype or values.get_device() != device:
        raise ValueError(f"expected matching [seqs, h, T, d] keys/values, got {tuple(shape)} {dtype} / {tuple(values.shape)} {values.dtype}")
    seqs, h, tokens, d = shape
    if st[3] != 1 or st[2] != d or values.stride() != st:
        st, vt = _meant(shape, st), _meant(shape, values.stride())
        if st[3] != 1 or (st[2] != d and tokens != 1) or vt != st:
            raise ValueError("rows must be contiguous with a token stride of head_dim, keys and values with the same strides")
    code = _row_dtype(dtype)
    return Rows(keys.data_ptr(), values.data_ptr(), None, None, st[:2], seqs, h, tokens, d, code, dtype, code, device, (keys, values))


def mx_rows(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype) -> Rows:
    """Rows in 8 bits: codes `[2, seqs, h, T, d]` (keys, values; float8_e4m3fn or uint8) and scales `[2, seqs, h, T, d / 32]`
    (uint8), for a model of `dtype`. Views are fine whose scales are cut like their codes."""
    _lib.require_cuda(codes, scales)
    model = _row_dtype(dtype)
    shape, cs, ss, device = codes.shape, codes.stride(), scales.stride(), codes.get_device()
    if len(shape) != 5 or shape[0] != 2 or codes.dtype not in _CODE_DTYPES or scales.dtype != torch.uint8 or scales.get_device() != device:
        raise ValueError(f"expected codes [2, seqs, h, T, d] and uint8 scales, got {tuple(shape)} {codes.dtype} / {tuple(scales.shape)} {scales.dtype}")
    _, seqs, h, tokens, d = shape
    if d % MX_GROUP or scales.shape != (2, seqs, h, tokens, d // MX_GROUP):
        raise ValueError(f"codes {tuple(shape)} take scales {(2, seqs, h, tokens, d // MX_GROUP)}, got {tuple(scales.shape)}")
    if cs[4] != 1 or cs[3] != d or ss[4] != 1 or ss[3] * MX_GROUP != d or ss[1] * MX_GROUP != cs[1] or ss[2] * MX_GROUP != cs[2]:
        raise ValueError("codes' and scales' rows must be contiguous, and their strides alike")
    k, k_scale = codes.data_ptr(), scales.data_ptr()
    return Rows(k, k + cs[0], k_scale, k_scale + ss[0], cs[1:3], seqs, h, tokens, d, _lib.MXFP8, dtype, model, device, (codes, scales))


def mx_empty(seqs: int, n_kv: int, tokens: int, head_dim: int, device: torch.device | str) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scales of a cache in 8 bits (`mx_rows`), zero-filled: every row stands for zeros."""
    codes = torch.zeros((2, seqs, n_kv, tokens, head_dim), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    return codes, torch.zeros((2, seqs, n_kv, tokens, head_dim // MX_GROUP), dtype=torch.uint8, device=device)


def _launch(index: int, fn, *args: object) -> int:  # noqa: ANN001
    """`fn(stream, *args)` on the device's current stream, with that device as the current one."""
    if index == _CURRENT_DEVICE():
        return fn(_raw_stream(index), *args)
    with torch.cuda.device(index):
        return fn(_raw_stream(index), *args)


_CURRENT_DEVICE = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


# The current stream of a device as an integer, without an object for it where torch offers that.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _meant(shape: tuple, strides: tuple) -> tuple:
    """A tensor's strides with 0 for dimensions of size 1, whose strides mean nothing: a decode token's keys and values, one contiguous and
    one a projection's transposed view, differ in those alone. The last dimension's stays."""
    return (*(s if n != 1 else 0 for n, s in zip(shape[:-1], strides)), strides[-1])


def _placed(x: torch.Tensor) -> tuple[torch.Tensor, tuple]:
    """`x` as the row kernels read it, and its strides: contiguous channels, rows on 16 bytes. A copy where it lies otherwise."""
    st = _meant(x.shape, x.stride())
    if st[3] != 1 or (st[0] | st[1] | st[2]) % 8 or x.data_ptr() % 16:
        x = x.clone(memory_format=torch.contiguous_format)
        st = _meant(x.shape, x.stride())
    return x, st


def _no_gradients(what: str, tensors: tuple) -> None:
    """Refuses tensors that autograd follows, in either mode: the calls over rows have no derivative, and leaving it out would be silent."""
    if _GRAD_ENABLED():
        for x in tensors:
            if x.requires_grad:
                raise RuntimeError(f"{what} has no gradient: call it (and a forward over its caches) under torch.no_grad() or inference_mode(), or detach "
                                   "its inputs")
    if _forward_level() >= 0 and any(_FORWARD_AD.unpack_dual(x).tangent is not None for x in tensors):
        raise RuntimeError(f"{what} has no forward-mode derivative; its inputs carry tangents")


_GRAD_ENABLED = torch.is_grad_enabled
_WRITTEN = getattr(torch._C, "_increment_version", torch.autograd.graph.increment_version)  # a graph that saved one of them sees the write, as after copy_


def _int32(name: str, x: int) -> None:
    """Refuses an integer that a C argument of 32 bits would cut."""
    if not -(1 << 31) <= x < 1 << 31:
        raise ValueError(f"{name} = {x} is out of range")


def _counts(x: torch.Tensor | None, seqs: int, device: int, name: str) -> int | None:
    """The address of a count for each sequence, int32 on the device."""
    if x is None:
        return None
    if x.get_device() != device or x.dtype != torch.int32 or x.shape != (seqs,) or not x.is_contiguous():
        raise ValueError(f"{name} must be contiguous int32 [{seqs}] on cuda:{device}, got {x.dtype} {tuple(x.shape)} on {x.device}")
    return x.data_ptr()


def append_rows(dst: Rows, keys: torch.Tensor, values: torch.Tensor, *, start: int = 0, starts: torch.Tensor | None = None) -> None:
    """New tokens' keys and values `[seqs, h, T, d]` into a cache's rows (lkv_append_rows): token t of sequence b becomes row
    `start + starts[b] + t`. Without `starts` the rows must exist (ValueError); with it, rows outside the cache are dropped. An
    8-bit cache takes them as E4M3 codes with a power-of-two scale for every 32 channels, another one as they are; they may be rows of
    that cache itself."""
    shape, dtype, index = keys.shape, dst.model_dtype, dst.device_index
    if len(shape) != 4 or values.shape != shape or keys.dtype != dtype or values.dtype != dtype:
        raise ValueError(f"expected matching {dtype} keys/values [seqs, h, T, d], got {tuple(shape)} {keys.dtype} / {tuple(values.shape)} {values.dtype}")
    seqs, n_kv, n, d = shape
    if seqs != dst.seqs or n_kv != dst.n_kv or d != dst.head_dim:
        raise ValueError(f"keys/values {tuple(shape)} do not match rows of {dst.seqs} sequences, {dst.n_kv} heads and head_dim {dst.head_dim}")
    if keys.get_device() != index or values.get_device() != index:
        raise ValueError(f"keys/values on {keys.device} / {values.device}, the cache on {dst.device}")
    _int32("start", start)
    _no_gradients("append_rows", (keys, values, *dst.owners))
    at = _counts(starts, seqs, index, "starts")
    if 0 in shape:
        return
    x, y, st = keys, values, keys.stride()
    at_x, at_y = x.data_ptr(), y.data_ptr()
    if values.stride() != st or st[3] != 1 or (st[0] | st[1] | st[2]) % 8 or (at_x | at_y) % 16:
        (x, st), (y, yt) = _placed(x), _placed(y)
        if yt != st:
            x, y = torch.stack([x, y]).unbind(0)
            st = x.stride()
        at_x, at_y = x.data_ptr(), y.data_ptr()
    n_bytes = 2 * ((seqs - 1) * st[0] + (n_kv - 1) * st[1] + (n - 1) * st[2] + d)
    if _meet(((at_x, at_x + n_bytes), (at_y, at_y + n_bytes)), dst.spans):
        x, y = torch.stack([x, y]).unbind(0)  # the cache's own rows, moved: none is written before all are read
        st, at_x, at_y = x.stride(), x.data_ptr(), y.data_ptr()
    _WRITTEN(dst.owners)
    rc = _launch(index, _lib.lib().lkv_append_rows, dst.ref, at_x, at_y, dst.model_code, st[0], st[1], st[2], seqs, n_kv, d, n, at, start)
    if rc:
        _lib.check(rc, "append_rows")


def read_rows(src: Rows, first: int, n: int, out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows first .. first + n - 1 of an 8-bit cache as keys and values `[seqs, h, n, d]` in the model dtype (lkv_read_rows),
    each code times its scale; into `out` where given."""
    if src.dtype != _lib.MXFP8:
        raise ValueError("read_rows takes 8-bit rows; others are read where they are")
    if first < 0 or n < 0 or first + n > src.tokens:
        raise ValueError(f"rows {first}..{first + n} exceed the {src.tokens} there are")
    shape, index = (src.seqs, src.n_kv, n, src.head_dim), src.device_index
    _no_gradients("read_rows", src.owners if out is None else (*src.owners, *out))
    if out is None:
        k = torch.empty(shape, dtype=src.model_dtype, device=src.device)
        v = torch.empty_like(k)
        out, st = (k, v), k.stride()
    else:
        for x in out:
            if x.shape != shape or x.dtype != src.model_dtype or x.get_device() != index:
                raise ValueError(f"out must be {src.model_dtype} {shape} on {src.device}, got {x.dtype} {tuple(x.shape)} on {x.device}")
        k, v = out
        st, vt = _meant(shape, k.stride()), _meant(shape, v.stride())
        if vt != st or st[3] != 1 or (st[0] | st[1] | st[2]) % 8 or (k.data_ptr() | v.data_ptr()) % 16:
            raise ValueError("out's rows must be contiguous and start on 16 bytes, both with the same strides")
        _WRITTEN(out)
    if 0 in shape:
        return out
    rc = _launch(index, _lib.lib().lkv_read_rows, src.ref, src.seqs, src.n_kv, src.head_dim, first, n, k.data_ptr(), v.data_ptr(), src.model_code, *st[:3])
    if rc:
        _lib.check(rc, "read_rows")
    return out


def shared_decode(
    q: torch.Tensor,
    *,
    scale: float,
    prefix: Rows | None = None,
    prefix_tokens: int = 0,
    own: Rows | None = None,
    own_tokens: int = 0,
    lengths: torch.Tensor | None = None,
    max_own: int | None = None,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
    lse: torch.Tensor | None = None,
    ws: Workspace | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """One decode token of each of B sequences, q `[B, n_q, d]` or `[B, n_q, 1, d]` (lkv_shared_decode): sequence b attends rows
    0 .. prefix_tokens-1 of `prefix`, one sequence's rows that are read once for the whole batch, and rows
    0 .. own_tokens + lengths[b] - 1 of its own in `own`, at most `max_own` of them (default: own_tokens without
    `lengths`, else all that `own` holds; a bound near the lengths divides the work better). Either may be left out: B = 1 over
    `own` alone is plain decode over an 8-bit cache. Returns (out [B, n_q, d], lse [B, n_q] float32, natural log); a sequence
    without any rows gets zeros and -inf. No gradient: inputs that autograd follows are refused. Without `ws` the scratch is torch's, so calls on several streams and in several graphs
    do not meet."""
    rows = own if own is not None else prefix
    if rows is None:
        raise ValueError("shared_decode needs a prefix's rows or the sequences' own")
    _lib.require_cuda(q)
    shape, index, dtype = q.shape, rows.device_index, rows.model_dtype
    if len(shape) == 4 and shape[2] == 1:
        shape = (shape[0], shape[1], shape[3])
    if len(shape) != 3 or q.dtype != dtype or shape[2] != rows.head_dim or shape[1] == 0 or shape[1] % rows.n_kv or q.get_device() != index:
        raise ValueError(f"query {tuple(q.shape)} {q.dtype} on {q.device} does not match {dtype} rows of {rows.n_kv} heads and head_dim {rows.head_dim} on "
                         f"{rows.device}")
    b, n_q, d = shape
    if own is None:
        if lengths is not None or own_tokens or max_own:
            raise ValueError("own_tokens, lengths and max_own describe `own`, which is not given")
        max_own = 0
    elif own.seqs != b:
        raise ValueError(f"own rows of {own.seqs} sequences, queries of {b}")
    elif max_own is None:
        max_own = own_tokens if lengths is None else own.tokens
    if prefix is not None and (prefix.seqs != 1 or prefix.n_kv != rows.n_kv or prefix.head_dim != d or prefix.model_dtype != dtype or prefix.device_index != index):
        raise ValueError(f"a prefix of {prefix.seqs} sequences, {prefix.n_kv} heads, head_dim {prefix.head_dim}, {prefix.model_dtype} on {prefix.device} "
                         f"does not match one of {rows.n_kv}, {d}, {dtype} on {rows.device}")
    given = () if out is None and lse is None else tuple(x for x in (out, lse) if x is not None)
    _no_gradients("shared_decode", (q, *rows.owners, *(prefix.owners if prefix is not None else ()), *given))
    at = _counts(lengths, b, index, "lengths")
    if (prefix_tokens | own_tokens | max_own) >> 31:
        for name, n in (("prefix_tokens", prefix_tokens), ("own_tokens", own_tokens), ("max_own", max_own)):
            _int32(name, n)
    if lengths is None and own_tokens > max_own:
        raise ValueError(f"own_tokens={own_tokens} exceed max_own={max_own}")
    if not q.is_contiguous() or q.data_ptr() % 16:
        q = q.clone(memory_format=torch.contiguous_format)
    if out is None:
        out = torch.empty_like(q) if out_dtype is None or out_dtype == dtype else torch.empty_like(q, dtype=out_dtype)
        if out.dim() == 4:
            out = out.view(shape)
    elif not out.is_contiguous() or out.numel() != b * n_q * d or out.get_device() != index or (out_dtype is not None and out.dtype != out_dtype) or out.data_ptr() % 16:
        raise ValueError(f"out must be contiguous [{b}, {n_q}, {d}] on {rows.device}, on 16 bytes")
    if lse is None:
        lse = torch.empty((b, n_q), dtype=torch.float32, device=q.device)
    elif not lse.is_contiguous() or lse.numel() != b * n_q or lse.dtype != torch.float32 or lse.get_device() != index:
        raise ValueError(f"lse must be contiguous float32 [{b}, {n_q}] on {rows.device}")
    if b == 0:
        return out, lse
    if given:
        _WRITTEN(given)
    lib = _lib.lib()
    desc = ctypes.byref(_lib.SharedDesc(b, n_q, rows.n_kv, d, scale, prefix_tokens, own_tokens, max_own))
    need = lib.lkv_shared_decode_workspace_bytes(desc)
    if ws is not None:
        ws_ptr, ws_n = ws.get(need)
    else:
        # Of the call's own: no other call's, on another stream or in a graph, can be in it.
        buf = torch.empty(need, dtype=torch.uint8, device=q.device) if need else lse
        ws_ptr, ws_n = buf.data_ptr(), need
    rc = _launch(index, lib.lkv_shared_decode, desc, q.data_ptr(), rows.model_code, prefix.ref if prefix is not None else None,
                 own.ref if own is not None else None, at, out.data_ptr(), _lib.dtype_code(out.dtype), lse.data_ptr(), ws_ptr, ws_n)
    if rc:
        _lib.check(rc, "shared_decode")
    return out, lse


# -- a layer's forward over a bounded cache in pages -------------------------------------------------------


def _paged(rows: Rows, pages: torch.Tensor | None, seqs: int) -> tuple[object, int]:
    """(the C call's page table or None, rows that a sequence can have): `rows` are `seqs` sequences' own, or a pool of pages that the table
    `pages` [seqs, n] (int32, on the device) names."""
    if pages is None:
        if rows.seqs != seqs:
            raise ValueError(f"rows of {rows.seqs} sequences, tokens of {seqs}")
        return None, rows.tokens
    shape, st = pages.shape, pages.stride()
    if len(shape) != 2 or shape[0] != seqs or pages.dtype != torch.int32 or pages.get_device() != rows.device_index or (st[1] != 1 and shape[1] > 1) or st[0] < 0:
        raise ValueError(f"pages must be int32 [{seqs}, n] with contiguous rows on {rows.device}, got {pages.dtype} {tuple(shape)} on {pages.device}")
    return _lib.Pages(pages.data_ptr(), st[0], shape[1]), rows.tokens * shape[1]


def _among(written: tuple, seqs: int, pages: torch.Tensor | None, *at: int | None) -> bool:
    """Whether a call's page table, or numbers at these addresses, one for each sequence, lie among spans of addresses that it writes."""
    n = 4 * seqs
    for a, b in written:
        for x in at:
            if x is not None and x < b and a < x + n:
                return True
    if pages is not None:
        x = pages.data_ptr()
        end = x + 4 * ((seqs - 1) * pages.stride(0) + pages.shape[1])
        for a, b in written:
            if x < b and a < end:
                return True
    return False


def _copies(*tensors: torch.Tensor | None) -> tuple:
    """Copies of numbers that lie among what a call writes: all are read before any is written."""
    return tuple(None if x is None else x.clone() for x in tensors)


def _reach(x: torch.Tensor) -> tuple[int, int]:
    """The addresses between which a tensor's elements lie."""
    at = x.data_ptr()
    if x.is_contiguous():
        return at, at + x.nbytes
    n = 1
    for m, s in zip(x.shape, x.stride()):
        n += (m - 1) * s
    return at, at + x.element_size() * n


def _meet(some: tuple, others: tuple) -> bool:
    """Whether any of some spans of addresses meets any of the others."""
    for a, b in some:
        for c, d in others:
            if a < d and c < b:
                return True
    return False


def rotate_append(
    dst: Rows,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    eps: float = 1e-6,
    start: int = 0,
    starts: torch.Tensor | None = None,
    counts: torch.Tensor | None = None,
    pages: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """New tokens on their way into a cache (lkv_rotate_append): queries q `[seqs, n_q, T, d]` and keys k `[seqs, h, T, d]` normalised over each head
    (where `q_weight` / `k_weight` `[d]` are given: x / sqrt(mean x^2 + eps) * weight) and their first r channels rotated by `cos` / `sin`
    `[seqs or 1, T, r]` (a model's rotary tables, halves paired: channel i with i + r / 2), in float32 and rounded once. Keys and values become rows
    `start + starts[b] + t` of `dst`, as with `append_rows`, with `pages` `[seqs, n]` those of a pool; tokens from `counts[b]` on go to no row.
    Tokens may be rows of `dst` itself; tables, weights, `starts`, `counts` and `pages` may not lie among the rows that are written. Returns the queries (in `out`, which must not
    be any of the inputs). No gradient."""
    shape, kv, dtype, index = q.shape, k.shape, dst.model_dtype, dst.device_index
    if len(shape) != 4 or len(kv) != 4 or v.shape != kv or kv[0] != shape[0] or kv[2] != shape[2] or kv[3] != shape[3] or q.dtype != dtype or k.dtype != dtype or v.dtype != dtype:
        raise ValueError(f"expected {dtype} queries [seqs, n_q, T, d] and matching keys/values [seqs, h, T, d], got {tuple(shape)} {q.dtype}, {tuple(kv)} {k.dtype}, "
                         f"{tuple(v.shape)} {v.dtype}")
    seqs, n_q, n, d = shape
    h = kv[1]
    if n_q == 0:
        raise ValueError(f"queries without heads: {tuple(shape)}")
    if h != dst.n_kv or d != dst.head_dim:
        raise ValueError(f"keys/values {tuple(kv)} do not match rows of {dst.n_kv} heads and head_dim {dst.head_dim}")
    if q.get_device() != index or k.get_device() != index or v.get_device() != index:
        raise ValueError(f"tokens on {q.device} / {k.device} / {v.device}, the cache on {dst.device}")
    _int32("start", start)
    rotary = table_stride = 0
    table = weight = dst.model_code
    read = (q, k, v)  # what the call reads
    cos_at = sin_at = q_at = k_at = None
    if cos is not None and sin is not None:
        cs = cos.shape
        kind = cos.dtype
        if len(cs) != 3 or (cs[0] != 1 and cs[0] != seqs) or cs[1] != n or sin.shape != cs or sin.dtype != kind or (kind != dtype and kind != torch.float32):
            raise ValueError(f"cos/sin must be {dtype} or float32 [{seqs} or 1, {n}, r], got {cos.dtype} {tuple(cs)} / {sin.dtype} {tuple(sin.shape)}")
        if cos.get_device() != index or sin.get_device() != index:
            raise ValueError(f"cos/sin on {cos.device} / {sin.device}, the cache on {dst.device}")
        rotary = cs[2]
        read = (q, k, v, cos, sin)
        cos_at, sin_at = cos.data_ptr(), sin.data_ptr()
        if (cos_at | sin_at) & 15 or not (cos.is_contiguous() and sin.is_contiguous()):
            cos, sin = _whole(cos), _whole(sin)
            cos_at, sin_at = cos.data_ptr(), sin.data_ptr()
        if cs[0] != 1:
            table_stride = n * rotary
        if kind != dtype:
            table = _lib.F32
    elif cos is not None or sin is not None:
        raise ValueError("cos and sin come together")
    if q_weight is not None or k_weight is not None:
        kind = (k_weight if q_weight is None else q_weight).dtype
        for w in (q_weight, k_weight):
            if w is not None:
                if w.shape != (d,) or w.dtype != kind or (kind != dtype and kind != torch.float32) or w.get_device() != index:
                    raise ValueError(f"weights must be {dtype} or float32, both the same, [{d}] on {dst.device}, got {w.dtype} {tuple(w.shape)} on {w.device}")
                read += (w,)
        if kind != dtype:
            weight = _lib.F32
        if q_weight is not None:
            q_weight = _whole(q_weight)
            q_at = q_weight.data_ptr()
        if k_weight is not None:
            k_weight = _whole(k_weight)
            k_at = k_weight.data_ptr()
    if _GRAD_ENABLED() or _forward_level() >= 0:
        _no_gradients("rotate_append", (*read, *dst.owners) if out is None else (*read, *dst.owners, out))
    at, count = _counts(starts, seqs, index, "starts"), _counts(counts, seqs, index, "counts")
    table_ref, _ = _paged(dst, pages, seqs)
    if out is not None:
        if out.shape != shape or out.dtype != dtype or out.get_device() != index:
            raise ValueError(f"out must be {dtype} {tuple(shape)} on {dst.device}, got {out.dtype} {tuple(out.shape)} on {out.device}")
        ot = _meant(shape, out.stride())
        if ot[3] != 1 or (ot[0] | ot[1] | ot[2]) % 8 or out.data_ptr() % 16:
            raise ValueError("out's rows must be contiguous and start on 16 bytes")
        if _meet((_reach(out),), (*map(_reach, read), *dst.spans)):
            raise ValueError("out must not lie among the inputs or the cache's rows")
        if _among((_reach(out),), seqs, pages, at, count):
            starts, counts, pages = _copies(starts, counts, pages)
            at, count, table_ref = _counts(starts, seqs, index, "starts"), _counts(counts, seqs, index, "counts"), _paged(dst, pages, seqs)[0]
    elif 0 in shape:
        return q.new_empty(shape)
    else:
        out = torch.empty_like(q)
        ot = out.stride()
        if ot[3] != 1 or (ot[0] | ot[1] | ot[2]) & 7:  # laid out as queries that the kernel does not read where they are
            out = q.new_empty(shape)
            ot = out.stride()
    if 0 in shape:
        return out
    qt, kt, vt = q.stride(), k.stride(), v.stride()
    x, y, z = q.data_ptr(), k.data_ptr(), v.data_ptr()
    if (qt[0] | qt[1] | qt[2] | kt[0] | kt[1] | kt[2] | vt[0] | vt[1] | vt[2]) & 7 or (x | y | z) & 15 or qt[3] != 1 or kt[3] != 1 or vt[3] != 1:
        (q, qt), (k, kt), (v, vt) = _placed(q), _placed(k), _placed(v)
        x, y, z = q.data_ptr(), k.data_ptr(), v.data_ptr()
    mine = ((x, x + 2 * ((seqs - 1) * qt[0] + (n_q - 1) * qt[1] + (n - 1) * qt[2] + d)), (y, y + 2 * ((seqs - 1) * kt[0] + (h - 1) * kt[1] + (n - 1) * kt[2] + d)),
            (z, z + 2 * ((seqs - 1) * vt[0] + (h - 1) * vt[1] + (n - 1) * vt[2] + d)))
    if _meet(mine, dst.spans):  # the cache's own rows: none is written before all are read
        q, k, v = (w.clone(memory_format=torch.contiguous_format) for w in (q, k, v))
        qt, kt, vt = q.stride(), k.stride(), v.stride()
        x, y, z = q.data_ptr(), k.data_ptr(), v.data_ptr()
    _WRITTEN((*dst.owners, out))
    desc = _lib.RotateDesc(seqs, n_q, h, d, n, dst.model_code, rotary, table, weight, eps, qt[0], qt[1], qt[2], kt[0], kt[1], kt[2], vt[0], vt[1], vt[2], ot[0], ot[1], ot[2],
                           table_stride)
    rc = _launch(index, _lib.lib().lkv_rotate_append, desc, x, y, z, cos_at, sin_at, q_at, k_at, out.data_ptr(), dst.struct, table_ref, at, start, count)
    if rc:
        _lib.check(rc, "rotate_append")
    return out


def _whole(x: torch.Tensor) -> torch.Tensor:
    """`x` as the kernels read tables: contiguous, on 16 bytes."""
    return x if x.is_contiguous() and x.data_ptr() % 16 == 0 else x.clone(memory_format=torch.contiguous_format)


def _chunk(what: str, q: torch.Tensor, rows: Rows, scale: float, tokens: int, lengths: torch.Tensor | None, counts: torch.Tensor | None, max_tokens: int | None,
           pages: torch.Tensor | None, others: tuple) -> tuple:
    """What the calls over a chunk of new tokens check alike: (descriptor, queries as the kernels read them, addresses of lengths and counts, page table, the
    most rows of a sequence)."""
    shape, index = q.shape, rows.device_index
    if len(shape) != 4 or q.dtype != rows.model_dtype or shape[3] != rows.head_dim or shape[1] == 0 or shape[1] % rows.n_kv or q.get_device() != index:
        raise ValueError(f"query {tuple(shape)} {q.dtype} on {q.device} does not match {rows.model_dtype} rows of {rows.n_kv} heads and head_dim {rows.head_dim} on "
                         f"{rows.device}")
    seqs, n_q, n, d = shape
    if _GRAD_ENABLED() or _forward_level() >= 0:
        _no_gradients(what, (q, *rows.owners, *others))
    table, room = _paged(rows, pages, seqs)
    if max_tokens is None:
        max_tokens = tokens if lengths is None else room
    if (tokens | max_tokens) >> 31:
        _int32("tokens", tokens)
        _int32("max_tokens", max_tokens)
        raise ValueError(f"bad extent: {tokens} rows of at most {max_tokens}")
    if lengths is None and tokens > max_tokens:
        raise ValueError(f"tokens={tokens} exceed max_tokens={max_tokens}")
    at, count = _counts(lengths, seqs, index, "lengths"), _counts(counts, seqs, index, "counts")
    st = q.stride()
    if (st[0] | st[1] | st[2]) & 7 or st[3] != 1 or q.data_ptr() & 15:
        q, st = _placed(q)
    return _lib.ChunkDesc(seqs, n_q, rows.n_kv, d, n, scale, tokens, max_tokens, st[0], st[1], st[2]), q, at, count, table, max_tokens


def _scratch(need: int, ws: Workspace | None, beside: torch.Tensor) -> tuple[int | None, int, object]:
    """A call's scratch: the workspace's, or torch's own allocation on a tensor's device, which no other call on another stream or in a graph can be in."""
    if ws is not None:
        return (*ws.get(need), ws)
    if not need:
        return None, 0, None
    buf = beside.new_empty(need, dtype=torch.uint8)
    return buf.data_ptr(), need, buf


def chunk_attend(
    q: torch.Tensor,
    rows: Rows,
    *,
    scale: float,
    tokens: int = 0,
    lengths: torch.Tensor | None = None,
    counts: torch.Tensor | None = None,
    max_tokens: int | None = None,
    pages: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype | None = None,
    lse: torch.Tensor | None = None,
    ws: Workspace | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """A chunk of new tokens of each sequence over its rows, q `[seqs, n_q, T, d]` (lkv_chunk_attend): sequence b has
    `len = tokens + lengths[b]` rows, at most `max_tokens` (default: `tokens` without `lengths`, else all there is room for; a bound near the lengths
    divides the work better), the last `counts[b]` (default: T) of which are the call's own, written before it. Token t attends rows
    0 .. len - counts[b] + t. `rows` are the sequences' own or, with `pages` `[seqs, n]`, a pool's pages, in the model dtype or in 8 bits; T = 1 is a
    decode step. Returns (out [seqs, n_q, T, d], lse [seqs, n_q, T] float32, natural log); tokens from `counts[b]` on and tokens without any row get zeros
    and -inf. No gradient: inputs that autograd follows are refused. Without `ws` the scratch is torch's, so calls on several streams and in
    several graphs do not meet. Weights are rounded to the model dtype for the product with the values, as the batch decode's are; all else is float32 up to `out`."""
    given = () if out is None and lse is None else tuple(x for x in (out, lse) if x is not None)
    desc, q, at, count, table, _ = _chunk("chunk_attend", q, rows, scale, tokens, lengths, counts, max_tokens, pages, given)
    shape, index = q.shape, rows.device_index
    if out is None:
        out = q.new_empty(shape, dtype=out_dtype)
    elif not out.is_contiguous() or out.shape != shape or out.get_device() != index or (out_dtype is not None and out.dtype != out_dtype) or out.data_ptr() % 16:
        raise ValueError(f"out must be contiguous {tuple(shape)} on {rows.device}, on 16 bytes")
    if lse is None:
        lse = q.new_empty(shape[:3], dtype=torch.float32)
    elif not lse.is_contiguous() or lse.shape != shape[:3] or lse.dtype != torch.float32 or lse.get_device() != index:
        raise ValueError(f"lse must be contiguous float32 {tuple(shape[:3])} on {rows.device}")
    if 0 in shape:
        return out, lse
    if given:
        mine = tuple(map(_reach, given))
        if _meet(mine, (_reach(q), *rows.spans)) or (len(mine) == 2 and _meet(mine[:1], mine[1:])):
            raise ValueError("out and lse must not lie among the inputs or each other")
        if _among(mine, len(q), pages, at, count):
            lengths, counts, pages = _copies(lengths, counts, pages)
            desc, q, at, count, table, _ = _chunk("chunk_attend", q, rows, scale, tokens, lengths, counts, max_tokens, pages, given)
        _WRITTEN(given)
    lib = _lib.lib()
    ref = ctypes.byref(desc)
    ws_ptr, ws_n, _held = _scratch(lib.lkv_chunk_attend_workspace_bytes(ref), ws, q)
    rc = _launch(index, lib.lkv_chunk_attend, ref, q.data_ptr(), rows.model_code, rows.ref, table, at, count, out.data_ptr(), _lib.dtype_code(out.dtype),
                 lse.data_ptr(), ws_ptr, ws_n)
    if rc:
        _lib.check(rc, "chunk_attend")
    return out, lse


def _account(name: str, x: torch.Tensor, dtype: torch.dtype, seqs: int, n_kv: int, n: int, device: int) -> tuple[object, tuple[int, int]]:
    """(strides, the addresses between which it lies) of a number for each row, `[seqs, h, n or more]`, of which no two share an address."""
    shape, st = x.shape, x.stride()
    if len(shape) != 3 or shape[0] != seqs or shape[1] != n_kv or shape[2] < n or x.dtype != dtype or x.get_device() != device or (st[2] != 1 and shape[2] > 1):
        raise ValueError(f"{name} must be {dtype} [{seqs}, {n_kv}, {n} or more] with contiguous rows on cuda:{device}, got {x.dtype} {tuple(shape)} on {x.device}")
    if x.is_contiguous():
        at = x.data_ptr()
        return _lib.Pair(st[0], st[1]), (at, at + x.nbytes)
    a, b, n = (st[0] if seqs > 1 else 0), (st[1] if n_kv > 1 else 0), shape[2]
    if (a and b and min(a, b) < n) or (n_kv > 1 and b < n) or (seqs > 1 and a < n) or (a > b > 0 and a < b * (n_kv - 1) + n) or (0 < a <= b and b < a * (seqs - 1) + n):
        raise ValueError(f"{name}'s rows share addresses")
    return _lib.Pair(a, b), _reach(x)


def _same_or_apart(what: str, out: torch.Tensor, x: torch.Tensor, at: tuple[int, int], x_at: tuple[int, int]) -> None:
    """Refuses an output that overlaps its input without being it. at, x_at: where they lie."""
    if at[0] < x_at[1] and x_at[0] < at[1] and (at[0] != x_at[0] or _meant(out.shape, out.stride()) != _meant(x.shape, x.stride())):
        raise ValueError(f"{what} overlap without being the same")


def weigh_rows(
    q: torch.Tensor,
    lse: torch.Tensor,
    rows: Rows,
    *,
    scale: float,
    tokens: int = 0,
    lengths: torch.Tensor | None = None,
    counts: torch.Tensor | None = None,
    max_tokens: int | None = None,
    pages: torch.Tensor | None = None,
    sums: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    seen: torch.Tensor | None = None,
    ws: Workspace | None = None,
) -> torch.Tensor:
    """The weights that rows get from a chunk's tokens, summed up (lkv_weigh_rows): with q, rows and extents as `chunk_attend` took them and the `lse` that it
    gave, each row of a KV head gets the sum of its softmax weights over the head's query heads and the tokens that attend it. That is added to
    `sums` (float32 `[seqs, h, max_tokens or more]`) for rows from before the chunk and is the sum itself for the chunk's own, in `out` (default: `sums`, or without it
    a new tensor of zeros); rows from a sequence's end on are left as they are. `positions` (int32, the same layout) of the chunk's rows become
    `seen[b] + 0, 1, ..` (`seen` int32 `[seqs]`: tokens that the sequence has had before the chunk; default: the rows it has before it). Both are
    what `evict_rows` goes by. No gradient."""
    given = tuple(x for x in (lse, sums, out, positions) if x is not None)
    desc, q, at, count, table, most = _chunk("weigh_rows", q, rows, scale, tokens, lengths, counts, max_tokens, pages, given)
    seqs, n_q, n, d = q.shape
    index = rows.device_index
    if not lse.is_contiguous() or lse.shape != q.shape[:3] or lse.dtype != torch.float32 or lse.get_device() != index:
        raise ValueError(f"lse must be contiguous float32 {tuple(q.shape[:3])} on {rows.device}")
    if out is None:
        out = sums if sums is not None else torch.zeros((seqs, rows.n_kv, most), dtype=torch.float32, device=q.device)
    h, of = rows.n_kv, torch.float32
    out_st, out_at = _account("sums" if out is sums else "out", out, of, seqs, h, most, index)
    if sums is None or sums is out:
        sums_st, sums_at = (None if sums is None else out_st), out_at
    else:
        sums_st, sums_at = _account("sums", sums, of, seqs, h, most, index)
        _same_or_apart("sums and out", out, sums, out_at, sums_at)
    if positions is None:
        if seen is not None:
            raise ValueError("seen says where positions start; there are none")
        positions_st, written, mine, first = None, (out,), (out_at,), None
    else:
        positions_st, positions_at = _account("positions", positions, torch.int32, seqs, h, most, index)
        written, mine, first = (out, positions), (out_at, positions_at), _counts(seen, seqs, index, "seen")
    st, x, y = q.stride(), q.data_ptr(), lse.data_ptr()
    inputs = ((x, x + 2 * ((seqs - 1) * st[0] + (n_q - 1) * st[1] + (n - 1) * st[2] + d)), (y, y + 4 * seqs * n_q * n), *rows.spans)
    if _meet(mine, inputs) or (positions is not None and _meet(mine[1:], (out_at, sums_at))):
        raise ValueError("out and positions must not lie among the inputs or each other")
    if seqs == 0 or most == 0:
        return out
    if _among(mine, seqs, pages, at, count, first):
        lengths, counts, pages, seen = _copies(lengths, counts, pages, seen)
        desc, q, at, count, table, _ = _chunk("weigh_rows", q, rows, scale, tokens, lengths, counts, max_tokens, pages, given)
        first = _counts(seen, seqs, index, "seen")
    _WRITTEN(written)
    lib = _lib.lib()
    ref = ctypes.byref(desc)
    ws_ptr, ws_n, _held = _scratch(lib.lkv_weigh_rows_workspace_bytes(ref), ws, q)
    rc = _launch(index, lib.lkv_weigh_rows, ref, x or y or out_at[0], rows.model_code, y or out_at[0], rows.ref, table, at, count,
                 None if sums is None else sums_at[0], sums_st, out_at[0], out_st, None if positions is None else positions_at[0], positions_st, first, ws_ptr, ws_n)
    if rc:
        _lib.check(rc, "weigh_rows")
    return out


def evict_rows(
    rows: Rows,
    sums: torch.Tensor,
    positions: torch.Tensor,
    *,
    keep: int,
    sinks: int = 0,
    recent: int = 0,
    tokens: int = 0,
    lengths: torch.Tensor | None = None,
    max_tokens: int | None = None,
    pages: torch.Tensor | None = None,
    out: tuple[torch.Tensor, torch.Tensor] | None = None,
    ws: Workspace | None = None,
) -> None:
    """A cache cut to `keep` rows of each sequence and KV head (lkv_evict_rows), of `len = tokens + lengths[b]` that it has: those of the tokens below position
    `sinks`, those of the `recent` newest positions, and of the rest those with the largest `sums`, ties to the lowest row, NaN after all others. Kept rows behind row
    `keep - 1` move into the places before it that are not kept, in their order, with their sums and `positions` (as `weigh_rows` leaves them): attention does not go by the
    order of rows. `out`: (sums, positions) go there instead of back. Afterwards `min(len, keep)` rows are the sequence's; what lies behind them is left as it is.
    Pages that a call may write to must be in one place of one sequence's table. No gradient."""
    _lib.require_cuda(sums, positions)
    seqs, index = sums.shape[0], rows.device_index
    table, room = _paged(rows, pages, seqs)
    if max_tokens is None:
        max_tokens = tokens if lengths is None else room
    if (tokens | max_tokens | keep | sinks | recent) >> 31:
        for name, n in (("tokens", tokens), ("max_tokens", max_tokens), ("keep", keep), ("sinks", sinks), ("recent", recent)):
            _int32(name, n)
    if lengths is None and tokens > max_tokens:
        raise ValueError(f"tokens={tokens} exceed max_tokens={max_tokens}")
    at = _counts(lengths, seqs, index, "lengths")
    h, least = rows.n_kv, max(0, max_tokens)
    sums_st, sums_at = _account("sums", sums, torch.float32, seqs, h, least, index)
    positions_st, positions_at = _account("positions", positions, torch.int32, seqs, h, least, index)
    if out is None:
        to_sums, to_positions, to_sums_st, to_positions_st, to_sums_at, to_positions_at = sums, positions, sums_st, positions_st, sums_at, positions_at
    else:
        to_sums, to_positions = out
        left = min(least, max(0, keep))
        to_sums_st, to_sums_at = _account("out's sums", to_sums, torch.float32, seqs, h, left, index)
        to_positions_st, to_positions_at = _account("out's positions", to_positions, torch.int32, seqs, h, left, index)
        _same_or_apart("sums", to_sums, sums, to_sums_at, sums_at)
        _same_or_apart("positions", to_positions, positions, to_positions_at, positions_at)
    if _GRAD_ENABLED() or _forward_level() >= 0:
        _no_gradients("evict_rows", (*rows.owners, sums, positions, to_sums, to_positions))
    if out is None:
        accounts, others = (sums_at,), (positions_at,)
    else:
        accounts, others = (sums_at, to_sums_at), (positions_at, to_positions_at)
    if _meet(accounts, others) or _meet((*accounts, *others), rows.spans):
        raise ValueError("sums, positions and rows share addresses")
    if seqs == 0 or max_tokens == 0:
        return
    if _among((to_sums_at, to_positions_at, *rows.spans), seqs, pages, at):
        lengths, pages = _copies(lengths, pages)
        at, table = _counts(lengths, seqs, index, "lengths"), _paged(rows, pages, seqs)[0]
    lib = _lib.lib()
    desc = _lib.EvictDesc(seqs, rows.n_kv, rows.head_dim, rows.model_code, keep, sinks, recent, tokens, max_tokens)
    ref = ctypes.byref(desc)
    ws_ptr, ws_n, _held = _scratch(max(16, lib.lkv_evict_rows_workspace_bytes(ref)), ws, sums)
    _WRITTEN((*rows.owners, to_sums, to_positions))
    rc = _launch(index, lib.lkv_evict_rows, ref, rows.ref, table, at, sums_at[0], sums_st, positions_at[0], positions_st, to_sums_at[0], to_sums_st, to_positions_at[0],
                 to_positions_st, ws_ptr, ws_n)
    if rc:
        _lib.check(rc, "evict_rows")


def packed_pair_bytes(block_size: int, head_dim: int) -> int:
    return int(_lib.lib().lkv_packed_pair_bytes(block_size, head_dim))


def pack_int8(pairs: torch.Tensor) -> torch.Tensor:
    """`[m, 2, bs, d]` model dtype -> `[m, P]` uint8 records (lkv_pack_int8)."""
    _lib.require_cuda(pairs)
    m, two, bs, d = pairs.shape
    x = pairs.contiguous()
    out = torch.empty((m, packed_pair_bytes(bs, d)), dtype=torch.uint8, device=pairs.device)
    _lib.check(_lib.lib().lkv_pack_int8(_lib.stream_of(x), x.data_ptr(), _lib.dtype_code(x.dtype), m, bs, d, out.data_ptr()), "pack_int8")
    return out


def unpack_int8(records: torch.Tensor, block_size: int, head_dim: int, dtype: torch.dtype) -> torch.Tensor:
    """`[m, P]` uint8 records -> `[m, 2, bs, d]` (lkv_unpack_int8)."""
    _lib.require_cuda(records)
    r = records.contiguous()
    out = torch.empty((r.shape[0], 2, block_size, head_dim), dtype=dtype, device=records.device)
    _lib.check(_lib.lib().lkv_unpack_int8(_lib.stream_of(r), r.data_ptr(), r.shape[0], block_size, head_dim, _lib.dtype_code(dtype), out.data_ptr()), "unpack_int8")
    return out


def stream_read(src_addr: int, nbytes: int, blocks: int, sink: torch.Tensor) -> None:
    """Launch the link probe over `nbytes` at a device-visible address; sink is uint32 [>= blocks] on the GPU."""
    _lib.check(_lib.lib().lkv_stream_read(_lib.stream_of(sink), src_addr, nbytes, blocks, sink.data_ptr()), "stream_read")


# -- prepared launches ------------------------------------------------------------------------------


class PreparedBoundTopk:
    """`bound_topk` with every argument converted once; calling it only launches.

    For loops that issue the same selection per step (a decode step over many layers), or for
    capture into a HIP graph: the stream is read at call time.
    """

    def __init__(self, q: torch.Tensor, kmin: torch.Tensor, kmax: torch.Tensor, k: int, *, cand_offset: int, n_cand: int, out_idx: torch.Tensor | None = None,
                 rank_mode: int = _lib.RANK_F32, ws: Workspace | None = None, out_bound: torch.Tensor | None = None) -> None:
        """k == 0 with `out_bound` [h, n_cand] float32: the bounds only."""
        _lib.require_cuda(q, kmin, kmax)
        n_kv, cap, d, hs = _meta_layout(kmin, kmax)
        if cand_offset < 1 or cand_offset + n_cand > cap or k > n_cand:
            raise ValueError("candidate range outside the metadata, or k > n_cand")
        if k > 0 and (out_idx is None or out_idx.dtype != torch.int32 or tuple(out_idx.shape) != (n_kv, k) or not out_idx.is_contiguous()):
            raise ValueError(f"out_idx must be contiguous int32 [{n_kv}, {k}]")
        if k == 0 and (out_bound is None or out_bound.dtype != torch.float32 or tuple(out_bound.shape) != (n_kv, n_cand) or not out_bound.is_contiguous()):
            raise ValueError(f"bounds only: out_bound must be contiguous float32 [{n_kv}, {n_cand}]")
        qq = q.reshape(-1, d)
        if not qq.is_contiguous() or qq.shape[0] % n_kv:
            raise ValueError("query must be contiguous [n_q, d] with n_q a multiple of the KV heads")
        ws = ws or default_workspace(q.device)
        ws_ptr, ws_n = ws.get(_lib.lib().lkv_bound_topk_workspace_bytes(n_kv, n_cand, k))
        self._keep = (q, kmin, kmax, out_idx, out_bound, ws.buf)
        self._fn = _lib.lib().lkv_bound_topk
        self._args = (qq.data_ptr(), _lib.dtype_code(qq.dtype), address(kmin), address(kmax),
                      _lib.dtype_code(kmin.dtype), hs, qq.shape[0], n_kv, d, cand_offset, n_cand, k, rank_mode, 0,
                      out_idx.data_ptr() if out_idx is not None else None, max(k, 1), out_bound.data_ptr() if out_bound is not None else None, ws_ptr, ws_n)
        self.device = q.device

    def __call__(self) -> None:
        rc = self._fn(torch.cuda.current_stream(self.device).cuda_stream, *self._args)
        if rc:
            _lib.check(rc, "bound_topk")


class PreparedDecode:
    """`sparse_decode` with every argument converted once; `desc` fields (fill, cur_block, rem
    range) may be updated between calls without re-preparing."""

    def __init__(self, q: torch.Tensor, *, n_kv: int, block_size: int, scale: float, sel: Source | None, idx: torch.Tensor | None, sink: Source | None, sink_block: int,
                 cur: Source | None, cur_block: int, fill: int, out: torch.Tensor, lse: torch.Tensor, rem: Source | None = None, rem_range: tuple[int, int] = (0, 0),
                 attend_selected: bool = True, ws: Workspace | None = None, max_rem_blocks: int = 0) -> None:
        qq = q.reshape(-1, q.shape[-1])
        n_q, d = qq.shape
        k = idx.shape[1] if idx is not None else 0
        self.desc = _lib.DecodeDesc(n_q, n_kv, d, block_size, float(scale), k, 1 if attend_selected else 0, sink_block, cur_block, fill, rem_range[0], rem_range[1])
        # Size the workspace for the largest remainder this call will be updated to.
        sizing = _lib.DecodeDesc(n_q, n_kv, d, block_size, float(scale), k, 1 if attend_selected else 0, sink_block, cur_block, fill, 0, max(rem_range[1] - rem_range[0], max_rem_blocks))
        ws = ws or default_workspace(q.device)
        ws_ptr, ws_n = ws.get(max(_lib.lib().lkv_sparse_decode_workspace_bytes(ctypes.byref(self.desc)), _lib.lib().lkv_sparse_decode_workspace_bytes(ctypes.byref(sizing))))
        self._c = [s.c() if s is not None else None for s in (sel, sink, cur, rem)]
        refs = [ctypes.byref(c) if c is not None else None for c in self._c]
        self._keep = (q, idx, out, lse, ws.buf, sel, sink, cur, rem)
        self._fn = _lib.lib().lkv_sparse_decode
        self._args = (ctypes.byref(self.desc), qq.data_ptr(), _lib.dtype_code(qq.dtype), refs[0], idx.data_ptr() if idx is not None else None, k,
                      refs[1], refs[2], refs[3], out.data_ptr(), _lib.dtype_code(out.dtype), lse.data_ptr(), ws_ptr, ws_n)
        self.device = q.device

    def __call__(self) -> None:
        rc = self._fn(torch.cuda.current_stream(self.device).cuda_stream, *self._args)
        if rc:
            _lib.check(rc, "sparse_decode")
