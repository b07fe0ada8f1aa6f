"""New tokens normalised, rotated and written to their rows, on the GPU against the definition in 64 bits.

With u = 2^-24 and h half a step of the model dtype: a sum of d squares in float32 is off by d u relative, its root and reciprocal by half of that and 3 u,
the products with the weight and the tables by 4 u more: a rotated value, of magnitude at most M = |y_i cos| + |y_j sin|, is off by at most (d / 2 + 8) u M
before it is rounded, by h relative (or half the least subnormal step of float16, 2^-25)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from chunk_cases import HALF, TYPES, U, Cache, int32, normal
from oracle import chunk as O
from oracle import rows as R

pytestmark = pytest.mark.gpu


def tables(positions: torch.Tensor, r: int, dtype: torch.dtype) -> tuple[torch.Tensor, torch.Tensor]:
    angle = positions.double()[..., None] * 10000.0 ** (-torch.arange(0, r, 2).double() / r)
    angle = torch.cat([angle, angle], -1)
    return angle.cos().to(dtype), angle.sin().to(dtype)


def close(got: np.ndarray, x: torch.Tensor, w: torch.Tensor | None, eps: float, cos: torch.Tensor | None, sin: torch.Tensor | None, dtype: torch.dtype) -> None:
    """got [heads, T, d] against the definition over x [heads, T, d]."""
    xd, d = x.double().cpu().numpy(), x.shape[-1]
    tab = [None if t is None else t.double().cpu().numpy() for t in (cos, sin)]
    wd = None if w is None else w.double().cpu().numpy()
    want = O.rotate(xd, wd, eps, *tab)
    y = np.abs(O.rotate(xd, wd, eps, None, None))
    size = y.copy()
    if cos is not None:
        r = tab[0].shape[-1]
        other = np.concatenate([y[..., r // 2 : r], y[..., : r // 2]], -1)
        size[..., :r] = y[..., :r] * np.abs(tab[0]) + other * np.abs(tab[1])
    tol = (d / 2 + 8) * U * size
    tol = tol * (1 + HALF[dtype]) + HALF[dtype] * np.abs(want) + (2.0**-25 if dtype == torch.float16 else 0.0)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4])


def case(seed: int, model: str, d: int, n_q: int, h: int, t: int, starts: list, counts: list | None, *, r: int, norm: bool, eight: bool = False, page: int = 0,
         wide: bool = False, shared: bool = False) -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(seed)
    dtype, seqs = TYPES[model], len(starts)
    room = max(starts) + t
    qkv = normal(gen, (seqs, t, n_q + 2 * h, d), model).cuda()
    q, k, v = (x.transpose(1, 2) for x in qkv.split((n_q, h, h), 2))
    cache = Cache(gen, seqs, h, room, d, model, eight=eight, page=page)
    before = cache.read()
    at = torch.arange(t)[None] + (0 if shared else torch.tensor(starts)[:, None])
    kind = torch.float32 if wide else dtype
    cos, sin = (x.cuda() for x in tables(at, r, kind)) if r else (None, None)
    wq, wk = ((torch.randn((2, d), generator=gen) * 0.3 + 1).to(kind).cuda().unbind(0)) if norm else (None, None)
    got = kernels.rotate_append(cache.rows, q, k, v, cos=cos, sin=sin, q_weight=wq, k_weight=wk, eps=1e-5, starts=int32(starts),
                                counts=None if counts is None else int32(counts), pages=cache.pages)
    torch.cuda.synchronize()
    out, after = got.double().cpu().numpy(), cache.read()
    same = kernels.rotate_append(kernels.dense_rows(*torch.empty((2, seqs, h, t, d), dtype=dtype, device="cuda")), q, k, v, cos=cos, sin=sin, q_weight=wq, k_weight=wk, eps=1e-5)
    assert torch.equal(same, got)
    for b in range(seqs):
        i = 0 if cos is not None and cos.shape[0] == 1 else b
        c, s = (None, None) if cos is None else (cos[i], sin[i])
        close(out[b], q[b], wq, 1e-5, c, s, dtype)
        n = t if counts is None else counts[b]
        mine = slice(starts[b], starts[b] + n)
        if eight:
            # As the rotated keys, rounded, are coded: those that a call into model-dtype rows gives.
            store = torch.empty((2, 1, h, t, d), dtype=dtype, device="cuda")
            kernels.rotate_append(kernels.dense_rows(store[0], store[1]), q[b : b + 1], k[b : b + 1], v[b : b + 1], cos=None if c is None else c[None],
                                  sin=None if s is None else s[None], q_weight=wq, k_weight=wk, eps=1e-5)
            close(store[0, 0].double().cpu().numpy(), k[b], wk, 1e-5, c, s, dtype)
            for x, y in zip(after, store.double().cpu().numpy()):
                assert np.array_equal(x[b, :, mine], R.mx_decode(*R.mx_encode(y[0, :, :n], model)))
        else:
            close(after[0][b, :, mine], k[b][:, :n], wk, 1e-5, None if c is None else c[:n], None if s is None else s[:n], dtype)
            assert np.array_equal(after[1][b, :, mine], v[b][:, :n].double().cpu().numpy())
        for x, y in zip(after, before):  # nothing else was written
            rest = np.ones(room, bool)
            rest[mine] = False
            assert np.array_equal(x[b][:, rest], y[b][:, rest])


@pytest.mark.parametrize("model", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("r", [0, 16, 48, 64])
@pytest.mark.parametrize(("eight", "page"), [(False, 0), (True, 16)])
def test_tokens_at_their_places(model: str, d: int, norm: bool, r: int, eight: bool, page: int) -> None:
    case(d + r, model, d, 4, 2, 5, [0, 30], None, r=r, norm=norm, eight=eight, page=page)


@pytest.mark.parametrize(("t", "starts", "counts"), [(1, [0], None), (1, [7, 0, 33], [1, 0, 1]), (17, [3, 20], [17, 1]), (100, [0, 1, 2], [99, 100, 0])])
@pytest.mark.parametrize(("n_q", "h"), [(1, 1), (3, 1), (5, 5), (14, 2)])
def test_counts_and_heads(t: int, starts: list, counts: list | None, n_q: int, h: int) -> None:
    case(t, "bf16", 128, n_q, h, t, starts, counts, r=128, norm=True, page=32)


@pytest.mark.parametrize("r", [32, 96, 112, 128])
def test_wide_tables_and_weights_and_one_table_for_all(r: int) -> None:
    case(r, "f16", 128, 4, 2, 9, [0, 0, 0], None, r=r, norm=True, wide=True, shared=True)


def test_far_positions_are_what_the_tables_say() -> None:
    case(3, "bf16", 128, 4, 2, 3, [131069], None, r=128, norm=False, wide=True, page=16)


def test_norms_of_zeros_large_and_small_values() -> None:
    from lazykv_amd import kernels

    x = torch.zeros((1, 2, 4, 64), dtype=torch.bfloat16, device="cuda")
    x[:, :, 1], x[:, :, 2], x[:, :, 3, 0] = 1e18, 1e-18, -2.0
    w = torch.ones(64, device="cuda")
    store = torch.empty((2, 1, 2, 4, 64), dtype=torch.bfloat16, device="cuda")
    q = kernels.rotate_append(kernels.dense_rows(store[0], store[1]), x, x, x, q_weight=w, k_weight=w, eps=1e-6)
    assert torch.all(q[:, :, 0] == 0) and torch.all((q[:, :, 1] - 1).abs() < 2**-7) and torch.all((q[:, :, 2].float() / 1e-15 - 1).abs() < 2**-7)
    assert torch.all((q[:, :, 3, 0] + 8).abs() < 2**-5) and torch.all(q[:, :, 3, 1:] == 0)
    assert torch.equal(store[0], q) and torch.equal(store[1], x)


def test_rows_outside_the_cache_and_pages_that_a_pool_lacks_are_dropped() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(1)
    k = normal(gen, (3, 2, 10, 64), "f16").cuda()
    for page in (0, 16):
        cache = Cache(gen, 3, 2, 32, 64, "f16", page=page)
        before = cache.read()
        pages = cache.pages
        if page:
            pages = pages.clone()
            pages[2, 1] = 1 << 20
        kernels.rotate_append(cache.rows, k, k, k, starts=int32([-4, 28, 12]), pages=pages)
        after, new = cache.read(), k.double().cpu().numpy()
        for x, y in zip(after, before):
            assert np.array_equal(x[0, :, :6], new[0, :, 4:]) and np.array_equal(x[0, :, 6:], y[0, :, 6:])
            assert np.array_equal(x[1, :, 28:], new[1, :, :4]) and np.array_equal(x[1, :, :28], y[1, :, :28])
            end = 16 if page else 22
            assert np.array_equal(x[2, :, 12:end], new[2, :, : end - 12]) and np.array_equal(x[2, :, end:], y[2, :, end:])


def test_a_captured_call_follows_starts_and_counts() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(2)
    q, k = normal(gen, (2, 4, 3, 64), "f16").cuda(), normal(gen, (2, 2, 3, 64), "f16").cuda()
    cos, sin = (x.cuda() for x in tables(torch.arange(3)[None], 64, torch.float16))
    starts, counts = int32([0, 0]), int32([3, 3])
    caches = [Cache(torch.Generator().manual_seed(3), 2, 2, 40, 64, "f16", page=16, eight=True) for _ in range(2)]
    call = lambda c: kernels.rotate_append(c.rows, q, k, k, cos=cos, sin=sin, starts=starts, counts=counts, pages=c.pages)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(caches[0])
    torch.cuda.current_stream().wait_stream(side)
    call(caches[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(caches[0])
    for a, b, c, d in [(0, 5, 3, 1), (20, 37, 2, 3), (11, 12, 0, 2)]:
        starts.copy_(int32([a, b]))
        counts.copy_(int32([c, d]))
        q.mul_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        want = call(caches[1])
        assert torch.equal(out, want)
        assert all(torch.equal(x, y) for x, y in zip(caches[0].held, caches[1].held))


def test_a_caches_own_rows_are_read_before_they_are_written() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(4)
    store = normal(gen, (2, 1, 2, 64, 128), "bf16").cuda()
    rows = kernels.dense_rows(store[0], store[1])
    want = store.clone()
    q = kernels.rotate_append(rows, store[0][:, :, 3:40], store[0][:, :, 3:40], store[1][:, :, 3:40], start=4)
    assert torch.equal(q, want[0][:, :, 3:40]) and torch.equal(store[:, :, :, 4:41], want[:, :, :, 3:40])


def test_what_is_refused() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(5)
    q, k = normal(gen, (2, 4, 3, 64), "f16").cuda(), normal(gen, (2, 2, 3, 64), "f16").cuda()
    cache = Cache(gen, 2, 2, 32, 64, "f16", page=16)
    kw = dict(pages=cache.pages)
    cos = torch.ones((1, 3, 64), dtype=torch.float16, device="cuda")
    for what, args, more in (
        ("expected", (q, k, k.bfloat16()), {}), ("do not match", (q, q, q), {}), ("come together", (q, k, k), {"cos": cos}), ("cos/sin", (q, k, k), {"cos": cos[:, :2], "sin": cos[:, :2]}),
        ("multiple of 16", (q, k, k), {"cos": cos[..., :24], "sin": cos[..., :24]}), ("weights must", (q, k, k), {"q_weight": cos[0, 0, :32]}), ("exceed", (q, k, k), {"start": 30}),
        ("exceed", (q, k, k), {"start": -1}), ("eps", (q, k, k), {"eps": -1.0}), ("must not lie among", (q, k, k), {"out": q}), ("out must be", (q, k, k), {"out": q[:, :2]}),
        ("starts must", (q, k, k), {"starts": torch.zeros(2, device="cuda")}), ("counts must", (q, k, k), {"counts": int32([1])}),
    ):
        with pytest.raises(ValueError, match=what):
            kernels.rotate_append(cache.rows, *args, **{**kw, **more})
    with pytest.raises(ValueError, match="share an address"):
        kernels.rotate_append(kernels.dense_rows(*(x.expand(2, -1, -1, -1) for x in torch.zeros((2, 1, 2, 8, 64), dtype=torch.float16, device="cuda"))), q, k, k)
    with pytest.raises(RuntimeError, match="no gradient"):
        kernels.rotate_append(cache.rows, q.clone().requires_grad_(), k, k, **kw)
    assert kernels.rotate_append(cache.rows, q[:, :, :0], k[:, :, :0], k[:, :, :0], **kw).shape == (2, 4, 0, 64)


@pytest.mark.parametrize("out_of", ["channels", "heads", "tokens of one"])
def test_queries_however_they_lie(out_of: str) -> None:
    """Queries whose channels are not innermost, or whose single token's stride is no multiple of 8: as contiguous ones, to the bit."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(11)
    t = 1 if out_of == "tokens of one" else 8
    q, k = normal(gen, (2, 4, t, 64), "bf16").cuda(), normal(gen, (2, 2, t, 64), "bf16").cuda()
    if out_of == "channels":
        x = q.transpose(2, 3).contiguous().transpose(2, 3)
    elif out_of == "heads":
        x = q.contiguous(memory_format=torch.channels_last)
    else:
        x = q.as_strided(q.shape, (256, 64, 3, 1))
    assert torch.equal(x, q) and (x.stride(3) != 1 or x.stride(2) == 3)
    cos, sin = (y.cuda() for y in tables(torch.arange(t)[None], 64, torch.bfloat16))
    stores = [torch.zeros((2, 2, 2, t, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    got, want = (kernels.rotate_append(kernels.dense_rows(s[0], s[1]), y, k, k, cos=cos, sin=sin) for s, y in zip(stores, (x, q)))
    assert torch.equal(got, want) and torch.equal(*stores)


def test_norms_without_eps_of_values_whose_squares_are_subnormal() -> None:
    """Squares of 1e-19 and less lie below float32's normal range, down to 2^-149: with a square of m steps of that, in float32, a mean is off by one step in m (half a step a
    square, half of the division), its root by half of that: 2^-7 at 3e-22 (m = 64), and bfloat16 rounds by 2^-8. Heads of zeros give 0 / 0."""
    from lazykv_amd import kernels

    sizes = (2.0**-62, 2.0**-63, 1e-19, 1e-20, 1e-21, 3e-22)
    x = torch.stack([torch.where(torch.arange(64) % 3 == 0, -s, s) for s in sizes] + [torch.zeros(64)]).bfloat16().cuda().expand(1, 2, 7, 64).contiguous()
    w = torch.full((64,), 1.5, device="cuda")
    store = torch.empty((2, 1, 2, 7, 64), dtype=torch.bfloat16, device="cuda")
    q = kernels.rotate_append(kernels.dense_rows(store[0], store[1]), x, x, x, q_weight=w, k_weight=w, eps=0.0)
    want = 1.5 * x[:, :, :6].sign().float()
    assert torch.all((q[:, :, :6].float() - want).abs() <= 1.5 * (2.0**-8 + 2.0**-7)) and q[:, :, 6].isnan().all()
    assert torch.equal(store[0][:, :, :6], q[:, :, :6])
