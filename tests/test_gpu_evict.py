"""The weights that rows get, summed up, and rows over a budget evicted by them, on the GPU against the definitions in 64 bits.

A weight exp(s - lse) is off by e = ((d + 8) S + 4 + 2 |lse|) u relative (u = 2^-24, S the largest sum of a score's magnitudes; the lse enters as lse / scale, rounded
twice), a sum of m weights in float32 by m u, so a row's sum by (e + (m + 4) u) times itself, and 2^-120 for weights below float32's normal range."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from chunk_cases import TYPES, U, Cache, int32, normal
from oracle import chunk as O

pytestmark = pytest.mark.gpu


def weigh_case(seed: int, model: str, d: int, h: int, g: int, t: int, lens: list, counts: list | None = None, *, eight: bool = False, page: int = 0, into: bool = True) -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(seed)
    seqs, most, scale = len(lens), max(lens), d**-0.5
    n = counts or [t] * seqs
    q = (torch.randn((seqs, t, h * g, d), generator=gen) * 1.5).to(TYPES[model]).cuda().transpose(1, 2)
    cache = Cache(gen, seqs, h, most, d, model, eight=eight, page=page, room=3)
    qd = q.double().cpu().numpy()
    lse = np.full((seqs, h * g, t), -np.inf, np.float32)
    for b in range(seqs):
        for j in range(h * g):
            k, v = (x[b, j // g, : lens[b]] for x in cache.values)
            lse[b, j] = O.attend(qd[b, j], k, v, n[b], scale)[1]
    old = torch.rand((seqs, h, most + 5), generator=gen).cuda()
    sums = old.clone()
    positions = torch.full((seqs, h, most + 2), -7, dtype=torch.int32, device="cuda")
    seen = int32([1000 * (b + 1) for b in range(seqs)])
    out = sums if into else torch.full_like(old, 5.0)
    got = kernels.weigh_rows(q, torch.from_numpy(lse).cuda(), cache.rows, scale=scale, lengths=int32(lens), counts=None if counts is None else int32(counts), max_tokens=most,
                             pages=cache.pages, sums=sums, out=None if into else out, positions=positions, seen=seen)
    assert got is out
    got, at = got.double().cpu().numpy(), positions.cpu().numpy()
    if not into:
        assert torch.equal(sums, old)
    old = old.double().cpu().numpy()
    for b in range(seqs):
        past = lens[b] - n[b]
        for j in range(h):
            mine = slice(j * g, (j + 1) * g)
            k = cache.values[0][b, j, : lens[b]]
            want = O.weigh(qd[b, mine], k, lse[b, mine].astype(np.float64), n[b], scale)
            size = max((np.abs(x) @ np.abs(k).T).max(initial=0.0) for x in qd[b, mine]) * scale
            top = np.abs(lse[b, mine], where=np.isfinite(lse[b, mine]), out=np.zeros((g, t), np.float32)).max(initial=0.0)
            tol = (((d + 8) * size + 4 + 2 * top) + g * t + 4) * U * want + 2.0**-120
            first = max(past, 0)
            want[:first] += old[b, j, :first]
            tol[:first] += 2 * U * want[:first]
            bad = ~(np.abs(got[b, j, : lens[b]] - want) <= tol)
            assert not bad.any(), (b, j, np.argwhere(bad)[:4].ravel(), got[b, j, : lens[b]][bad][:4], want[bad][:4])
            assert np.all(got[b, j, lens[b] :] == (old[b, j, lens[b] :] if into else 5.0))
            assert np.all(at[b, j, first : lens[b]] == 1000 * (b + 1) + np.arange(first - past, n[b])) and np.all(at[b, j, :first] == -7) and np.all(at[b, j, lens[b] :] == -7)


@pytest.mark.parametrize("model", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize(("eight", "page"), [(False, 0), (False, 16), (True, 0), (True, 48)])
@pytest.mark.parametrize(("t", "n"), [(1, 1), (1, 63), (1, 64), (1, 300), (3, 17), (20, 20), (33, 290), (70, 129)])
def test_weights_summed(model: str, d: int, eight: bool, page: int, t: int, n: int) -> None:
    weigh_case(n, model, d, 2, 4, t, [n, max(t, n // 2)], eight=eight, page=page)


@pytest.mark.parametrize("g", [1, 2, 3, 5, 16, 17])
@pytest.mark.parametrize("t", [1, 9])
def test_weights_of_groups(g: int, t: int) -> None:
    weigh_case(g, "bf16", 64, 3, g, t, [t + 50, t], page=16, into=False)


@pytest.mark.parametrize(("t", "lens", "counts"), [(1, [0, 5, 200], [0, 1, 1]), (5, [9, 0, 5, 33], [5, 0, 1, 4]), (40, [90, 40, 7, 300], [40, 1, 7, 39]), (4, [2, 1], [4, 3])])
def test_weights_of_ragged_batches(t: int, lens: list, counts: list) -> None:
    weigh_case(t, "bf16", 128, 2, 4, t, lens, counts, page=16)


@pytest.mark.parametrize(("t", "n"), [(500, 500), (300, 3000)])
def test_weights_in_parts(t: int, n: int) -> None:
    weigh_case(t, "f16", 64, 1, 4, t, [n], page=64)


def test_weights_of_what_is_not_attended_or_not_there() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(3)
    t, n, d = 20, 90, 64
    q = normal(gen, (1, 4, t, d), "f16").cuda()
    cache = Cache(gen, 1, 1, n, d, "f16", page=16)
    kw = dict(scale=0.125, tokens=n, pages=cache.pages)
    lse = kernels.chunk_attend(q, cache.rows, **kw)[1]
    want = kernels.weigh_rows(q, lse, cache.rows, **kw)
    assert abs(want.double().sum().item() - 4 * t) < 1e-3
    # A key of the chunk that is not finite: only its own row shows it.
    where, i = cache.place(0, 80)
    cache.held[0][0, where, 0, i, 3] = float("nan")
    got = kernels.weigh_rows(q, lse, cache.rows, **kw)
    assert got[0, 0, 80].isnan() and torch.equal(got[0, 0, :80], want[0, 0, :80]) and torch.equal(got[0, 0, 81:], want[0, 0, 81:])
    # Tokens whose lse is -inf add nothing, whatever their queries hold.
    q2, lse2 = q.clone(), lse.clone()
    q2[:, :, 7:], lse2[:, :, 7:] = float("nan"), -float("inf")
    table = cache.pages.clone()
    table[0, 2] = -1
    some = kernels.weigh_rows(q2[:, :, :7], lse2[:, :, :7].contiguous(), cache.rows, scale=0.125, lengths=int32([n]), counts=int32([7]), max_tokens=n, pages=table)
    assert torch.all(some[0, 0, 32:48] == 0) and some[0, 0, :32].isfinite().all()
    more = kernels.weigh_rows(q2, lse2, cache.rows, scale=0.125, lengths=int32([n]), counts=int32([7]), max_tokens=n, pages=table)
    # Seven tokens and twenty may take different kernels, each within the bound above of the same sums: they differ by twice that at the most.
    k = torch.from_numpy(cache.values[0][0, 0]).cuda()
    size = (q[:, :, :7].double().abs() @ k.abs().T).max().item() * 0.125
    rel = 2 * ((d + 8) * size + 4 + 2 * lse[:, :, :7].abs().max().item() + 4 * 7 + 4) * U
    assert torch.all((more[0, 0, :80] - some[0, 0, :80]).abs() <= rel * some[0, 0, :80])
    # (The chunk's rows are 70 .. 89 here: its first seven tokens attend up to row 76.)
    less = kernels.weigh_rows(q2, lse2, cache.rows, scale=0.125, tokens=n, pages=cache.pages)
    assert less[0, 0, :80].isfinite().all() and torch.all(less[0, 0, 77:80] == 0)


@pytest.mark.parametrize(("t", "d"), [(20, 64), (20, 128), (6, 128)])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_a_query_reaches_only_the_rows_that_it_attends(t: int, d: int, what: float) -> None:
    """One token's query, or its lse, is not finite: the rows behind those that it attends are as without it, to the bit."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(t)
    past, at = 300, t // 2
    n = past + t
    q = normal(gen, (1, 8, t, d), "bf16").cuda()
    cache = Cache(gen, 1, 2, n, d, "bf16", page=16)
    kw = dict(scale=0.1, tokens=n, pages=cache.pages)
    lse = kernels.chunk_attend(q, cache.rows, **kw)[1]
    want = kernels.weigh_rows(q, lse, cache.rows, **kw)
    q2, lse2 = q.clone(), lse.clone()
    q2[0, 1, at], lse2[0, 5, at] = what, float("nan")
    for x, y, head in ((q2, lse, 0), (q, lse2, 1)):
        got = kernels.weigh_rows(x, y, cache.rows, **kw)
        assert torch.equal(got[0, 1 - head], want[0, 1 - head]) and torch.equal(got[0, head, past + at + 1 :], want[0, head, past + at + 1 :])
    got = kernels.weigh_rows(q, lse2, cache.rows, **kw)
    assert got[0, 1, : past + at + 1].isnan().all()


def test_a_captured_account_follows_lengths_and_pages() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(9)
    for t in (2, 40, 200):
        q = normal(gen, (2, 8, t, 64), "f16").cuda()
        cache = Cache(gen, 2, 2, 700, 64, "f16", page=16)
        lengths, counts, seen, pages = int32([700, 213]), int32([t, t]), int32([0, 5]), cache.pages.clone()
        lse = torch.randn((2, 8, t), generator=gen).cuda() + 4
        old = torch.rand((2, 2, 700), generator=gen).cuda()
        kw = dict(scale=0.09, lengths=lengths, counts=counts, max_tokens=700, pages=pages, seen=seen)
        held = [[old.clone(), torch.zeros((2, 2, 700), dtype=torch.int32, device="cuda")] for _ in range(2)]
        call = lambda i: kernels.weigh_rows(q, lse, cache.rows, sums=held[i][0], positions=held[i][1], **kw)  # noqa: E731, B023
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(0)
        torch.cuda.current_stream().wait_stream(side)
        call(1)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            call(0)
        for i, (a, b, c, d) in enumerate([(700, 213, t, 1), (5, 699, min(5, t), t), (0, 1, 0, 1), (350, 351, t, t)]):
            lengths.copy_(int32([a, b]))
            counts.copy_(int32([c, d]))
            pages.copy_(cache.pages.flip(0) if i == 3 else cache.pages)
            lse.add_(0.25)
            graph.replay()
            torch.cuda.synchronize()
            call(1)
            for x, y in zip(*held):  # to the bit; swapped pages bring rows of nobody's, which hold NaN, before the end
                torch.testing.assert_close(x, y, rtol=0, atol=0, equal_nan=True)


def test_weights_past_32_bits_of_bytes() -> None:
    """One head of 17 million rows: the last ones get what they would at a cache's start, in the few rows' form and in the other."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(10)
    n = (1 << 24) + 4096
    keys = torch.zeros((1, 1, n, 128), dtype=torch.bfloat16, device="cuda")
    tail = normal(gen, (1, 1, 4096, 128), "bf16").cuda()
    keys[:, :, -4096:] = tail
    for t in (1, 40):
        q, lse = normal(gen, (1, 2, t, 128), "bf16").cuda(), torch.full((1, 2, t), 20.0, device="cuda")
        got = kernels.weigh_rows(q, lse, kernels.dense_rows(keys, keys), scale=0.09, tokens=n)
        want = kernels.weigh_rows(q, lse, kernels.dense_rows(tail, tail), scale=0.09, tokens=4096)
        assert torch.equal(got[..., -4096:], want) or t > 1  # parts may differ with the length: their order of sums too
        # g t weights, each the same number, summed in float32 in two orders.
        assert torch.all((got[..., -4096:] - want).abs() <= 2 * 2 * t * U * want)
        assert torch.all((got[..., :-4096] - 2 * t * np.exp(-20.0)).abs() <= (2 * t + 60) * U * 2 * t * np.exp(-20.0))


def evict_case(seed: int, seqs: int, h: int, n: int, keep: int, sinks: int, recent: int, lens: list | None = None, *, eight: bool = False, page: int = 0, d: int = 64,
               ties: bool = False, apart: bool = False, special: bool = False) -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(seed)
    lens = lens or [n] * seqs
    cache = Cache(gen, seqs, h, n, d, "f16", eight=eight, page=page)
    sums = torch.randint(0, 4, (seqs, h, n + 3), generator=gen).float() if ties else torch.randn((seqs, h, n + 3), generator=gen).exp()
    if special:
        for i, x in enumerate((float("nan"), float("inf"), -float("inf"), -0.0, 0.0, 1e-42, -1.0, float("nan"))):
            sums[:, :, i::11] = x
    positions = torch.stack([torch.randperm(3 * n + 3, generator=gen)[: n + 3] for _ in range(seqs * h)]).view(seqs, h, n + 3).int()
    args = [sums.cuda(), positions.cuda()]
    to = [torch.full_like(x, -3) for x in args] if apart else args
    before = cache.read()
    kernels.evict_rows(cache.rows, *args, keep=keep, sinks=sinks, recent=recent, lengths=int32(lens), max_tokens=n, pages=cache.pages, out=tuple(to) if apart else None)
    torch.cuda.synchronize()
    after = cache.read()
    got = [x.cpu().numpy() for x in to]
    for b in range(seqs):
        for j in range(h):
            m = lens[b]
            s, p = sums[b, j].numpy().copy(), positions[b, j].numpy().copy()
            dst, src = O.evict(s[:m], p[:m], keep, sinks, recent)
            want = [x[b, j].copy() for x in before]
            for x in (*want, s, p):
                x[dst] = x[src]
            left = min(m, keep)
            for x, y in zip(want, after):
                assert np.array_equal(x, y[b, j]), (b, j)
            assert np.array_equal(got[0][b, j][:left], s[:left], equal_nan=True) and np.array_equal(got[1][b, j][:left], p[:left]), (b, j)
            if apart:
                assert np.all(got[0][b, j][left:] == -3) and np.all(got[1][b, j][left:] == -3)
            else:
                assert np.array_equal(got[0][b, j][left:], s[left:], equal_nan=True) and np.array_equal(got[1][b, j][left:], p[left:])


@pytest.mark.parametrize(("n", "keep"), [(1, 1), (2, 1), (17, 16), (17, 1), (64, 63), (100, 50), (1000, 37), (1000, 999), (5000, 1234), (300, 300), (300, 400)])
@pytest.mark.parametrize(("eight", "page", "d"), [(False, 0, 64), (True, 16, 128), (False, 48, 128)])
@pytest.mark.parametrize("ties", [False, True])
def test_the_rows_that_stay(n: int, keep: int, eight: bool, page: int, d: int, ties: bool) -> None:
    evict_case(n, 1, 2, n, keep, 0, 0, eight=eight, page=page, d=d, ties=ties)


@pytest.mark.parametrize(("keep", "sinks", "recent"), [(40, 4, 16), (40, 40, 0), (40, 0, 40), (40, 20, 20), (100, 1, 60)])
@pytest.mark.parametrize("apart", [False, True])
def test_first_and_newest_tokens(keep: int, sinks: int, recent: int, apart: bool) -> None:
    evict_case(keep, 3, 2, 130, keep, sinks, recent, [130, 0, 77], page=16, apart=apart)


@pytest.mark.parametrize("keep", [3, 30, 75])
def test_sums_that_are_not_finite_or_alike(keep: int) -> None:
    evict_case(keep, 2, 2, 90, keep, 2, 1, special=True)


@pytest.mark.parametrize(("n", "keep"), [(20000, 5000), (40007, 39000), (70001, 128)])
def test_long_caches(n: int, keep: int) -> None:
    """Rows by their keys' one channel alone: which rows stay, in which places."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(n)
    store = torch.zeros((2, 1, 2, n, 64), dtype=torch.float16, device="cuda")
    mark = torch.arange(n, device="cuda")
    store[0, 0, :, :, 0], store[0, 0, :, :, 1], store[1, 0, :, :, 2] = (mark % 1000).half(), (mark // 1000).half(), (mark % 777).half()
    was = store.clone()
    sums = torch.randn((1, 2, n), generator=gen).exp().cuda()
    sums[0, 1] = (sums[0, 1] * 4).floor()
    positions = torch.randperm(n, generator=gen).int().expand(1, 2, n).contiguous().cuda()
    s, p = sums.cpu().numpy().copy(), positions.cpu().numpy().copy()
    kernels.evict_rows(kernels.dense_rows(store[0], store[1]), sums, positions, keep=keep, sinks=4, recent=100, tokens=n)
    for j in range(2):
        to, of = (torch.from_numpy(x).cuda() for x in O.evict(s[0, j], p[0, j], keep, 4, 100))
        want = was[:, 0, j].clone()
        want[:, to] = want[:, of]
        assert torch.equal(store[:, 0, j], want)
        wanted = torch.from_numpy(p[0, j]).cuda()
        wanted[to] = wanted[of]
        assert torch.equal(positions[0, j], wanted)


def test_a_captured_eviction_follows_lengths() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(4)
    caches = [Cache(torch.Generator().manual_seed(5), 2, 2, 100, 64, "f16", page=16) for _ in range(2)]
    sums, positions = torch.rand((2, 2, 100), generator=gen).cuda(), torch.arange(100, dtype=torch.int32).expand(2, 2, 100).contiguous().cuda()
    lengths = int32([100, 70])
    to = [[torch.zeros_like(x) for x in (sums, positions)] for _ in range(2)]
    call = lambda i: kernels.evict_rows(caches[i].rows, sums, positions, keep=40, recent=8, lengths=lengths, max_tokens=100, pages=caches[i].pages, out=tuple(to[i]))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(0)
    torch.cuda.current_stream().wait_stream(side)
    call(1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(0)
    for a, b in ((100, 41), (40, 99), (0, 100)):
        lengths.copy_(int32([a, b]))
        sums.copy_(torch.rand((2, 2, 100), generator=gen))
        graph.replay()
        torch.cuda.synchronize()
        call(1)
        for x, y in zip((*caches[0].held, *to[0]), (*caches[1].held, *to[1])):  # to the bit; pages of nobody's hold NaN
            torch.testing.assert_close(x, y, rtol=0, atol=0, equal_nan=True)


def test_a_captured_long_eviction_follows_lengths_and_sums() -> None:
    """Twice the long form in one graph, on caches and scratch of their own."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(14)
    n, keep = 20011, 5000
    stores = [torch.zeros((2, 2, 1, n, 64), dtype=torch.float16, device="cuda") for _ in range(3)]
    sums, positions = torch.rand((2, 1, n), generator=gen).cuda(), torch.arange(n, dtype=torch.int32, device="cuda").expand(2, 1, n).contiguous()
    lengths = int32([n, n])
    to = [[torch.zeros_like(x) for x in (sums, positions)] for _ in range(3)]
    call = lambda i: kernels.evict_rows(kernels.dense_rows(*stores[i]), sums, positions, keep=keep, sinks=4, recent=100, lengths=lengths, max_tokens=n, out=tuple(to[i]))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(0)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(0)
        call(1)
    fresh = normal(gen, (2, 2, 1, n, 64), "f16").cuda()
    for a, b in ((n, 16000), (5001, 0), (4999, n - 1)):
        lengths.copy_(int32([a, b]))
        sums.copy_(torch.rand((2, 1, n), generator=gen).mul_(8).floor() if b == 0 else torch.rand((2, 1, n), generator=gen))
        for x in stores:
            x.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        call(2)
        for i in range(2):
            assert torch.equal(stores[i], stores[2]) and all(torch.equal(x, y) for x, y in zip(to[i], to[2]))


def test_pages_that_a_pool_lacks_are_not_moved() -> None:
    """A row whose page is not there keeps its rank: its sums and positions move, and no keys or values."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(15)
    cache = Cache(gen, 1, 1, 64, 64, "f16", page=16)
    before = cache.read()
    sums, positions = torch.arange(64.0, device="cuda").expand(1, 1, 64).contiguous(), torch.arange(64, dtype=torch.int32, device="cuda").expand(1, 1, 64).contiguous()
    pages = cache.pages.clone()
    pages[0, 0], pages[0, 3] = -5, cache.rows.seqs
    kernels.evict_rows(cache.rows, sums, positions, keep=32, tokens=64, pages=pages)  # rows 32 .. 63 stay, in places 0 .. 31
    assert torch.equal(sums[0, 0, :32], torch.arange(32.0, 64.0, device="cuda")) and torch.equal(positions[0, 0, :32].cpu(), torch.arange(32, 64, dtype=torch.int32))
    for x, y in zip(cache.read(), before):
        assert np.array_equal(x, y)  # rows 32 .. 47 to a page that is not there, rows 48 .. 63 from one


def test_calls_without_tokens_or_rows() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(17)
    cache = Cache(gen, 2, 2, 64, 64, "f16", page=16)
    sums, out = torch.rand((2, 2, 64), generator=gen).cuda(), torch.full((2, 2, 64), 5.0, device="cuda")
    q, lse = torch.zeros((2, 4, 0, 64), dtype=torch.float16, device="cuda"), torch.zeros((2, 4, 0), device="cuda")
    got = kernels.weigh_rows(q, lse, cache.rows, scale=0.1, lengths=int32([50, 0]), pages=cache.pages, sums=sums, out=out)
    assert torch.equal(got[0, :, :50], sums[0, :, :50]) and torch.all(got[0, :, 50:] == 5) and torch.all(got[1] == 5)
    before = cache.read()
    none, nowhere = torch.zeros((2, 2, 0), device="cuda"), torch.zeros((2, 2, 0), dtype=torch.int32, device="cuda")
    kernels.evict_rows(cache.rows, none, nowhere, keep=4, tokens=0, pages=cache.pages)
    kernels.evict_rows(cache.rows, sums[:0], torch.zeros((0, 2, 64), dtype=torch.int32, device="cuda"), keep=4, tokens=9, pages=cache.pages[:0])
    assert all(np.array_equal(x, y) for x, y in zip(cache.read(), before))
    for tokens, most in ((-1, 4), (4, -1)):
        with pytest.raises(ValueError, match="bad extent"):
            kernels.weigh_rows(torch.zeros((2, 4, 1, 64), dtype=torch.float16, device="cuda"), torch.zeros((2, 4, 1), device="cuda"), cache.rows, scale=0.1, tokens=tokens,
                               max_tokens=most, lengths=int32([1, 1]), pages=cache.pages)


def test_two_streams_evict_and_account_at_once() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(16)
    n, keep = 18000, 6000
    first = normal(gen, (2, 1, 2, n, 64), "f16").cuda()
    q, lse = normal(gen, (1, 8, 100, 64), "f16").cuda(), torch.full((1, 8, 100), 9.0, device="cuda")
    results = []

    def both() -> tuple:
        store = first.clone()
        rows = kernels.dense_rows(store[0], store[1])
        positions = torch.zeros((1, 2, n), dtype=torch.int32, device="cuda")
        sums = kernels.weigh_rows(q, lse, rows, scale=0.1, tokens=n, positions=positions)
        positions[..., : n - 100] = torch.arange(n - 100, device="cuda")
        kernels.evict_rows(rows, sums, positions, keep=keep, sinks=2, recent=500, tokens=n)
        return store, sums, positions

    want = both()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                results.append(both())
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for got in results for x, y in zip(got, want))


def test_what_is_refused() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(6)
    cache = Cache(gen, 2, 2, 64, 64, "f16", page=16)
    sums, positions = torch.zeros((2, 2, 64), device="cuda"), torch.zeros((2, 2, 64), dtype=torch.int32, device="cuda")
    kw = dict(tokens=64, pages=cache.pages)
    for what, args, more in (
        ("first and", (sums, positions), {"keep": 4, "sinks": 3, "recent": 2}), ("first and", (sums, positions), {"keep": 0}), ("sums must", (sums.half(), positions), {"keep": 4}),
        ("positions must", (sums, positions.long()), {"keep": 4}), ("sums must", (sums[:, :, :63], positions), {"keep": 4}), ("share addresses", (sums[:, :1].expand(2, 2, 64), positions), {"keep": 4}),
        ("share addresses", (sums, sums.view(torch.int32)), {"keep": 4}), ("rows of a sequence over", (torch.zeros((2, 2, 99), device="cuda"), positions.new_zeros((2, 2, 99))), {"keep": 4, "tokens": 65}),
        ("overlap", (sums, positions), {"keep": 4, "out": (torch.zeros((2, 2, 64), device="cuda"), positions[:, :, 1:])}),
    ):
        with pytest.raises(ValueError, match=what):
            kernels.evict_rows(cache.rows, *args, **{**kw, **more})
    q = normal(gen, (2, 4, 3, 64), "f16").cuda()
    lse = torch.zeros((2, 4, 3), device="cuda")
    for what, args, more in (
        ("lse must", (q, lse[:, :, :2]), {}), ("sums must", (q, lse), {"sums": sums[:1]}), ("seen says", (q, lse), {"seen": int32([1, 2])}), ("positions must", (q, lse), {"positions": sums}),
        ("must not lie", (q, lse), {"out": sums, "positions": sums.view(torch.int32)}), ("overlap", (q, lse), {"sums": torch.zeros((2, 2, 65), device="cuda")[:, :, 1:], "out": sums[:, :, :0]}),
    ):
        if what == "overlap":
            both = torch.zeros((2, 2, 65), device="cuda")
            more = {"sums": both[:, :, 1:], "out": both[:, :, :64]}
        with pytest.raises(ValueError, match=what):
            kernels.weigh_rows(*args, cache.rows, scale=0.1, **{**kw, **more})
    with pytest.raises(RuntimeError, match="no gradient"):
        kernels.evict_rows(cache.rows, sums.clone().requires_grad_(), positions, keep=4, **kw)


@pytest.mark.parametrize("eight", [False, True])
def test_a_layers_decode_over_a_bounded_cache(eight: bool) -> None:
    """A prompt and forty steps of two sequences through one layer, all four calls: the cache stays at its budget, and at each step the attention is that over the
    rows that a plain account of the same rules has."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(7)
    seqs, h, g, d, keep, room, page = 2, 2, 2, 64, 48, 64, 16
    cache = Cache(gen, seqs, h, room, d, "bf16", eight=eight, page=page)
    sums, positions = torch.zeros((seqs, h, room), device="cuda"), torch.zeros((seqs, h, room), dtype=torch.int32, device="cuda")
    lengths, seen = int32([0, 0]), int32([0, 0])
    lens = [0, 0]
    held = [[{} for _ in range(h)] for _ in range(seqs)]  # position: its sum, as the plain account has it
    scale, weight = d**-0.5, (torch.rand((d,), generator=gen) + 0.5).bfloat16().cuda()
    angle = torch.arange(400.0)[:, None] * 10000.0 ** (-torch.arange(0, d, 2) / d)
    cos, sin = (torch.cat([x, x], -1).bfloat16().cuda() for x in (angle.cos(), angle.sin()))
    for step in range(41):
        t = 30 if step == 0 else 16 if step % 7 == 3 else 1
        q, k, v = (normal(gen, (seqs, n, t, d), "bf16").cuda() for n in (h * g, h, h))
        at = seen.long()[:, None] + torch.arange(t, device="cuda")
        q = kernels.rotate_append(cache.rows, q, k, v, cos=cos[at], sin=sin[at], q_weight=weight, k_weight=weight, starts=lengths, pages=cache.pages)
        lengths += t
        lens = [n + t for n in lens]
        kw = dict(scale=scale, lengths=lengths, max_tokens=room, pages=cache.pages)
        out, lse = kernels.chunk_attend(q, cache.rows, **kw)
        kernels.weigh_rows(q, lse, cache.rows, sums=sums, positions=positions, seen=seen, **kw)
        rows, places = cache.read(), positions.cpu().numpy()
        qd, od, sd = q.double().cpu().numpy(), out.double().cpu().numpy(), sums.double().cpu().numpy()
        for b in range(seqs):
            for j in range(h):
                kk, vv = (x[b, j, : lens[b]] for x in rows)
                for i in range(j * g, (j + 1) * g):
                    want, _, a, _ = O.attend(qd[b, i], kk, vv, t, scale)
                    assert np.all(np.abs(od[b, i] - want) <= 2.0**-7 * a + 2.0**-8 * np.abs(want) + 1e-6)
                ls = np.stack([O.attend(qd[b, i], kk, vv, t, scale)[1] for i in range(j * g, (j + 1) * g)])
                got = O.weigh(qd[b, j * g : (j + 1) * g], kk, ls, t, scale)
                account = held[b][j]
                for row, p in enumerate(places[b, j, : lens[b]]):
                    account[int(p)] = account.get(int(p), 0.0) + got[row]
                assert set(account) == set(places[b, j, : lens[b]].tolist())
                assert np.allclose(sd[b, j, : lens[b]], [account[int(p)] for p in places[b, j, : lens[b]]], rtol=1e-4, atol=1e-6)
        kernels.evict_rows(cache.rows, sums, positions, keep=keep, sinks=2, recent=8, lengths=lengths, max_tokens=room, pages=cache.pages)
        lengths.clamp_(max=keep)
        seen += t
        lens = [min(n, keep) for n in lens]
        places, newest = positions.cpu().numpy(), int(seen[0]) - 1
        for b in range(seqs):
            for j in range(h):
                left = set(places[b, j, : lens[b]].tolist())
                assert len(left) == lens[b] and all(p in left for p in [0, 1, *range(newest - 7, newest + 1)])
                held[b][j] = {p: s for p, s in held[b][j].items() if p in left}


@pytest.mark.parametrize("t", [1, 40])
def test_accounts_of_the_smallest_scale(t: int) -> None:
    """Every row as good as the next: 1 / n of a weight from each token and head, in the few rows' form and in the other."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(19)
    n, scale = 4096, 2.0**-120
    q = normal(gen, (1, 8, t, 64), "bf16").cuda()
    cache = Cache(gen, 1, 2, n, 64, "bf16", page=16)
    kw = dict(scale=scale, tokens=n, pages=cache.pages)
    lse = kernels.chunk_attend(q, cache.rows, **kw)[1]
    # Token t attends n - T + t + 1 rows. n u for the sum behind an lse of ln n (off by 16 u of 1 + ln n besides), 2 |lse| u of a weight, and the account's sum of 4 t of them.
    rows = torch.arange(n - t + 1, n + 1, device="cuda").double()
    assert torch.all((lse.double() - rows.log()).abs() <= (n + 16 * (1 + np.log(n))) * U)
    got = kernels.weigh_rows(q, lse, cache.rows, **kw).double()
    i = torch.arange(n, device="cuda")
    want = torch.where(i[:, None] <= n - t + torch.arange(t, device="cuda"), 1 / rows, 0.0).sum(-1) * 4
    assert torch.all((got - want).abs() <= (n + 18 * (1 + np.log(n)) + 4 * t + 8) * U * want)


@pytest.mark.parametrize(("t", "counts"), [(1, 1), (3, 3), (3, 2), (20, 20), (20, 17), (70, 70)])
@pytest.mark.parametrize(("model", "d", "eight"), [("bf16", 128, False), ("f16", 64, False), ("f16", 64, True)])
def test_tokens_that_add_nothing_and_lanes_without_one_show_no_key(t: int, counts: int, model: str, d: int, eight: bool) -> None:
    """A token whose lse is -inf adds nothing to a row whose key is not finite, nor does a lane that has no token; a score of -inf is a weight of 0."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(t)
    past = 300
    n = past + counts
    q = normal(gen, (1, 8, t, d), model).cuda()
    q[..., 0] = 1.0
    cache = Cache(gen, 1, 2, n, d, model, eight=eight, page=16)
    kw = dict(scale=0.1, lengths=int32([n]), counts=int32([counts]), max_tokens=n, pages=cache.pages)
    lse = kernels.chunk_attend(q, cache.rows, **kw)[1]
    lse[:, :, counts - 1] = -float("inf")
    want = kernels.weigh_rows(q, lse, cache.rows, **kw)
    assert want.isfinite().all() and torch.all(want[0, :, n - 1] == 0)
    where, i = cache.place(0, n - 1)
    if eight:  # NaN is the code 0x7f; there is no infinity
        cache.held[0][0, where, :, i, 3] = 0x7F
    else:
        cache.held[0][0, where, :, i, 3] = float("nan")
        where, i = cache.place(0, 5)
        cache.held[0][0, where, :, i, 0] = -float("inf")
        want[0, :, 5] = 0
    got = kernels.weigh_rows(q, lse, cache.rows, **kw)
    assert torch.equal(got, want), (got != want).nonzero()[:4]


def marked(n: int, d: int, *, seqs: int, h: int, eight: bool, page: int, gen: torch.Generator) -> tuple:
    """(rows, page table, what the rows hold as a function, their number): a cache in which sequence b's row i of head j is told by its first channels, b, j and i in small numbers, built
    without a step a row."""
    from lazykv_amd import kernels

    each = -(-n // page) if page else 1
    store = (seqs * each + 2, h, page, d) if page else (seqs, h, n, d)
    table = torch.randperm(store[0], generator=gen)[: seqs * each].view(seqs, each) if page else None
    at = torch.full((*store[:1], 1, store[2], 2), -1)
    place = torch.arange(n)
    for b in range(seqs):
        where, i = (table[b, place // page], place % page) if page else (torch.full_like(place, b), place)
        at[where, 0, i] = torch.stack([torch.full_like(place, b), place], -1)
    b, i = at.expand(-1, h, -1, -1).unbind(-1)
    j = torch.arange(h)[None, :, None].expand_as(b)
    marks = torch.stack([b + 1, j + 1, i % 128 + 1, i // 128 + 1], -1)  # 8-bit codes take them as bytes
    both = torch.zeros((2, *store), dtype=torch.uint8 if eight else torch.float16)
    both[..., :4], both[1, ..., 4] = marks.to(both.dtype), 9
    both = both.cuda()
    if eight:
        scales = torch.where(torch.arange(d // 32) == 0, 100, 7).to(torch.uint8).expand(2, *store[:3], d // 32).clone()
        scales[..., 0] += (i % 32).to(torch.uint8)
        held = [both, scales.cuda()]
        rows = kernels.mx_rows(*held, torch.float16)
    else:
        held, rows = [both], kernels.dense_rows(both[0], both[1])
    pages = None if table is None else table.int().cuda()

    def read(b: int, j: int) -> list:
        if table is None:
            return [x[:, b, j] for x in held]
        where, i = table[b, place // page].cuda(), (place % page).cuda()
        return [x[:, where, j, i] for x in held]

    return rows, pages, read, held


SPECIAL = (float("nan"), float("inf"), -float("inf"), -0.0, 0.0, 1e-42, -1.0, float("nan"))


def border_case(n: int, keep: int, *, sums_of: str, eight: bool = False, page: int = 0, d: int = 64, lens: list | None = None, apart: bool = False) -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(n + keep)
    seqs, h = len(lens or [n]), 2
    lens = lens or [n]
    rows, pages, read, held = marked(n, d, seqs=seqs, h=h, eight=eight, page=page, gen=gen)
    sums = torch.randn((seqs, h, n), generator=gen).exp()
    if sums_of == "ties":
        sums = torch.randint(0, 3, (seqs, h, n), generator=gen).float()
    elif sums_of == "special":
        for i, x in enumerate(SPECIAL):
            sums[:, :, i::11] = x
    elif sums_of == "nan":
        sums = torch.where(torch.rand((seqs, h, n), generator=gen) < 0.9, float("nan"), sums)
    positions = torch.stack([torch.randperm(n, generator=gen) for _ in range(seqs * h)]).view(seqs, h, n).int()
    args = [sums.cuda(), positions.cuda()]
    to = [torch.full_like(x, -3) for x in args] if apart else args
    before = [[[x.clone() for x in read(b, j)] for j in range(h)] for b in range(seqs)]
    kernels.evict_rows(rows, *args, keep=keep, sinks=min(2, keep), recent=min(5, max(0, keep - 2)), lengths=int32(lens), max_tokens=n, pages=pages, out=tuple(to) if apart else None)
    torch.cuda.synchronize()
    for b in range(seqs):
        for j in range(h):
            m = lens[b]
            s, p = sums[b, j].numpy().copy(), positions[b, j].numpy().copy()
            dst, src = O.evict(s[:m], p[:m], keep, min(2, keep), min(5, max(0, keep - 2))) if m else (np.zeros(0, np.int64),) * 2
            s[dst], p[dst] = s[src], p[src]
            to_rows, of_rows = torch.from_numpy(dst).cuda(), torch.from_numpy(src).cuda()
            for want, got in zip(before[b][j], read(b, j)):
                want[:, to_rows] = want[:, of_rows]
                assert torch.equal(got, want), (b, j)
            end = min(m, keep)
            left = slice(0, end if apart else n)
            assert np.array_equal(to[0][b, j].cpu().numpy()[left], s[left], equal_nan=True) and np.array_equal(to[1][b, j].cpu().numpy()[left], p[left]), (b, j)
            if apart:
                assert torch.all(to[0][b, j, end:] == -3) and torch.all(to[1][b, j, end:] == -3)


# Two, four, eight and sixteen rows a thread, and the first size by spans.
BORDERS = [2047, 2048, 2049, 4095, 4096, 4097, 8191, 8192, 8193, 16383, 16384, 16385]


@pytest.mark.parametrize("n", BORDERS)
@pytest.mark.parametrize("over", [1, 256, 257, 1500])
@pytest.mark.parametrize("sums_of", ["exp", "ties", "special"])
def test_both_sides_of_each_size(n: int, over: int, sums_of: str) -> None:
    """Rows over the budget: as many as the planning workgroup moves by itself, one more, and many."""
    border_case(n, n - over, sums_of=sums_of)


@pytest.mark.parametrize("n", [2049, 4097, 16384, 16385, 20001])
@pytest.mark.parametrize("keep", [1, 7, 200, 1024])
@pytest.mark.parametrize(("eight", "page", "d"), [(False, 16, 128), (True, 0, 64), (True, 48, 128)])
def test_few_rows_of_many_stay_in_pages_and_in_8_bits(n: int, keep: int, eight: bool, page: int, d: int) -> None:
    border_case(n, keep, sums_of="ties", eight=eight, page=page, d=d)


@pytest.mark.parametrize("n", [4096, 16384, 16385, 33000])
@pytest.mark.parametrize("sums_of", ["special", "nan", "ties"])
@pytest.mark.parametrize("share", [0.02, 0.3, 0.6, 0.97])
@pytest.mark.parametrize(("eight", "page"), [(False, 0), (True, 64)])
def test_special_sums_by_spans(n: int, sums_of: str, share: float, eight: bool, page: int) -> None:
    """NaN, which has the lowest rank of all, infinities, zeros of both signs and ties on both sides of row `keep`, in one workgroup and across spans."""
    border_case(n, max(1, int(n * share)), sums_of=sums_of, eight=eight, page=page)


@pytest.mark.parametrize(("n", "keep"), [(4097, 3000), (16384, 12000), (20001, 4096), (20001, 4095)])
@pytest.mark.parametrize("apart", [False, True])
def test_ragged_lengths_of_every_size(n: int, keep: int, apart: bool) -> None:
    """Sequences without rows, within the budget, one over it, at the last row of a span and one behind, and full."""
    border_case(n, keep, sums_of="ties", page=16, apart=apart, lens=[0, 1, keep - 1, keep, keep + 1, min(n, 4096 * (n // 4096)), min(n, 4096 * (n // 4096) + 1), n])
