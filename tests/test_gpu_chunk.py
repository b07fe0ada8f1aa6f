"""A chunk of new tokens over a cache's rows, on the GPU against attention in 64 bits.

How far a result may be off is derived as for the batch decode (tests/test_gpu_shared_decode.py): with u = 2^-24, S the largest sum of a score's
magnitudes, e = ((d + 8) S + 4) u the error of a weight, h half a step of the model dtype, A = sum p |v| and V the largest value, an output is off by at most
(2 e + h + (2 n + 16) u) A + n 2^-25 V (float16 only) and its own rounding; the lse by e + n u + 16 u (1 + |lse|). Here the reference level is taken
off inside the exponent's one multiply-add, which its rounding at the size of the scores, S log2 e u, covers with the 8 S u that e has for it.
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from chunk_cases import HALF, TYPES, U, Cache, int32, normal
from oracle import chunk as O

pytestmark = pytest.mark.gpu


def check(got: tuple, q: torch.Tensor, cache: Cache, lens: list, counts: list, scale: float, there: np.ndarray | None = None) -> None:
    out, lse = (x.double().cpu().numpy() for x in got)
    half, out_half = HALF[q.dtype], HALF[got[0].dtype]
    seqs, n_q, t, d = q.shape
    g = n_q // cache.shape[1]
    qd = q.double().cpu().numpy()
    for b in range(seqs):
        n = lens[b]
        for j in range(n_q):
            k, v = (x[b, j // g, :n] for x in cache.values)
            seen = None if there is None else there[b, :n]
            want_o, want_l, a, s = O.attend(qd[b, j], k, v, counts[b], scale, seen)
            none = np.isneginf(want_l)
            assert np.all(out[b, j][none] == 0) and np.all(np.isneginf(lse[b, j][none])), (b, j)
            e = ((d + 8) * s + 4) * U
            big = np.abs(v).max(initial=0.0)
            tol = (2 * e[:, None] + half + (2 * n + 16) * U) * a + n * 2.0**-25 * big * (q.dtype == torch.float16) + out_half * np.abs(want_o)
            bad = ~(np.abs(out[b, j] - want_o) <= tol)
            assert not bad.any(), (b, j, np.argwhere(bad)[:4], out[b, j][bad][:4], want_o[bad][:4], tol[bad][:4])
            tol_l = e + n * U + 16 * U * (1 + np.abs(want_l, where=~none, out=np.zeros_like(want_l)))
            assert np.all(np.abs(lse[b, j][~none] - want_l[~none]) <= tol_l[~none]), (b, j)


def case(seed: int, model: str, d: int, h: int, g: int, t: int, lens: list, counts: list | None = None, *, eight: bool = False, page: int = 0,
         out_dtype: torch.dtype | None = None, q_scale: float = 1.5, strided: bool = True) -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(seed)
    seqs, most = len(lens), max(lens)
    q = (torch.randn((seqs, t, h * g, d), generator=gen) * q_scale).to(TYPES[model]).cuda().transpose(1, 2)
    q = q if strided else q.contiguous()
    cache = Cache(gen, seqs, h, most, d, model, eight=eight, page=page, room=3)
    got = kernels.chunk_attend(q, cache.rows, scale=d**-0.5, lengths=int32(lens), counts=None if counts is None else int32(counts), max_tokens=most, pages=cache.pages,
                               out_dtype=out_dtype)
    torch.cuda.synchronize()
    check(got, q, cache, lens, counts or [t] * seqs, d**-0.5)


@pytest.mark.parametrize("model", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize(("eight", "page"), [(False, 0), (False, 16), (True, 0), (True, 48)])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 33, 64, 127, 129, 300, 1037])
def test_single_tokens(model: str, d: int, eight: bool, page: int, n: int) -> None:
    case(n, model, d, 2, 4, 1, [n, max(1, n // 2)], eight=eight, page=page)


@pytest.mark.parametrize(("model", "d", "eight", "page"), [("bf16", 128, False, 16), ("f16", 64, False, 0), ("f16", 128, True, 64), ("bf16", 64, True, 16), ("bf16", 64, False, 32),
                                                           ("f16", 128, False, 80)])
@pytest.mark.parametrize(("t", "past"), [(2, 0), (3, 40), (7, 1), (8, 250), (9, 63), (16, 0), (31, 5), (33, 100), (64, 0), (65, 129), (130, 300)])
def test_chunks(model: str, d: int, eight: bool, page: int, t: int, past: int) -> None:
    case(t, model, d, 2, 4, t, [past + t, t], eight=eight, page=page)


@pytest.mark.parametrize("g", [1, 2, 3, 5, 7, 8, 16, 17, 40])
@pytest.mark.parametrize(("d", "eight", "page", "t"), [(64, False, 0, 1), (128, True, 16, 1), (128, False, 32, 5), (64, True, 0, 11)])
def test_groups_of_query_heads(g: int, d: int, eight: bool, page: int, t: int) -> None:
    case(g, "bf16", d, 3, g, t, [t + 70, t + 3], eight=eight, page=page)


@pytest.mark.parametrize(("model", "d", "eight", "page"), [("bf16", 128, False, 16), ("f16", 64, True, 0)])
@pytest.mark.parametrize(("t", "lens", "counts"), [
    (1, [0, 5, 200], [0, 1, 1]), (1, [3, 4], [0, 1]), (5, [9, 0, 5, 33], [5, 0, 1, 4]), (40, [90, 40, 7, 0, 300], [40, 1, 7, 0, 39]), (4, [2, 1], [4, 3]), (70, [30, 200], [70, 64]),
])
def test_ragged_batches_and_tokens_without_rows(model: str, d: int, eight: bool, page: int, t: int, lens: list, counts: list) -> None:
    """A sequence may have fewer tokens than the call, none, or fewer rows than tokens: the first of them attend nothing."""
    case(t, model, d, 2, 4, t, lens, counts, eight=eight, page=page)


@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize(("t", "past"), [(1, 600), (1, 40), (50, 900), (200, 0)])
def test_output_types_one_part_and_several(out_dtype: torch.dtype, t: int, past: int) -> None:
    case(t, "bf16", 128, 1, 4, t, [past + t], out_dtype=out_dtype, page=64, strided=False)


@pytest.mark.parametrize(("model", "d"), [("f16", 64), ("bf16", 128)])
@pytest.mark.parametrize(("t", "past"), [(1, 9000), (6, 5000), (40, 4500)])
def test_long_caches_in_many_parts(model: str, d: int, t: int, past: int) -> None:
    case(t, model, d, 1, 4, t, [past + t], page=16)


@pytest.mark.parametrize(("seqs", "h", "g", "t", "long", "short"), [
    (70, 1, 4, 1, 900, 300), (100, 3, 4, 1, 700, 400), (64, 8, 2, 1, 500, 40), (300, 1, 2, 1, 300, 80), (33, 1, 8, 3, 900, 200), (5, 4, 4, 70, 1500, 200), (8, 8, 4, 70, 900, 200),
    (3, 2, 16, 130, 700, 150), (2, 8, 4, 200, 900, 250),
])
@pytest.mark.parametrize("kind", ["alike", "any", "one long"])
def test_batches_of_lengths_alike_and_far_apart(seqs: int, h: int, g: int, t: int, long: int, short: int, kind: str) -> None:
    """However the rows are divided among parts, sequences of one part and of several."""
    gen = torch.Generator().manual_seed(seqs + t)
    lens = [long // 2] * seqs if kind == "alike" else torch.randint(0, long + 1, (seqs,), generator=gen).tolist() if kind == "any" else [short] * seqs
    lens[seqs // 2] = long if kind == "one long" else lens[seqs // 2]
    lens[-1] = long if kind == "any" else lens[-1]
    case(seqs, "bf16", 64, h, g, t, lens, [min(n, t) for n in lens])


def test_a_captured_batch_follows_lengths_from_alike_to_far_apart() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(13)
    q = normal(gen, (40, 8, 1, 64), "f16").cuda()
    cache = Cache(gen, 40, 4, 600, 64, "f16")
    lengths = int32([600] * 40)
    kw = dict(scale=0.1, lengths=lengths, max_tokens=600)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.chunk_attend(q, cache.rows, **kw)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = kernels.chunk_attend(q, cache.rows, **kw)
    for lens in ([600] + [1] * 39, [0] * 40, [300] * 40, list(range(40)), [600] * 40):
        lengths.copy_(int32(lens))
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        check((out, lse), q, cache, lens, [1] * 40, 0.1)


@pytest.mark.parametrize("q_scale", [0.0, 40.0])
@pytest.mark.parametrize("t", [1, 40])
def test_scores_that_are_alike_and_far_apart(q_scale: float, t: int) -> None:
    case(t, "bf16", 64, 2, 4, t, [t + 100], q_scale=q_scale)
    case(t, "f16", 128, 2, 4, t, [t + 100], q_scale=q_scale / 4, page=16)


@pytest.mark.parametrize(("model", "d", "page"), [("bf16", 128, 0), ("f16", 64, 16), ("f16", 128, 0), ("bf16", 64, 32)])
@pytest.mark.parametrize("t", [3, 7, 40, 100])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_what_a_token_does_not_attend_does_not_reach_it(model: str, d: int, page: int, t: int, what: float) -> None:
    """One token of the chunk has a value (a key) that is not finite: the tokens before it are as without it, those from it on show it."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(t)
    past, at = 21, t // 2
    q = normal(gen, (1, 8, t, d), model).cuda()
    cache = Cache(gen, 1, 2, past + t, d, model, page=page)
    kw = dict(scale=d**-0.5, tokens=past + t, pages=cache.pages)
    clean, lse = kernels.chunk_attend(q, cache.rows, **kw)
    where, i = cache.place(0, past + at)
    cache.held[0][1, where, 0, i, 5] = what
    out, lse2 = kernels.chunk_attend(q, cache.rows, **kw)
    assert torch.equal(out[:, 4:], clean[:, 4:]) and torch.equal(lse, lse2)
    assert torch.equal(out[:, :4, :at], clean[:, :4, :at])
    keep = [c for c in range(d) if c != 5]
    assert torch.equal(out[:, :4, at:, keep], clean[:, :4, at:, keep])
    shown = out[:, :4, at:, 5].float()
    assert torch.all(shown.isnan() if math.isnan(what) else shown == what)
    cache.held[0][1, where, 0, i, 5] = 0.5
    cache.held[0][0, where, 0, i, 5] = float("nan")
    out, lse2 = kernels.chunk_attend(q, cache.rows, **kw)
    assert torch.equal(out[:, :4, :at].isnan(), torch.zeros_like(out[:, :4, :at], dtype=torch.bool)) and torch.equal(lse2[:, :4, :at], lse[:, :4, :at])
    assert torch.all(out[:, :4, at:].isnan()) and torch.all(lse2[:, :4, at:].isnan())


@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("t", [1, 5, 40])
@pytest.mark.parametrize("bad", [-1, 1 << 30, -(1 << 31)])
def test_pages_that_a_pool_lacks_are_not_attended(eight: bool, t: int, bad: int) -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(5)
    n, page = 150, 16
    q = normal(gen, (2, 4, t, 128), "bf16").cuda()
    cache = Cache(gen, 2, 1, n, 128, "bf16", eight=eight, page=page)
    there = np.ones((2, n), bool)
    table = cache.pages.clone()
    for b, i in ((0, 0), (0, 3), (1, 4), (1, 9)):
        table[b, i] = bad if b else cache.rows.seqs
        there[b, i * page : (i + 1) * page] = False
    got = kernels.chunk_attend(q, cache.rows, scale=0.1, tokens=n, pages=table)
    check(got, q, cache, [n, n], [t, t], 0.1, there)
    out, lse = kernels.chunk_attend(q, cache.rows, scale=0.1, tokens=n, pages=torch.full_like(table, bad))
    assert torch.all(out == 0) and torch.all(lse == -math.inf)


@pytest.mark.parametrize("t", [1, 40])
def test_pages_that_sequences_share_and_repeat(t: int) -> None:
    """Two sequences with the same first pages, and one page twice in a table."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(6)
    n = 100
    q = normal(gen, (2, 4, t, 64), "f16").cuda()
    cache = Cache(gen, 2, 1, n, 64, "f16", page=16)
    cache.table[1, :3] = cache.table[0, :3]
    cache.table[1, 4] = cache.table[1, 3]
    cache.pages = cache.table.int().cuda()
    cache.values = cache.read()
    cache.values = [x[:, :, :n] for x in cache.values]
    lens = [n, n - 10]
    got = kernels.chunk_attend(q, cache.rows, scale=0.125, lengths=int32(lens), pages=cache.pages)
    check(got, q, cache, lens, [t, t], 0.125)


@pytest.mark.parametrize(("t", "n"), [(4, 40), (4, 3000), (60, 200), (60, 3000)])
def test_tokens_behind_a_count_show_nothing_of_their_queries(t: int, n: int) -> None:
    """Few rows and many, in one part and in several; under inference mode too."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(t + n)
    q = normal(gen, (2, 8, t, 64), "f16").cuda()
    cache = Cache(gen, 2, 2, n, 64, "f16", page=16)
    kw = dict(scale=0.1, lengths=int32([n, n]), counts=int32([t // 2, 0]), max_tokens=n, pages=cache.pages)
    want = kernels.chunk_attend(q, cache.rows, **kw)
    q[0, :, t // 2 :], q[1] = float("nan"), float("inf")
    with torch.inference_mode():
        out, lse = kernels.chunk_attend(q, cache.rows, **kw)
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
        assert torch.all(out[0, :, t // 2 :] == 0) and torch.all(out[1] == 0) and torch.all(lse[0, :, t // 2 :] == -math.inf) and torch.all(lse[1] == -math.inf)
        sums = kernels.weigh_rows(q, lse, cache.rows, **kw)
        assert sums.isfinite().all() and torch.all(sums[1] == 0)
        turned = kernels.rotate_append(cache.rows, q, *(normal(gen, (2, 2, t, 64), "f16").cuda() for _ in range(2)), starts=int32([0, n - t]), pages=cache.pages)
        assert turned.is_inference() and torch.equal(turned[0, :, : t // 2], q[0, :, : t // 2])


def test_queries_that_lie_past_32_bits() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(18)
    far = (1 << 31) + 64
    base, other = (torch.empty(far + 4096 * 8, dtype=torch.float16, device="cuda") for _ in range(2))
    cache = Cache(gen, 2, 2, 200, 64, "f16", page=16)
    for t in (2, 40):
        near = normal(gen, (2, 4, t, 64), "f16").cuda()
        q = base.as_strided((2, 4, t, 64), (far, 64 * t, 64, 1))
        q.copy_(near)
        kw = dict(scale=0.1, tokens=200, pages=cache.pages)
        got, want = (kernels.chunk_attend(x, cache.rows, **kw) for x in (q, near))
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        sums = [kernels.weigh_rows(x, want[1], cache.rows, **kw) for x in (q, near)]
        assert torch.equal(*sums)
        k = normal(gen, (2, 2, t, 64), "f16").cuda()
        out = other.as_strided((2, 4, t, 64), (far, 64 * t, 64, 1))
        assert torch.equal(kernels.rotate_append(cache.rows, q, k, k, start=0, pages=cache.pages, out=out), near)


def test_results_repeat_to_the_bit() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(8)
    q = normal(gen, (3, 8, 50, 128), "bf16").cuda()
    cache = Cache(gen, 3, 2, 400, 128, "bf16", page=32)
    kw = dict(scale=0.09, lengths=int32([400, 90, 222]), pages=cache.pages)
    a = kernels.chunk_attend(q, cache.rows, **kw)
    for _ in range(5):
        b = kernels.chunk_attend(q, cache.rows, **kw)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_a_captured_call_follows_lengths_counts_and_pages() -> None:
    """Replays between eager work, each compared with the eager call on what the device holds then."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(9)
    q = normal(gen, (2, 8, 6, 128), "bf16").cuda()
    cache = Cache(gen, 2, 2, 700, 128, "bf16", page=16)
    lengths, counts, pages = int32([700, 13]), int32([6, 2]), cache.pages.clone()
    kw = dict(scale=0.09, lengths=lengths, counts=counts, max_tokens=700, pages=pages)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.chunk_attend(q, cache.rows, **kw)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = kernels.chunk_attend(q, cache.rows, **kw)
    for i, (a, b, c, d) in enumerate([(700, 13, 6, 2), (5, 699, 5, 6), (0, 1, 0, 1), (350, 351, 6, 6)]):
        lengths.copy_(int32([a, b]))
        counts.copy_(int32([c, d]))
        pages.copy_(cache.pages.roll(i, 0) if i < 3 else cache.pages.flip(1))
        out.fill_(9.0)
        graph.replay()
        torch.cuda.synchronize()
        want = kernels.chunk_attend(q, cache.rows, **kw)
        for x, y in zip((out, lse), want):  # to the bit; the pages' order brings rows of nobody's, which hold NaN, before the end
            torch.testing.assert_close(x, y, rtol=0, atol=0, equal_nan=True)


def test_two_streams_at_once_and_a_workspace() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(10)
    q = normal(gen, (2, 8, 40, 64), "f16").cuda()
    caches = [Cache(gen, 2, 2, 900, 64, "f16", page=16) for _ in range(2)]
    want = [kernels.chunk_attend(q, c.rows, scale=0.1, tokens=900, pages=c.pages) for c in caches]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    spaces = [kernels.Workspace("cuda", 0), None]
    got = [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(kernels.chunk_attend(q, caches[i].rows, scale=0.1, tokens=900, pages=caches[i].pages, ws=spaces[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, want[i][0]) and torch.equal(b, want[i][1]) for a, b in got[i])


def test_rows_behind_32_bits_of_bytes_decide_the_result() -> None:
    """A pool of 5 GB: the only page that is attended lies at its end, and at its start there is something else."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(11)
    pool = torch.zeros((2, 10000, 8, 128, 128), dtype=torch.bfloat16, device="cuda")
    page = normal(gen, (2, 8, 128, 128), "bf16").cuda()
    pool[:, -1] = page
    rows = kernels.dense_rows(pool[0], pool[1])
    small = kernels.dense_rows(page[0][None], page[1][None])
    for t in (1, 3, 50):
        q = normal(gen, (1, 8, t, 128), "bf16").cuda()
        got = kernels.chunk_attend(q, rows, scale=0.1, tokens=120, pages=int32([[9999]]))
        want = kernels.chunk_attend(q, small, scale=0.1, tokens=120)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_long_cache_past_32_bits_of_bytes() -> None:
    """One sequence of 2.3 million rows of one head (a table of the same pages again and again): the chunk's own rows, at its end, have all the weight."""
    from lazykv_amd import kernels

    pool = torch.zeros((2, 3, 1, 16384, 128), dtype=torch.bfloat16, device="cuda")
    n = 140 * 16384 + 77
    table = torch.zeros((1, 141), dtype=torch.int32, device="cuda")
    table[0, 140] = 2
    pool[0, 2, 0, 76], pool[1, 2, 0, 76] = 4.0, 3.0
    rows = kernels.dense_rows(pool[0], pool[1])
    q = torch.full((1, 2, 1, 128), 1.0, dtype=torch.bfloat16, device="cuda")
    out, lse = kernels.chunk_attend(q, rows, scale=1.0, tokens=n, pages=table)
    assert torch.all(out == 3.0) and torch.all((lse - 512).abs() < 1e-3)
    dense = torch.zeros((2, 1, 1, (1 << 24) + 4096, 128), dtype=torch.bfloat16, device="cuda")
    dense[0, 0, 0, -1], dense[1, 0, 0, -1] = 4.0, 3.0
    out, lse = kernels.chunk_attend(q, kernels.dense_rows(dense[0], dense[1]), scale=1.0, tokens=dense.shape[3])
    assert torch.all(out == 3.0) and torch.all((lse - 512).abs() < 1e-3)


def test_what_is_refused() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(12)
    q = normal(gen, (2, 8, 3, 64), "f16").cuda()
    cache = Cache(gen, 2, 2, 50, 64, "f16", page=16)
    kw = dict(scale=0.1, pages=cache.pages)
    with pytest.raises(ValueError, match="does not match"):
        kernels.chunk_attend(q.bfloat16(), cache.rows, tokens=9, **kw)
    with pytest.raises(ValueError, match="does not match"):
        kernels.chunk_attend(q[:, :3], cache.rows, tokens=9, **kw)
    with pytest.raises(ValueError, match="rows of a sequence over"):
        kernels.chunk_attend(q, cache.rows, tokens=65, **kw)
    with pytest.raises(ValueError, match="sequences"):
        kernels.chunk_attend(q, cache.rows, scale=0.1, tokens=9)
    with pytest.raises(ValueError, match="pages must be"):
        kernels.chunk_attend(q, cache.rows, scale=0.1, tokens=9, pages=cache.pages.long())
    with pytest.raises(ValueError, match="lengths must be"):
        kernels.chunk_attend(q, cache.rows, lengths=torch.tensor([1, 2], device="cuda"), **kw)
    with pytest.raises(ValueError, match="exceed max_tokens"):
        kernels.chunk_attend(q, cache.rows, tokens=9, max_tokens=8, **kw)
    with pytest.raises(ValueError, match="scale"):
        kernels.chunk_attend(q, cache.rows, scale=-1.0, tokens=9, pages=cache.pages)
    with pytest.raises(ValueError, match="out must be"):
        kernels.chunk_attend(q, cache.rows, tokens=9, out=q.transpose(1, 2), **kw)
    with pytest.raises(ValueError, match="must not lie among"):
        kernels.chunk_attend(q, cache.rows, tokens=9, out=q, **kw)
    with pytest.raises(RuntimeError, match="no gradient"):
        kernels.chunk_attend(q.clone().requires_grad_(), cache.rows, tokens=9, **kw)
    out, lse = kernels.chunk_attend(q[:, :, :0], cache.rows, tokens=9, **kw)
    assert out.shape == (2, 8, 0, 64) and lse.shape == (2, 8, 0)
    out, lse = kernels.chunk_attend(q, cache.rows, **kw)
    assert torch.all(out == 0) and torch.all(lse == -math.inf)
