"""Decode of a batch over a shared prefix and rows of each sequence's own, in the model dtype or in 8 bits, on the GPU against
attention in 64 bits.

How far a result may be off, from what is rounded on the way (u = 2^-24, float32's half step):
- a score sums d products in float32 and is scaled once, so it is off by at most (d + 4) u S, S the largest sum of a
  score's magnitudes; the exponential's argument (in base 2, of size up to S log2 e) and the exponential itself add 4 u S + 4 u: e in all,
  relative, of a weight;
- a weight is rounded to the model dtype for the product with the values: h = 2^-8 (bfloat16) or 2^-11 (float16) relative,
  and in float16, where a weight below 2^-14 has fewer bits, 2^-25 absolute;
- a sum over n tokens in float32 adds n u, and joining partial sums 8 u.
With A = sum p |v| of an output (at least its size) and V the values' largest magnitude, an output is off by at most
(2 e + h + 2 n u + 16 u) A + n 2^-25 V, plus its own rounding, h |out| (none in float32); the lse by e + n u + 16 u (1 + |lse|).
"""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import rows as O

pytestmark = pytest.mark.gpu

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
U = 2.0**-24


def _kv(gen: torch.Generator, shape: tuple, model: str) -> tuple[torch.Tensor, torch.Tensor]:
    loud = torch.where(torch.rand(shape[-1:], generator=gen) < 0.06, 5.0, 0.8)
    return (torch.randn(shape, generator=gen) * loud).to(TYPES[model]), torch.randn(shape, generator=gen).to(TYPES[model])


class Part:
    """Rows of `seqs` sequences with room behind them that holds NaN (codes and scales too), and their values in 64 bits."""

    def __init__(self, gen: torch.Generator, seqs: int, h: int, n: int, d: int, model: str, eight: bool, room: int = 3) -> None:
        from lazykv_amd import kernels

        kv = _kv(gen, (seqs, h, n, d), model)
        t = TYPES[model]
        if eight:
            coded = [O.mx_encode(x.double().numpy(), model) for x in kv]
            self.values = [O.mx_decode(*c) for c in coded]
            self.codes = torch.full((2, seqs, h, n + room, d), 0x7F, dtype=torch.uint8, device="cuda")
            self.scales = torch.full((2, seqs, h, n + room, d // 32), 0xFF, dtype=torch.uint8, device="cuda")
            for i, (c, s) in enumerate(coded):
                self.codes[i, :, :, :n] = torch.from_numpy(c).to(torch.float8_e4m3fn).view(torch.uint8).cuda()
                self.scales[i, :, :, :n] = torch.from_numpy(s).cuda()
            self.rows = kernels.mx_rows(self.codes, self.scales, t)
        else:
            self.values = [x.double().numpy() for x in kv]
            self.store = torch.full((2, seqs, h, n + room, d), float("nan"), dtype=t, device="cuda")
            for i, x in enumerate(kv):
                self.store[i, :, :, :n] = x.cuda()
            self.rows = kernels.dense_rows(self.store[0], self.store[1])

    def of(self, b: int, n: int) -> tuple[np.ndarray, np.ndarray]:
        return self.values[0][b, :, :n], self.values[1][b, :, :n]


def _check(got: tuple, q: torch.Tensor, prefix: tuple | None, own: list, scale: float) -> None:
    out, lse = got
    model_half = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
    half = model_half[q.dtype]
    out_half = {torch.float32: 0.0, **model_half}[out.dtype]
    b, n_q, d = q.shape
    want_o, want_l, a, s = O.shared_decode(q.double().cpu().numpy(), prefix, own, scale)
    o, l = out.double().cpu().numpy().reshape(want_o.shape), lse.double().cpu().numpy().reshape(want_l.shape)
    for i in range(b):
        n = own[i][0].shape[1] + (prefix[0].shape[1] if prefix is not None else 0)
        if n == 0:
            assert np.all(o[i] == 0) and np.all(np.isneginf(l[i]))
            continue
        big = max(np.abs(x).max(initial=0.0) for x in ([own[i][1]] + ([prefix[1]] if prefix is not None else [])))
        e = ((d + 8) * s[i] + 4) * U
        tol = (2 * e[:, None] + half + (2 * n + 16) * U) * a[i] + n * 2.0**-25 * big * (q.dtype == torch.float16) + out_half * np.abs(want_o[i])
        bad = ~(np.abs(o[i] - want_o[i]) <= tol)
        assert not bad.any(), (i, np.argwhere(bad)[:4], o[i][bad][:4], want_o[i][bad][:4], tol[bad][:4])
        tol_l = e + n * U + 16 * U * (1 + np.abs(want_l[i]))
        assert np.all(np.abs(l[i] - want_l[i]) <= tol_l), (i, np.abs(l[i] - want_l[i]).max(), tol_l.min())


def _case(seed: int, model: str, d: int, h: int, g: int, prefix: int, lens: list, prefix8: bool, own8: bool, out_dtype: torch.dtype | None = None,
          q_scale: float = 1.5, room: int = 3) -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(seed)
    seqs, most = len(lens), max(lens)
    q = (torch.randn((seqs, h * g, d), generator=gen) * q_scale).to(TYPES[model])
    p = Part(gen, 1, h, prefix, d, model, prefix8, room) if prefix else None
    o = Part(gen, seqs, h, most, d, model, own8, room) if most else None
    scale = d**-0.5
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda") if most else None
    got = kernels.shared_decode(q.cuda(), scale=scale, prefix=p.rows if p else None, prefix_tokens=prefix, own=o.rows if o else None, lengths=lengths,
                                max_own=most if o else None, out_dtype=out_dtype)
    torch.cuda.synchronize()
    none = np.zeros((h, 0, d))
    _check(got, q, p.of(0, prefix) if p else None, [o.of(b, n) if o else (none, none) for b, n in enumerate(lens)], scale)


@pytest.mark.parametrize("model", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("eight", [False, True])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 129, 255, 257, 1000, 4099])
def test_one_sequence_over_rows_of_its_own(model: str, d: int, eight: bool, n: int) -> None:
    _case(n, model, d, 2, 4, 0, [n], False, eight)


@pytest.mark.parametrize("model", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize(("prefix8", "own8"), [(False, False), (True, True), (True, False), (False, True)])
@pytest.mark.parametrize(("prefix", "lens"), [
    (1, [0]), (1, [1, 0]), (31, [3, 0, 33]), (32, [1] * 5), (33, [17, 2, 64, 65]), (128, [0] * 9), (300, [40, 1, 7, 128, 129]), (1021, [19, 5, 0, 18]),
])
def test_a_batch_over_a_prefix(model: str, d: int, prefix8: bool, own8: bool, prefix: int, lens: list) -> None:
    _case(prefix, model, d, 2, 4, prefix, lens, prefix8, own8)


@pytest.mark.parametrize("g", [1, 2, 3, 5, 7, 8, 16, 17, 40])
@pytest.mark.parametrize(("d", "eight"), [(64, False), (128, True)])
def test_groups_of_query_heads(g: int, d: int, eight: bool) -> None:
    _case(g, "bf16", d, 3, g, 150, [33, 0, 6], eight, eight)


@pytest.mark.parametrize("seqs", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17, 31, 33, 64, 70])
@pytest.mark.parametrize(("model", "d", "eight"), [("f16", 64, True), ("bf16", 128, False)])
def test_batches_of_every_width(seqs: int, model: str, d: int, eight: bool) -> None:
    """Rows of a KV head from 4 to 280: every number of row tiles, whole and not."""
    _case(seqs, model, d, 2, 4, 517, [(7 * i) % 20 for i in range(seqs)], eight, eight)


@pytest.mark.parametrize(("model", "d", "prefix8", "own8"), [("bf16", 128, False, False), ("f16", 64, True, True), ("bf16", 128, True, False)])
def test_a_long_prefix(model: str, d: int, prefix8: bool, own8: bool) -> None:
    _case(5, model, d, 1, 4, 20011, [300, 0, 299, 1, 64, 65, 128, 31, 7, 200, 11, 12], prefix8, own8)


@pytest.mark.parametrize("model", ["f16", "bf16"])
@pytest.mark.parametrize("out_dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_output_types(model: str, out_dtype: torch.dtype) -> None:
    _case(1, model, 128, 2, 4, 77, [5, 0, 40], False, False, out_dtype)


@pytest.mark.parametrize("q_scale", [0.0, 12.0])
def test_flat_and_peaked_scores(q_scale: float) -> None:
    """Weights all alike, and one token that outweighs the rest: a running maximum that rises late."""
    for model, d in (("f16", 64), ("bf16", 128)):
        _case(2, model, d, 2, 4, 700, [90, 0, 33], True, False, q_scale=q_scale)


def test_a_maximum_that_rises_with_every_token() -> None:
    """Scores that climb from -60 to 60 along the prefix and on through the own rows, and the same falling."""
    from lazykv_amd import kernels

    d, n, m = 64, 400, 100
    q = torch.zeros((2, 4, d), dtype=torch.bfloat16)
    q[..., 0] = 1.0
    gen = torch.Generator().manual_seed(3)
    for sign in (1.0, -1.0):
        ramp = torch.linspace(-60, 60, n + m).mul(sign)
        k = torch.zeros((2, 1, n + m, d))
        k[..., 0] = ramp
        k, v = k.bfloat16(), torch.randn((2, 1, n + m, d), generator=gen).bfloat16()
        pk, pv, ok, ov = (x.contiguous().cuda() for x in (k[:1, :, :n], v[:1, :, :n], k[:, :, n:], v[:, :, n:]))
        got = kernels.shared_decode(q.cuda(), scale=1.0, prefix=kernels.dense_rows(pk, pv), prefix_tokens=n, own=kernels.dense_rows(ok, ov), own_tokens=m)
        torch.cuda.synchronize()
        _check(got, q, (k[0, :, :n].double().numpy(), v[0, :, :n].double().numpy()),
               [(k[b, :, n:].double().numpy(), v[b, :, n:].double().numpy()) for b in range(2)], 1.0)


def test_lengths_are_limited_and_added_to() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(6)
    h, g, d, cap = 2, 4, 64, 50
    p, o = Part(gen, 1, h, 40, d, "f16", True), Part(gen, 5, h, cap, d, "f16", False)
    q = torch.randn((5, h * g, d), generator=gen).half()
    lengths = torch.tensor([0, -3, -2147483648, 40, 2147483647], dtype=torch.int32, device="cuda")
    got = kernels.shared_decode(q.cuda(), scale=0.125, prefix=p.rows, prefix_tokens=37, own=o.rows, own_tokens=7, lengths=lengths, max_own=45)
    torch.cuda.synchronize()
    _check(got, q, p.of(0, 37), [o.of(b, n) for b, n in enumerate([7, 4, 0, 45, 45])], 0.125)


@pytest.mark.parametrize("eight", [False, True])
def test_what_lies_behind_the_rows_is_not_seen(eight: bool) -> None:
    """NaN keys, values, codes and scales right behind a prefix and every sequence's rows, whose ends fall at every place of a
    tile of 32; and a NaN or an infinity among one sequence's rows stays with that sequence."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(7)
    h, g, d, seqs = 2, 2, 64, 34
    lens = list(range(seqs))
    o = Part(gen, seqs, h, seqs - 1, d, "bf16", eight, room=40)
    if eight:
        for b, n in enumerate(lens):
            o.codes[:, b, :, n:] = 0x7F
            o.scales[:, b, :, n:] = 0xFF
    else:
        for b, n in enumerate(lens):
            o.store[:, b, :, n:] = float("nan")
            o.store[1, b, :, n:, ::3] = float("inf")
    q = torch.randn((seqs, h * g, d), generator=gen).bfloat16()
    lengths = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for prefix in (0, 1, 29, 64):
        p = Part(gen, 1, h, max(prefix, 1), d, "bf16", eight, room=70)
        got = kernels.shared_decode(q.cuda(), scale=0.125, prefix=p.rows if prefix else None, prefix_tokens=prefix, own=o.rows, lengths=lengths, max_own=seqs - 1)
        torch.cuda.synchronize()
        _check(got, q, p.of(0, prefix) if prefix else None, [o.of(b, n) for b, n in enumerate(lens)], 0.125)
    clean = [x.clone() for x in got]
    if eight:
        o.codes[1, 20, :, 3] = 0x7F
    else:
        o.store[1, 20, :, 3] = float("inf")
    got = kernels.shared_decode(q.cuda(), scale=0.125, prefix=p.rows, prefix_tokens=64, own=o.rows, lengths=lengths, max_own=seqs - 1)
    torch.cuda.synchronize()
    assert bool((~got[0][20].isfinite()).all())
    keep = [b for b in range(seqs) if b != 20]
    assert torch.equal(got[0][keep], clean[0][keep]) and torch.equal(got[1], clean[1])


def test_infinite_values_that_are_attended_come_out_infinite() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(8)
    for n, at in ((33, 32), (20, 3), (64, 63)):
        o = Part(gen, 1, 2, n, 64, "f16", False)
        o.store[1, 0, :, at, 5] = float("inf")
        q = (torch.randn((1, 8, 64), generator=gen) * 0.1).half().cuda()
        out, lse = kernels.shared_decode(q, scale=0.125, own=o.rows, own_tokens=n)
        torch.cuda.synchronize()
        assert bool((out[:, :, 5] == float("inf")).all())
        rest = [c for c in range(64) if c != 5]
        assert bool(out[:, :, rest].isfinite().all()) and bool(lse.isfinite().all())


def test_large_scores_stay_finite() -> None:
    """Keys and queries as large as float16 allows: scores of +-1e9 and more, whose weights are zeros and ones."""
    from lazykv_amd import kernels

    d, n = 64, 70
    k = torch.full((1, 1, n, d), -3e4)
    k[:, :, 41] = 3e4
    v = torch.arange(n).float().view(1, 1, n, 1).expand(1, 1, n, d)
    q = torch.full((1, 4, d), 3e4).half().cuda()
    out, lse = kernels.shared_decode(q, scale=0.125, own=kernels.dense_rows(k.half().cuda(), v.half().contiguous().cuda()), own_tokens=n)
    torch.cuda.synchronize()
    assert bool((out == 41).all())
    want = 64 * float(torch.tensor(3e4).half()) ** 2 * 0.125
    assert bool(((lse.double() - want).abs() < want * 2.0**-20).all())


def test_queries_and_outputs_of_any_layout() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(9)
    h, g, d, seqs = 2, 3, 64, 4
    p, o = Part(gen, 1, h, 50, d, "f16", False), Part(gen, seqs, h, 20, d, "f16", True)
    q = torch.randn((seqs, h * g, d), generator=gen).half().cuda()
    call = dict(scale=0.125, prefix=p.rows, prefix_tokens=50, own=o.rows, own_tokens=20)
    want = kernels.shared_decode(q, **call)
    shapes = [q.unsqueeze(2), q.transpose(0, 1).contiguous().transpose(0, 1), torch.cat([q.new_zeros(5), q.flatten()])[5:].view(q.shape),
              torch.nn.functional.pad(q, (0, 7))[..., :d]]
    for x in shapes:
        got = kernels.shared_decode(x, **call)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    out, lse = torch.empty_like(want[0]), torch.empty_like(want[1])
    got = kernels.shared_decode(q, out=out, lse=lse, ws=kernels.Workspace("cuda"), **call)
    assert got[0] is out and got[1] is lse and torch.equal(out, want[0]) and torch.equal(lse, want[1])


def test_strided_rows() -> None:
    """A prefix that is one sequence's middle tokens in a larger cache, own rows that are every other sequence of one."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(10)
    h, g, d = 3, 4, 128
    for eight in (False, True):
        p, o = Part(gen, 3, h, 90, d, "bf16", eight), Part(gen, 6, h, 31, d, "bf16", eight)
        if eight:
            pr = kernels.mx_rows(p.codes[:, 1:2, :, 5:82], p.scales[:, 1:2, :, 5:82], torch.bfloat16)
            own = kernels.mx_rows(o.codes[:, ::2], o.scales[:, ::2], torch.bfloat16)
        else:
            pr = kernels.dense_rows(p.store[0, 1:2, :, 5:82], p.store[1, 1:2, :, 5:82])
            own = kernels.dense_rows(o.store[0, ::2], o.store[1, ::2])
        q = torch.randn((3, h * g, d), generator=gen).bfloat16()
        got = kernels.shared_decode(q.cuda(), scale=0.09, prefix=pr, prefix_tokens=77, own=own, own_tokens=31)
        torch.cuda.synchronize()
        _check(got, q, tuple(x[1, :, 5:82] for x in p.values), [o.of(2 * b, 31) for b in range(3)], 0.09)


def test_calls_repeat_to_the_bit_and_on_any_stream() -> None:
    """Two streams at once, each with calls of another size in between: no scratch is shared."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(11)
    parts = [(Part(gen, 1, 2, n, 128, "bf16", True), Part(gen, s, 2, 40, 128, "bf16", False), torch.randn((s, 8, 128), generator=gen).bfloat16().cuda())
             for n, s in ((3000, 5), (700, 21))]

    def call(i: int):  # noqa: ANN202
        p, o, q = parts[i]
        return kernels.shared_decode(q, scale=0.09, prefix=p.rows, prefix_tokens=p.rows.tokens - 3, own=o.rows, own_tokens=40)

    want = [call(0), call(1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, call(i)))
    torch.cuda.synchronize()
    for i, (out, lse) in got:
        assert torch.equal(out, want[i][0]) and torch.equal(lse, want[i][1])


def test_captured_calls_follow_lengths_and_inputs() -> None:
    """A step's write and attention in one graph, two graphs of different batches replayed in turn with eager calls between:
    each replay against the eager call, to the bit, and against 64 bits."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(12)
    h, g, d, cap = 2, 4, 64, 48
    made = []
    for seqs, eight in ((3, True), (6, False)):
        p = Part(gen, 1, h, 900, d, "f16", True)
        if eight:
            codes, scales = kernels.mx_empty(seqs, h, cap, d, "cuda")
            own = kernels.mx_rows(codes, scales, torch.float16)
        else:
            store = torch.zeros((2, seqs, h, cap, d), dtype=torch.float16, device="cuda")
            own = kernels.dense_rows(store[0], store[1])
        q, kv = torch.zeros((seqs, h * g, d), dtype=torch.float16, device="cuda"), torch.zeros((2, seqs, h, 1, d), dtype=torch.float16, device="cuda")
        lengths = torch.zeros(seqs, dtype=torch.int32, device="cuda")

        def step(own=own, q=q, kv=kv, lengths=lengths, p=p):  # noqa: ANN001, ANN202
            kernels.append_rows(own, kv[0], kv[1], starts=lengths)
            return kernels.shared_decode(q, scale=0.125, prefix=p.rows, prefix_tokens=900, own=own, own_tokens=1, lengths=lengths, max_own=cap)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        made.append((graph, got, step, q, kv, lengths, p, [[] for _ in range(seqs)], eight, seqs))
    for turn in range(5):
        for graph, got, step, q, kv, lengths, p, kept, eight, seqs in made:
            new = _kv(gen, (seqs, h, 1, d), "f16")
            kv.copy_(torch.stack(new))
            q.copy_(torch.randn(q.shape, generator=gen).half())
            lengths.fill_(turn)
            graph.replay()
            torch.cuda.synchronize()
            out, lse = (x.clone() for x in got)
            eager = step()
            torch.cuda.synchronize()
            assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1])
            for b in range(seqs):
                kept[b].append([O.mx_decode(*O.mx_encode(x[b].double().numpy(), "f16")) if eight else x[b].double().numpy() for x in new])
            own = [tuple(np.concatenate([t[i] for t in kept[b]], 1) for i in range(2)) for b in range(seqs)]
            _check((out, lse), q.cpu(), p.of(0, 900), own, 0.125)


def test_empty_batches_and_empty_calls() -> None:
    from lazykv_amd import kernels

    x = torch.zeros((0, 2, 5, 64), dtype=torch.float16, device="cuda")
    out, lse = kernels.shared_decode(x.new_zeros((0, 4, 64)), scale=1.0, own=kernels.dense_rows(x, x), own_tokens=5)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    y = torch.zeros((2, 2, 0, 64), dtype=torch.float16, device="cuda")
    out, lse = kernels.shared_decode(x.new_ones((2, 4, 64)), scale=1.0, own=kernels.dense_rows(y, y), own_tokens=0)
    torch.cuda.synchronize()
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


@pytest.mark.parametrize("bad", ["none", "dtype", "head_dim", "heads", "batch", "prefix_batch", "scale", "prefix_tokens", "own_tokens", "lengths", "lengths_only",
                                 "out", "lse", "mixed", "negative"])
def test_refusals(bad: str) -> None:
    from lazykv_amd import kernels

    x = torch.zeros((2, 2, 5, 64), dtype=torch.float16, device="cuda")
    q = torch.zeros((2, 4, 64), dtype=torch.float16, device="cuda")
    rows, one = kernels.dense_rows(x, x), kernels.dense_rows(x[:1], x[:1])
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    call = dict(scale=0.1, prefix=one, prefix_tokens=5, own=rows, own_tokens=5)
    change = {
        "none": dict(prefix=None, own=None), "scale": dict(scale=-1.0), "prefix_batch": dict(prefix=rows), "prefix_tokens": dict(prefix_tokens=6),
        "own_tokens": dict(own_tokens=6), "lengths": dict(lengths=lengths.long()), "lengths_only": dict(own=None, own_tokens=0, lengths=lengths),
        "out": dict(out=q.new_zeros((2, 4, 65))), "lse": dict(lse=q.new_zeros((2, 4))), "mixed": dict(prefix=kernels.dense_rows(x[:1].bfloat16(), x[:1].bfloat16())),
        "negative": dict(prefix_tokens=-1),
    }.get(bad, {})
    call.update(change)
    query = {"dtype": q.bfloat16(), "head_dim": q[..., :32], "heads": q[:, :3], "batch": q[:1]}.get(bad, q)
    with pytest.raises(ValueError):
        kernels.shared_decode(query, **call)


@pytest.mark.parametrize("seqs", [12, 20, 33, 75])
@pytest.mark.parametrize(("model", "d", "prefix8"), [("f16", 64, False), ("f16", 128, True), ("bf16", 64, True), ("bf16", 128, False)])
def test_prefixes_that_end_anywhere_in_a_stage(seqs: int, model: str, d: int, prefix8: bool) -> None:
    """Rows of a KV head of 36, 60, 99 and 225 over prefixes that end at every kind of place of a stage of 64 or 128 tokens and
    of the tiles in it, with NaN right behind the end, in parts of one stage and of several."""
    for prefix in (1, 31, 33, 63, 65, 95, 97, 127, 129, 191, 193, 255, 257, 319, 385, 1023):
        _case(prefix, model, d, 1, 3, prefix, [i % 3 for i in range(seqs)], prefix8, False)


@pytest.mark.parametrize("seqs", [3, 9, 20, 70])
def test_a_prefixs_last_values_may_be_infinite_and_what_lies_behind_is_zero(seqs: int) -> None:
    """An infinite value in a prefix's last row comes out infinite in its channel and nowhere else, whatever the tile's other
    tokens behind the end are."""
    from lazykv_amd import kernels

    gen = torch.Generator().manual_seed(13)
    for prefix in (40, 65, 200):
        p = Part(gen, 1, 2, prefix, 64, "f16", False, room=100)
        p.store[1, 0, :, prefix - 1, 7] = float("inf")
        q = (torch.randn((seqs, 8, 64), generator=gen) * 0.1).half().cuda()
        out, lse = kernels.shared_decode(q, scale=0.125, prefix=p.rows, prefix_tokens=prefix)
        torch.cuda.synchronize()
        assert bool((out[:, :, 7] == float("inf")).all())
        assert bool(out[:, :, [c for c in range(64) if c != 7]].isfinite().all()) and bool(lse.isfinite().all())


def _check64(got: tuple, q: torch.Tensor, parts: list, scale: float, n: int) -> None:
    """Against attention in 64 bits on the GPU, over lists of keys and values [h, t, d] taken piece by piece; bounds as above."""
    b, n_q, d = q.shape
    h = parts[0][0].shape[0]
    g = n_q // h
    x = q.double().view(b, h, g, d).transpose(0, 1).reshape(h, b * g, d)
    m = torch.full((h, b * g), float("-inf"), dtype=torch.float64, device="cuda")
    big_s, big_v = torch.zeros_like(m), 0.0
    for k, v in parts:
        kd = k.double().transpose(1, 2).contiguous()
        m = torch.maximum(m, (x @ kd).amax(-1) * scale)
        big_s = torch.maximum(big_s, (x.abs() @ kd.abs()).amax(-1) * scale)
        big_v = max(big_v, float(v.abs().max()))
    total, o, a = torch.zeros_like(m), torch.zeros((h, b * g, d), dtype=torch.float64, device="cuda"), torch.zeros((h, b * g, d), dtype=torch.float64, device="cuda")
    for k, v in parts:
        p = ((x @ k.double().transpose(1, 2).contiguous()) * scale - m.unsqueeze(-1)).exp()
        total += p.sum(-1)
        o += p @ v.double()
        a += p @ v.double().abs()
    o, a, lse = o / total.unsqueeze(-1), a / total.unsqueeze(-1), m + total.log()
    half = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}[q.dtype]
    e = ((d + 8) * big_s + 4) * U
    # The sums over n tokens: each lane's over its own, 32 times fewer at the least, and these joined.
    n = n / 32 + 64
    tol = (2 * e.unsqueeze(-1) + half + (2 * n + 16) * U) * a + n * 32 * 2.0**-25 * big_v * (q.dtype == torch.float16) / total.unsqueeze(-1) + half * o.abs()
    tol_l = e + n * U + 16 * U * (1 + lse.abs())
    back = lambda y: y.view(h, b, g, -1).transpose(0, 1).reshape(b, n_q, -1)  # noqa: E731
    assert bool(((got[0].double() - back(o)).abs() <= back(tol)).all())
    assert bool(((got[1].double() - back(lse).squeeze(-1)).abs() <= back(tol_l).squeeze(-1)).all())


@pytest.mark.parametrize(("seqs", "prefix", "h", "eight"), [(20, 140000, 4, True), (20, 140001, 4, False), (70, 70007, 4, False)])
def test_many_rows_over_a_long_prefix(seqs: int, prefix: int, h: int, eight: bool) -> None:
    """Prefixes long enough for two workgroups a CU, whose last part is short."""
    from lazykv_amd import kernels

    gen = torch.Generator(device="cuda").manual_seed(14)
    kv = [torch.randn((1, h, prefix, 64), device="cuda", generator=gen).bfloat16() for _ in range(2)]
    q = torch.randn((seqs, 4 * h, 64), device="cuda", generator=gen).bfloat16()
    if eight:
        codes, scales = kernels.mx_empty(1, h, prefix, 64, "cuda")
        rows = kernels.mx_rows(codes, scales, torch.bfloat16)
        kernels.append_rows(rows, *kv)
        kv = kernels.read_rows(rows, 0, prefix)
    else:
        rows = kernels.dense_rows(*kv)
    got = kernels.shared_decode(q, scale=0.125, prefix=rows, prefix_tokens=prefix)
    pieces = [tuple(x[0, :, i : i + 20000] for x in kv) for i in range(0, prefix, 20000)]
    _check64(got, q, pieces, 0.125, prefix)


def test_rows_past_32_bits_of_bytes() -> None:
    """Keys and values of 4.3 GB each: one sequence of four query heads, and twelve over the same rows as a prefix."""
    from lazykv_amd import kernels

    gen = torch.Generator(device="cuda").manual_seed(15)
    n = (1 << 25) + 77
    kv = torch.randn((2, 1, 1, n, 64), device="cuda", generator=gen, dtype=torch.bfloat16)
    rows = kernels.dense_rows(kv[0], kv[1])
    for seqs, as_prefix in ((1, False), (12, True)):
        q = (torch.randn((seqs, 4, 64), device="cuda", generator=gen) * 2).bfloat16()
        call = dict(prefix=rows, prefix_tokens=n) if as_prefix else dict(own=rows, own_tokens=n)
        got = kernels.shared_decode(q, scale=0.125, **call)
        pieces = [(kv[0, 0, :, i : i + (1 << 22)], kv[1, 0, :, i : i + (1 << 22)]) for i in range(0, n, 1 << 22)]
        _check64(got, q, pieces, 0.125, n)


def test_a_prefix_of_no_tokens_and_no_rows() -> None:
    from lazykv_amd import kernels

    x = torch.zeros((1, 2, 5, 64), dtype=torch.float16, device="cuda")
    out, lse = kernels.shared_decode(x.new_ones((3, 4, 64)), scale=1.0, prefix=kernels.dense_rows(x, x), prefix_tokens=0)
    torch.cuda.synchronize()
    assert bool((out == 0).all()) and bool((lse == -math.inf).all())


def test_a_nan_far_below_the_maximum_is_not_lost() -> None:
    """A NaN value whose weight is nothing beside another part's: it is attended, and shows, as in attention in 64 bits."""
    from lazykv_amd import kernels

    for seqs in (2, 10, 40):
        k = torch.zeros((1, 1, 4096, 64), device="cuda", dtype=torch.float16)
        k[:, :, 4000] = 60.0
        v = torch.ones_like(k)
        v[:, :, 17, 3] = float("nan")
        q = torch.ones((seqs, 4, 64), device="cuda", dtype=torch.float16)
        out, lse = kernels.shared_decode(q, scale=1.0, prefix=kernels.dense_rows(k, v), prefix_tokens=4096)
        torch.cuda.synchronize()
        assert bool(out[:, :, 3].isnan().all()) and bool((out[:, :, 4:] == 1).all()) and bool(lse.isfinite().all())


@pytest.mark.parametrize("name", ["prefix_tokens", "own_tokens", "max_own"])
@pytest.mark.parametrize("by", [1 << 31, 1 << 32, -(1 << 32)])
def test_counts_beyond_32_bits_are_refused(name: str, by: int) -> None:
    """2^32 more than a valid count is that count in 32 bits."""
    from lazykv_amd import kernels

    x = torch.zeros((2, 2, 5, 64), dtype=torch.float16, device="cuda")
    lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
    call = dict(scale=0.1, prefix=kernels.dense_rows(x[:1], x[:1]), prefix_tokens=5, own=kernels.dense_rows(x, x), own_tokens=5, max_own=5, lengths=lengths)
    call[name] += by
    with pytest.raises(ValueError):
        kernels.shared_decode(x.new_zeros((2, 4, 64)), **call)


def test_rows_that_sequences_share_are_read() -> None:
    """The same rows for every sequence, by a stride of 0: as copies of them."""
    from lazykv_amd import kernels

    gen = torch.Generator(device="cuda").manual_seed(5)
    kv = torch.randn((2, 1, 2, 77, 64), device="cuda", generator=gen).half()
    q = torch.randn((5, 4, 64), device="cuda", generator=gen).half()
    shared = kernels.dense_rows(kv[0].expand(5, 2, 77, 64), kv[1].expand(5, 2, 77, 64))
    copies = kernels.dense_rows(kv[0].repeat(5, 1, 1, 1), kv[1].repeat(5, 1, 1, 1))
    a, b = (kernels.shared_decode(q, scale=0.125, own=r, own_tokens=77) for r in (shared, copies))
    torch.cuda.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_an_output_in_the_querys_place() -> None:
    from lazykv_amd import kernels

    gen = torch.Generator(device="cuda").manual_seed(6)
    for n, seqs in ((100, 1), (3000, 2), (300, 40)):
        kv = torch.randn((2, 1, 2, n, 64), device="cuda", generator=gen).half()
        q = torch.randn((seqs, 8, 64), device="cuda", generator=gen).half()
        rows = kernels.dense_rows(kv[0], kv[1])
        call = dict(own=rows, own_tokens=n) if seqs == 1 else dict(prefix=rows, prefix_tokens=n)
        want, _ = kernels.shared_decode(q, scale=0.125, **call)
        got = q.clone()
        kernels.shared_decode(got, scale=0.125, out=got, **call)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
