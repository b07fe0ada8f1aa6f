"""Calls over rows of dense caches at the edges of what their documentation allows, on the GPU. Tolerances of the batch decode are those
of test_gpu_shared_decode.py."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import rows as O
from test_gpu_shared_decode import _case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs", [9, 20, 33])
@pytest.mark.parametrize(("model", "d", "own8"), [("f16", 64, True), ("bf16", 128, False)])
def test_long_rows_behind_a_short_prefix(seqs: int, model: str, d: int, own8: bool) -> None:
    """Rows of a KV head of 36, 80 and 132, each sequence's own rows in several pieces, some of them empty."""
    _case(seqs, model, d, 1, 4, 70, [(997 * i) % 2600 for i in range(seqs)], False, own8)


def _no_copies(monkeypatch: pytest.MonkeyPatch) -> None:
    def copied(*args: object, **kwargs: object) -> None:
        raise AssertionError("a copy")

    monkeypatch.setattr(torch, "stack", copied)
    monkeypatch.setattr(torch.Tensor, "clone", copied)


@pytest.mark.parametrize("eight", [True, False])
@pytest.mark.parametrize(("seqs", "h"), [(1, 8), (16, 8), (1, 1), (3, 1)])
def test_a_tokens_keys_and_values_are_read_where_they_are(monkeypatch: pytest.MonkeyPatch, seqs: int, h: int, eight: bool) -> None:
    """A decode token's, as a model hands them over: rotated keys contiguous, values a projection's transposed view. They differ in the
    strides of dimensions of size 1 alone, which mean nothing."""
    from lazykv_amd import kernels

    d, cap = 64, 7
    gen = torch.Generator().manual_seed(seqs + h)
    k = torch.randn((seqs, h, 1, d), generator=gen).half().cuda()
    v = torch.randn((seqs, 1, h * d), generator=gen).half().cuda().view(seqs, 1, h, d).transpose(1, 2)
    odd = torch.as_strided(v, v.shape, tuple(s if n > 1 else 13 for n, s in zip(v.shape, v.stride())))
    assert h == 1 or k.stride() != v.stride()
    if eight:
        codes, scales = kernels.mx_empty(seqs, h, cap, d, "cuda")
        rows = kernels.mx_rows(codes, scales, torch.float16)
    else:
        store = torch.zeros((2, seqs, h, cap, d), dtype=torch.float16, device="cuda")
        rows = kernels.dense_rows(store[0], store[1])
    with monkeypatch.context() as m:
        _no_copies(m)
        kernels.append_rows(rows, k, v, start=2)
        kernels.append_rows(rows, k, odd, start=5)
    torch.cuda.synchronize()
    for which, x in enumerate((k, v)):
        if eight:
            c, s = O.mx_encode(x.double().cpu().numpy(), "f16")
            for t in (2, 5):
                assert np.array_equal(codes[which, :, :, t : t + 1].double().cpu().numpy(), c)
                assert np.array_equal(scales[which, :, :, t : t + 1].cpu().numpy(), s)
        else:
            assert all(torch.equal(store[which, :, :, t : t + 1], x) for t in (2, 5))


def test_rows_of_one_token_or_head_are_described_and_read_into() -> None:
    """A transposed view of one token is rows as it stands, and one is taken as an output, whatever its unused strides are."""
    from lazykv_amd import kernels

    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((2, 3, 1, 4 * 64), device="cuda", generator=gen).half().view(2, 3, 1, 4, 64).transpose(2, 3)  # [2, 3, 4, 1, 64]
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device).copy_(x)
    assert x.stride() != y.stride()
    q = torch.randn((3, 8, 64), device="cuda", generator=gen).half()
    a, b = (kernels.shared_decode(q, scale=0.1, own=kernels.dense_rows(t[0], t[1]), own_tokens=1) for t in (x, y))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    mixed = kernels.shared_decode(q, scale=0.1, own=kernels.dense_rows(x[0], y[1]), own_tokens=1)
    assert torch.equal(mixed[0], b[0])
    codes, scales = kernels.mx_empty(3, 4, 5, 64, "cuda")
    rows = kernels.mx_rows(codes, scales, torch.float16)
    kernels.append_rows(rows, y[0], y[1])
    want = kernels.read_rows(rows, 0, 1)
    out = (torch.empty(y[0].shape, dtype=y.dtype, device=y.device), torch.empty((3, 1, 4, 64), dtype=y.dtype, device=y.device).transpose(1, 2))
    assert out[0].stride() != out[1].stride()
    kernels.read_rows(rows, 0, 1, out=out)
    torch.cuda.synchronize()
    assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


@pytest.mark.parametrize(("seqs", "prefix"), [(1, False), (6, True), (12, True), (20, True)])
@pytest.mark.parametrize("eight", [False, True])
def test_rows_behind_32_bits_of_bytes_decide_the_result(seqs: int, prefix: bool, eight: bool) -> None:
    """The last 77 of 2^25 + 77 rows of 128 bytes lie behind 2^32 bytes, those of the second head behind 2^33. Their keys score 40, all
    others' 0 but the first 77's, which lie where a 32-bit offset would look for them and score -40: the others' share, 2^25 e^-40, is below
    2^-32, and the output is the last rows' value, 2. Its weights are alike, so rounded alike; products and sums of up to 77 such are exact, and what is
    left is the division's roundings and the output's: 2 (2^-22 + 2^-8) at most. lse: as in test_gpu_shared_decode.py, with n = 77, as the other
    rows' sum is nothing."""
    from lazykv_amd import kernels

    n, last, h, d = (1 << 25) + 77, 77, 2, 128 if eight else 64
    k, v = torch.zeros((1, h, last, d), dtype=torch.bfloat16, device="cuda"), torch.full((1, h, last, d), 2.0, dtype=torch.bfloat16, device="cuda")
    k[..., 0] = 40.0
    if eight:
        codes, scales = kernels.mx_empty(1, h, n, d, "cuda")
        rows = kernels.mx_rows(codes, scales, torch.bfloat16)
    else:
        store = torch.zeros((2, 1, h, n, d), dtype=torch.bfloat16, device="cuda")
        store[1] = 1.0
        rows = kernels.dense_rows(store[0], store[1])
    kernels.append_rows(rows, -k, -v)
    kernels.append_rows(rows, k, v, start=n - last)
    q = torch.zeros((seqs, 4 * h, d), dtype=torch.bfloat16, device="cuda")
    q[..., 0] = 1.0
    out, lse = kernels.shared_decode(q, scale=1.0, **(dict(prefix=rows, prefix_tokens=n) if prefix else dict(own=rows, own_tokens=n)))
    torch.cuda.synchronize()
    assert float((out.double() - 2.0).abs().max()) <= 2 * (2.0**-22 + 2.0**-8)
    want = 40.0 + np.log(77.0)
    assert float((lse.double() - want).abs().max()) <= (3 * 40 + 4 + 77 + 16 * (1 + want)) * 2.0**-24


def test_sequences_of_their_own_behind_32_bits_of_bytes() -> None:
    """The third sequence's rows begin behind 2^32 bytes and hold another value than the first's: each gets its own."""
    from lazykv_amd import kernels

    n = (1 << 24) + 5
    store = torch.zeros((2, 3, 1, n, 64), dtype=torch.bfloat16, device="cuda")
    for b in range(3):
        store[1, b] = 1.0 + b
    q = torch.ones((3, 4, 64), dtype=torch.bfloat16, device="cuda")
    lengths = torch.tensor([200, 3, 200], dtype=torch.int32, device="cuda")
    out, _ = kernels.shared_decode(q, scale=1.0, own=kernels.dense_rows(store[0], store[1]), lengths=lengths, max_own=200)
    torch.cuda.synchronize()
    for b in range(3):
        assert bool((out[b] == 1.0 + b).all())


def _overlap(shape: tuple, strides: tuple, apart: int, d: int) -> bool:
    """Whether any two of the rows of d elements at these strides, of keys and of values `apart` elements on, share an element."""
    at = np.zeros((), dtype=np.int64)
    for n, s in zip((2, *shape), (apart, *strides)):
        at = at[..., None] + np.arange(n) * s
    at = np.sort(at.ravel())
    return bool((np.diff(at) < d).any())


@pytest.mark.parametrize("seed", range(24))
def test_layouts_that_are_written_are_those_whose_rows_are_apart(seed: int) -> None:
    """Random strides of one buffer, which may interleave sequences, heads, keys and values or make them overlap: the write of a cache and the
    output of a read-back are taken where no two rows overlap, and then hold what they should, and refused otherwise."""
    from lazykv_amd import kernels

    rng = np.random.default_rng(seed)
    taken = refused = 0
    for _ in range(40):
        seqs, h, n, d = int(rng.integers(1, 4)), int(rng.integers(1, 4)), int(rng.integers(1, 6)), 64
        unit = n * d
        ss, hs, apart = (int(x) * unit + int(rng.choice([0, 0, 0, 32, d])) for x in rng.integers(0, 13, 3))
        buf = torch.zeros(400 * d, dtype=torch.float16, device="cuda")
        k = torch.randn((seqs, h, n, d), device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).half()
        dst = [buf.as_strided((seqs, h, n, d), (ss, hs, d, 1), off) for off in (0, apart)]
        bad = _overlap((seqs, h, n), (ss, hs, d), apart, d)
        if (seqs == 1 or ss % 32 == 0) and (h == 1 or hs % 32 == 0) and apart % 8 == 0:
            if bad:
                with pytest.raises(ValueError, match="share an address"):
                    kernels.append_rows(kernels.dense_rows(*dst), k, -k)
            else:
                kernels.append_rows(kernels.dense_rows(*dst), k, -k)
                torch.cuda.synchronize()
                assert torch.equal(dst[0], k) and torch.equal(dst[1], -k)
            taken, refused = taken + (not bad), refused + bad
        # The read-back's output, with a token stride of its own.
        ts = d * int(rng.integers(1, 4)) + int(rng.choice([0, 8]))
        codes, scales = kernels.mx_empty(seqs, h, n, d, "cuda")
        rows = kernels.mx_rows(codes, scales, torch.float16)
        kernels.append_rows(rows, k, -k)
        want = kernels.read_rows(rows, 0, n)
        out = [buf.zero_().as_strided((seqs, h, n, d), (ss, hs, ts, 1), off) for off in (0, apart)]
        bad = _overlap((seqs, h, n), (ss, hs, ts), apart, d)
        if bad:
            with pytest.raises(ValueError, match="share an address"):
                kernels.read_rows(rows, 0, n, out=tuple(out))
        else:
            kernels.read_rows(rows, 0, n, out=tuple(out))
            torch.cuda.synchronize()
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])
        taken, refused = taken + (not bad), refused + bad
    assert taken > 5 and refused > 5


@pytest.mark.parametrize("by", [1, -1, 8, 300])
def test_a_caches_own_rows_are_moved_within_it(by: int) -> None:
    """A block of rows to a place that overlaps it, keys and values swapped: what was read is what stood there before."""
    from lazykv_amd import kernels

    gen = torch.Generator(device="cuda").manual_seed(by + 2)
    store = torch.randn((2, 3, 4, 4000, 64), device="cuda", generator=gen).half()
    before = store.clone()
    rows = kernels.dense_rows(store[0], store[1])
    part = store[:, :, :, 500:3500]
    kernels.append_rows(rows, part[1], part[0], start=500 + by)
    torch.cuda.synchronize()
    want = before.clone()
    want[:, :, :, 500 + by : 3500 + by] = before[:, :, :, 500:3500].flip(0)
    assert torch.equal(store, want)
