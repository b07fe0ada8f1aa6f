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
