"""Weights far below the largest one in the batch decode, on the GPU against attention in 64 bits.

One token's score lies `gap` above n equal ones, its value is 0 and theirs 1, so that the output is the small weights' sum alone:
n exp(-gap) / (1 + n exp(-gap)) = A. Scores are products of one factor of 1, so exact. With u = 2^-24: an exponential's argument, of size
up to 1.45 gap, and the exponential are off by (3 gap + 4) u relative of a weight, on both sides of the division; a weight's rounding is
h = 2^-11 (float16) or 2^-8 (bfloat16) relative and, in float16, where the largest weight is held at 2^13 or more and steps below 2^-14 are 2^-24,
2^-38 of the largest weight absolute (2^-25 / 2^13, half a step); float32 sums over n tokens add (2 n + 16) u. The output is read in float32:
    |error| <= (2 (3 gap + 4) u + h + (2 n + 16) u) A + n 2^-38,
which is less than a fiftieth of A at every gap here."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24


@pytest.mark.parametrize("gap", [9.75, 12.0, 17.375, 20.0, 22.0])
@pytest.mark.parametrize("model", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize(("seqs", "n", "own"), [(1, 200, True), (3, 1000, False), (7, 255, False), (12, 500, False), (40, 255, False), (300, 3000, True)])
def test_small_weights_beside_a_large_one_are_not_lost(seqs: int, n: int, own: bool, d: int, model: torch.dtype, gap: float) -> None:
    """Each form of the call, by the rows of a KV head (4, 12, 28, 48, 160) and own rows in one part."""
    from lazykv_amd import kernels

    half = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}[model]
    exact = float(torch.tensor(gap).to(model))
    for at in (0, n // 2, n):
        k, v = torch.zeros((1, 1, n + 1, d)), torch.ones((1, 1, n + 1, d))
        k[:, :, at, 3], v[:, :, at] = exact, 0.0
        q = torch.zeros((seqs, 4, d))
        q[..., 3] = 1.0
        k, v, q = (x.to(model).cuda() for x in (k, v, q))
        call = dict(own=kernels.dense_rows(k.expand(seqs, 1, n + 1, d), v.expand(seqs, 1, n + 1, d)), own_tokens=n + 1) if own else dict(
            prefix=kernels.dense_rows(k, v), prefix_tokens=n + 1)
        out, lse = kernels.shared_decode(q, scale=1.0, out_dtype=torch.float32, **call)
        torch.cuda.synchronize()
        small = n * math.exp(-exact)
        want = small / (1.0 + small)
        tol = (2 * (3 * exact + 4) * U + half + (2 * n + 16) * U) * want + (n * 2.0**-38 if model == torch.float16 else 0.0)
        assert tol < want / 50
        assert float((out.double() - want).abs().max()) <= tol, (at, float(out.min()), float(out.max()), want)
        lse_want = exact + math.log1p(small)
        assert float((lse.double() - lse_want).abs().max()) <= (3 * exact + 4 + n + 16 * (1 + lse_want)) * U
