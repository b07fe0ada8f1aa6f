"""The oracle of a layer's forward over a bounded cache (CPU): known answers and independent restatements."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import chunk as O


def test_a_rotation_by_quarter_turns_swaps_the_halves() -> None:
    x = np.arange(8.0).reshape(1, 8)
    zero, one = np.zeros((1, 8)), np.ones((1, 8))
    assert np.array_equal(O.rotate(x, None, 0.0, one, zero), x)
    assert np.array_equal(O.rotate(x, None, 0.0, zero, one), [[-4, -5, -6, -7, 0, 1, 2, 3]])
    assert np.array_equal(O.rotate(x, None, 0.0, zero[:, :4], one[:, :4]), [[-2, -3, 0, 1, 4, 5, 6, 7]])


def test_a_rotation_keeps_lengths_and_relative_angles() -> None:
    rng = np.random.default_rng(0)
    angle = np.tile(np.arange(3.0)[:, None] * [1.0, 0.1, 0.01], (1, 2))
    q, k = rng.normal(size=(2, 1, 6)).repeat(3, 1)
    a, b = (O.rotate(x, None, 0.0, np.cos(angle), np.sin(angle)) for x in (q, k))
    assert np.allclose((a * a).sum(-1), (q * q).sum(-1))
    assert np.allclose(a[1] @ b[0], a[2] @ b[1])


def test_the_norm_is_the_root_mean_square() -> None:
    x = np.array([[3.0, 4.0, 0.0, 0.0]])
    assert np.allclose(O.rotate(x, np.array([1.0, 2.0, 1.0, 1.0]), 0.0, None, None), [[1.2, 3.2, 0.0, 0.0]])


@pytest.mark.parametrize(("length", "n", "t"), [(9, 4, 4), (9, 2, 4), (3, 3, 3), (2, 4, 4), (0, 0, 3), (5, 0, 2)])
def test_attention_is_torchs_with_the_mask_written_out(length: int, n: int, t: int) -> None:
    rng = np.random.default_rng(length)
    q, k, v = rng.normal(size=(t, 8)), rng.normal(size=(length, 8)), rng.normal(size=(length, 8))
    out, lse, _, _ = O.attend(q, k, v, n, 0.3)
    for i in range(t):
        seen = length - n + i + 1 if i < n else 0
        if seen <= 0:
            assert np.all(out[i] == 0) and np.isneginf(lse[i])
            continue
        s = torch.from_numpy(q[i] @ k[:seen].T * 0.3)
        assert np.allclose(out[i], (torch.softmax(s, -1) @ torch.from_numpy(v[:seen])).numpy())
        assert np.isclose(lse[i], torch.logsumexp(s, -1).item())


def test_a_tokens_weights_sum_to_one() -> None:
    rng = np.random.default_rng(3)
    q, k = rng.normal(size=(2, 5, 8)), rng.normal(size=(11, 8))
    lse = np.stack([O.attend(x, k, k, 4, 0.5)[1] for x in q])
    got = O.weigh(q, k, lse, 4, 0.5)
    assert np.isclose(got.sum(), 2 * 4)  # two heads, four tokens; the fifth attends nothing
    one = O.weigh(q[:1, :1], k, lse[:1, :1], 1, 0.5)
    assert one[-1] > 0 and not np.isclose(one.sum(), 1.0)  # as the last token it attends rows that its own lse does not count


def test_eviction_by_hand() -> None:
    sums = np.array([1.0, 9.0, 2.0, 8.0, 2.0, 7.0, np.nan, 0.0])
    at = np.arange(8)
    to, of = O.evict(sums, at, 4, 0, 0)
    assert to.tolist() == [0] and of.tolist() == [5]  # 9, 8, 7 and the first 2 stay
    to, of = O.evict(sums, at, 4, 1, 2)
    assert to.tolist() == [2, 3] and of.tolist() == [6, 7]  # the first token, the newest two, and 9
    to, of = O.evict(sums, at[::-1].copy(), 4, 1, 2)
    assert to.tolist() == [2] and of.tolist() == [7]  # row 7 holds the first token, rows 1 and 0 the newest; of the rest 8 is the largest
    assert O.evict(sums, at, 8, 0, 0)[0].size == 0
