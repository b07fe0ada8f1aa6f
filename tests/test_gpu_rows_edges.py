"""Calls over rows of dense caches at the edges of what their documentation allows, on the GPU. Tolerances of the batch decode are those
of test_gpu_shared_decode.py."""

from __future__ import annotations

import pytest

from test_gpu_shared_decode import _case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs", [9, 20, 33])
@pytest.mark.parametrize(("model", "d", "own8"), [("f16", 64, True), ("bf16", 128, False)])
def test_long_rows_behind_a_short_prefix(seqs: int, model: str, d: int, own8: bool) -> None:
    """Rows of a KV head of 36, 80 and 132, each sequence's own rows in several pieces, some of them empty."""
    _case(seqs, model, d, 1, 4, 70, [(997 * i) % 2600 for i in range(seqs)], False, own8)
