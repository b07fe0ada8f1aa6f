"""What the calls over rows of dense caches do on the host (CPU): the division of a call's work and its scratch, and checks that
come before any launch."""

from __future__ import annotations

import ctypes

import pytest


def _scratch(n_seqs: int, n_q: int, n_kv: int, d: int, prefix: int, own: int) -> int:
    from lazykv_amd import _lib

    desc = _lib.SharedDesc(n_seqs, n_q, n_kv, d, 0.1, prefix, 0, own)
    return _lib.lib().lkv_shared_decode_workspace_bytes(ctypes.byref(desc))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize(("n_q", "n_kv"), [(1, 1), (4, 1), (17, 1), (32, 8), (40, 1), (128, 128)])
def test_scratch_does_not_grow_with_the_rows_there_is_room_for(n_q: int, n_kv: int, d: int) -> None:
    """A part's row takes d sums, a maximum and a weight in float32. However many tokens: a prefix's parts are 513 at the most (a
    workgroup each on two a CU, and one that the rounding adds); the pieces of all own rows 1,024 (two for each of two workgroups a CU) and
    one a sequence, KV head and 16 query heads."""
    g_tiles = -(-(n_q // n_kv) // 16)
    for n_seqs in (1, 2, 3, 9, 16, 65, 4096):
        items = n_seqs * n_kv * g_tiles
        for prefix in (0, 1, 127, 1021, 32768, 131072, 1 << 30):
            for own in (0, 1, 257, 1024, 5000, 32768, 100000, 1 << 20, (1 << 30) - 1, 1 << 30):
                parts = 513 + 1024 // items + 1
                assert _scratch(n_seqs, n_q, n_kv, d, prefix, own) <= n_seqs * n_q * parts * (d + 2) * 4 + 16, (n_seqs, prefix, own)


@pytest.mark.parametrize(("prefix", "own"), [(0, 100000), (1, 100000), (1, 1 << 20), (1021, 32768), (32768, 1 << 30)])
def test_a_short_prefix_does_not_cut_long_rows_behind_it_into_small_parts(prefix: int, own: int) -> None:
    """64 sequences of 32 query heads over 8 KV heads: room for many tokens of their own costs a few MiB of scratch, with a prefix as
    without one."""
    assert _scratch(64, 32, 8, 128, prefix, own) <= 45 << 20
    if prefix <= 1021:
        assert _scratch(64, 32, 8, 128, prefix, own) <= 10 << 20


@pytest.mark.parametrize(("fn", "change", "call"), [
    ("append", dict(head_stride=32), {}),
    ("append", dict(head_stride=99 * 128), {}),
    ("append", dict(seq_stride=7 * (1 << 14) + 99 * 128), {}),
    ("append", dict(seq_stride=3 * (1 << 14)), {}),
    ("append", dict(head_stride=-99 * 128), {}),
    ("append", dict(v_off=128), {}),
    ("append", dict(v_off=-128), {}),
    ("append", dict(v_off=5 * (1 << 14)), {}),
    ("append", dict(v_scale_off=4), {}),
    ("append", dict(v_scale_off=-(1 << 9)), {}),
    ("read", {}, dict(v_off=256)),
    ("read", {}, dict(v_off=9 * 256)),
    ("read", {}, dict(strides=(1 << 20, 8, 128))),
    ("read", {}, dict(strides=(1 << 20, 1 << 16, 8))),
    ("read", {}, dict(strides=(128, 1 << 16, 128))),
    ("read", {}, dict(strides=(1 << 20, 1 << 16, 120))),
    ("read", {}, dict(strides=(1 << 16, 1 << 16, 128))),
])
def test_rows_that_overlap_are_not_written(fn: str, change: dict, call: dict) -> None:
    """Strides and addresses that are all different and none 0: a row's end in another's, a head's last rows another's first, values in
    the keys' place of another head."""
    from lazykv_amd import _lib

    lib = _lib.lib()
    at = dict(k=1 << 40, v_off=1 << 30, k_scale=1 << 42, v_scale_off=1 << 30, seq_stride=8 << 14, head_stride=1 << 14)
    at.update(change)
    r = _lib.KVRows(at["k"], at["k"] + at["v_off"], at["k_scale"], at["k_scale"] + at["v_scale_off"], at["seq_stride"], at["head_stride"], 100, 2, _lib.MXFP8,
                    _lib.BF16)
    have = dict(k=1 << 41, v_off=1 << 30, strides=(1 << 20, 1 << 16, 128))
    have.update(call)
    if fn == "append":
        rc = lib.lkv_append_rows(0, ctypes.byref(r), have["k"], have["k"] + have["v_off"], _lib.BF16, *have["strides"], 2, 8, 128, 10, None, 0)
    else:
        rc = lib.lkv_read_rows(0, ctypes.byref(r), 2, 8, 128, 0, 10, have["k"], have["k"] + have["v_off"], _lib.BF16, *have["strides"])
    assert rc == _lib.LKV_ERR_INVALID
    assert b"share an address" in lib.lkv_last_error()
