"""The 64-bit oracle of the 8-bit rows (CPU), and the refusals that the library makes before any launch."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import rows as O

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def _every(model: str) -> torch.Tensor:
    return torch.arange(65536, dtype=torch.int32).to(torch.uint16).view(TYPES[model])


def test_e4m3_rounding_is_torchs() -> None:
    """Every float16 value of at most 448 against torch's conversion, itself to nearest even."""
    x = _every("f16")
    x = x[x.abs() <= 448]
    want = x.to(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(O.round_e4m3(x.double().numpy()), want)
    table = O.e4m3_table()
    ours = torch.arange(256, dtype=torch.int32).to(torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(table, ours, equal_nan=True)


@pytest.mark.parametrize("model", ["f16", "bf16"])
def test_codes_cover_every_finite_value_and_read_back_as_model_values(model: str) -> None:
    """Groups led by a value that sets the scale: no code exceeds 448, the scale is the least that allows it, and what is read
    back is a finite value of the model dtype within half a step of four significant bits, 2^-4, of the value."""
    x = _every(model)
    x = x[x.isfinite()].double().numpy()
    x = x[: len(x) // GROUPED * GROUPED].reshape(-1, GROUPED)
    codes, scales = O.mx_encode(x, model)
    assert np.abs(codes).max() <= 448
    back = O.mx_decode(codes, scales)
    most = np.abs(x).max(-1)
    assert np.all((most <= 448 * np.ldexp(1.0, scales[:, 0].astype(int) - 127)) | (most > O.LARGEST[model]))
    assert np.all((most > 224 * np.ldexp(1.0, scales[:, 0].astype(int) - 127)) | (scales[:, 0] == 0))
    rounded = torch.from_numpy(back).to(TYPES[model])
    exact = np.abs(back) >= 2.0**-126 if model == "bf16" else np.ones(back.shape, bool)  # below, bfloat16 has fewer bits
    assert torch.isfinite(rounded).all()
    assert np.array_equal(rounded.double().numpy()[exact], back[exact])
    limited = np.clip(x, -O.LARGEST[model], O.LARGEST[model])
    floor = np.ldexp(1.0, scales.astype(int) - 127 - 10)  # half a step of the smallest codes
    assert np.all(np.abs(back - limited) <= np.maximum(np.abs(limited) * 2.0**-4, floor))


GROUPED = O.GROUP


def test_non_finite_values_are_held_as_nan_and_leave_the_scale() -> None:
    x = np.linspace(-3, 3, 64)
    codes, scales = O.mx_encode(np.r_[x][None], "f16")
    y = x.copy()
    y[[5, 40]] = [np.inf, np.nan]
    codes2, scales2 = O.mx_encode(y[None], "f16")
    assert np.array_equal(scales, scales2)
    assert np.isnan(codes2[0, [5, 40]]).all()
    keep = np.ones(64, bool)
    keep[[5, 40]] = False
    assert np.array_equal(codes[0, keep], codes2[0, keep])


# -- refusals, before any device is touched ----------------------------------------------------------


def _rows(**change):  # noqa: ANN003, ANN202
    from lazykv_amd import _lib

    have = dict(k=4096, v=8192, k_scale=64, v_scale=128, seq_stride=1 << 20, head_stride=1 << 16, tokens=100, seqs=2, dtype=_lib.MXFP8, deq_dtype=_lib.BF16)
    have.update(change)
    return _lib.KVRows(*(have[f[0]] for f in _lib.KVRows._fields_))


@pytest.mark.parametrize(("change", "call", "says"), [
    ({}, dict(head_dim=96), b"head_dim 96"),
    ({}, dict(dtype="f32"), b"dtype 2"),
    ({}, dict(n_seqs=3), b"rows of 2 sequences"),
    ({}, dict(tokens=101), b"exceed the 100"),
    ({}, dict(start=-1), b"exceed the 100"),
    ({}, dict(start=2147483647, tokens=5), b"exceed the 100"),
    ({}, dict(k=4098), b"16 bytes"),
    ({}, dict(strides=(1 << 20, 1 << 16, 132)), b"multiples of 8"),
    (dict(seq_stride=8), {}, b"multiples of 32"),
    (dict(k=4097), {}, b"16 bytes"),
    (dict(k_scale=None), {}, b"need their scales"),
    (dict(k_scale=65), {}, b"scales must start"),
    (dict(deq_dtype=0), {}, b"dtype 0"),
    (dict(dtype=3), {}, b"dtype 3"),
    (dict(v=None), {}, b"NULL"),
    (dict(tokens=1 << 31), {}, b"2147483648 tokens"),
])
@pytest.mark.parametrize("fn", ["append", "read"])
def test_rows_calls_refuse_bad_arguments(fn: str, change: dict, call: dict, says: bytes) -> None:
    from lazykv_amd import _lib

    lib = _lib.lib()
    have = dict(k=4096, v=4096, dtype="bf16", strides=(1 << 20, 1 << 16, 128), n_seqs=2, n_kv=8, head_dim=128, tokens=10, start=0)
    have.update(call)
    dt = {"f16": _lib.F16, "bf16": _lib.BF16, "f32": _lib.F32}[have["dtype"]]
    r = _rows(**change)
    if fn == "append":
        rc = lib.lkv_append_rows(0, ctypes.byref(r), have["k"], have["v"], dt, *have["strides"], have["n_seqs"], have["n_kv"], have["head_dim"],
                                 have["tokens"], None, have["start"])
    else:
        rc = lib.lkv_read_rows(0, ctypes.byref(r), have["n_seqs"], have["n_kv"], have["head_dim"], have["start"], have["tokens"], have["k"], have["v"],
                               dt, *have["strides"])
    assert rc == _lib.LKV_ERR_INVALID
    assert says in lib.lkv_last_error(), lib.lkv_last_error()


@pytest.mark.parametrize(("fn", "change", "call"), [
    ("append", dict(seq_stride=0), {}),
    ("append", dict(head_stride=0), {}),
    ("append", dict(v=4096), {}),
    ("read", {}, dict(v=4096)),
    ("read", {}, dict(strides=(0, 1 << 16, 128))),
    ("read", {}, dict(strides=(1 << 20, 0, 128))),
    ("read", {}, dict(strides=(1 << 20, 1 << 16, 0))),
])
def test_rows_that_are_written_must_be_distinct(fn: str, change: dict, call: dict) -> None:
    from lazykv_amd import _lib

    lib = _lib.lib()
    have = dict(k=4096, v=8192, strides=(1 << 20, 1 << 16, 128))
    have.update(call)
    r = _rows(**change)
    if fn == "append":
        rc = lib.lkv_append_rows(0, ctypes.byref(r), have["k"], have["v"], _lib.BF16, *have["strides"], 2, 8, 128, 10, None, 0)
    else:
        rc = lib.lkv_read_rows(0, ctypes.byref(r), 2, 8, 128, 0, 10, have["k"], have["v"], _lib.BF16, *have["strides"])
    assert rc == _lib.LKV_ERR_INVALID
    assert b"share an address" in lib.lkv_last_error()


@pytest.mark.parametrize(("desc", "prefix", "own", "more", "says"), [
    (dict(head_dim=80), {}, {}, {}, b"head_dim 80"),
    (dict(n_q=30), {}, {}, {}, b"30 query heads over 8"),
    (dict(scale=0.0), {}, {}, {}, b"scale 0"),
    (dict(scale=float("nan")), {}, {}, {}, b"scale"),
    (dict(scale=float("inf")), {}, {}, {}, b"scale inf"),
    (dict(prefix_tokens=-1), {}, {}, {}, b"bad extent"),
    (dict(prefix_tokens=101), {}, {}, {}, b"101 tokens over 100"),
    (dict(max_own=101), {}, {}, {}, b"101 own tokens over 100"),
    ({}, None, {}, {}, b"without rows"),
    ({}, {}, None, {}, b"without rows"),
    ({}, dict(seqs=2), {}, {}, b"not 1"),
    ({}, {}, dict(seqs=1), {}, b"not 2"),
    ({}, {}, {}, dict(ws_bytes=0), b"workspace"),
    ({}, {}, {}, dict(q_dtype=2), b"dtype 2"),
    ({}, {}, {}, dict(out_dtype=4), b"output dtype 4"),
    ({}, {}, {}, dict(q=24), b"16 bytes"),
    (dict(n_seqs=1 << 23), {}, {}, {}, b"query rows"),
])
def test_shared_decode_refuses_bad_arguments(desc: dict, prefix: dict | None, own: dict | None, more: dict, says: bytes) -> None:
    from lazykv_amd import _lib

    lib = _lib.lib()
    have = dict(n_seqs=2, n_q=32, n_kv=8, head_dim=128, scale=0.1, prefix_tokens=50, own_tokens=0, max_own=50)
    have.update(desc)
    d = _lib.SharedDesc(*(have[f[0]] for f in _lib.SharedDesc._fields_))
    p = ctypes.byref(_rows(**{"seqs": 1, **prefix})) if prefix is not None else None
    o = ctypes.byref(_rows(**own)) if own is not None else None
    a = dict(q=4096, q_dtype=_lib.BF16, out_dtype=_lib.BF16, ws_bytes=1 << 40)
    a.update(more)
    rc = lib.lkv_shared_decode(0, ctypes.byref(d), a["q"], a["q_dtype"], p, o, None, 4096, a["out_dtype"], 4096, 4096, a["ws_bytes"])
    assert rc == _lib.LKV_ERR_INVALID
    assert says in lib.lkv_last_error(), lib.lkv_last_error()


def test_a_scale_that_leaves_float32_in_base_2_is_refused() -> None:
    from lazykv_amd import _lib

    lib = _lib.lib()
    d = _lib.SharedDesc(1, 8, 8, 64, 3.0e38, 0, 0, 0)
    assert lib.lkv_shared_decode(0, ctypes.byref(d), 4096, _lib.F16, None, None, None, 4096, _lib.F16, 4096, None, 0) == _lib.LKV_ERR_INVALID
    assert b"scale" in lib.lkv_last_error()


def test_every_shape_has_a_division() -> None:
    """The division of the work and its scratch, on the host: any shape without an error, none for one part, and never more than
    the partial results of 600 parts a row."""
    from lazykv_amd import _lib

    lib = _lib.lib()
    for n_seqs in (0, 1, 3, 16, 65, 4096):
        for n_q, n_kv in ((1, 1), (32, 8), (40, 1), (128, 128)):
            for d in (64, 128):
                for prefix in (0, 1, 127, 128, 5000, 131072, 1 << 30):
                    for own in (0, 1, 256, 257, 513, 100000, 1 << 30):
                        desc = _lib.SharedDesc(n_seqs, n_q, n_kv, d, 0.1, prefix, 0, own)
                        got = lib.lkv_shared_decode_workspace_bytes(ctypes.byref(desc))
                        rows = n_seqs * n_q
                        if prefix == 0 and own * d <= 32768:
                            assert got == 0
                        if not (prefix == 1 << 30 or own == 1 << 30):
                            assert got <= rows * 600 * (d + 2) * 4 + 16, (n_seqs, n_q, n_kv, d, prefix, own, got)


def test_python_calls_refuse_cpu_tensors() -> None:
    from lazykv_amd import kernels

    x = torch.zeros((1, 2, 4, 64), dtype=torch.float16)
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.dense_rows(x, x)
    with pytest.raises(RuntimeError, match="GPU"):
        kernels.mx_rows(*kernels.mx_empty(1, 2, 4, 64, "cpu"), torch.float16)
