"""Rows of dense caches in 64 bits: E4M3 codes under shared power-of-two scales, and decode attention of a
batch over a shared prefix and rows of each sequence's own. numpy, from the definitions; nothing of the
product is imported."""

from __future__ import annotations

import numpy as np

GROUP = 32
LARGEST = {"f16": 61440.0, "bf16": 1.875 * 2.0**127}  # the largest values of four significant bits


def e4m3_table() -> np.ndarray:
    """The value of each of the 256 codes: sign, 4 exponent bits (bias 7), 3 mantissa bits; 0x7f and 0xff are NaN."""
    got = np.empty(256)
    for code in range(256):
        sign, e, m = code >> 7, (code >> 3) & 15, code & 7
        value = np.nan if code & 0x7F == 0x7F else (m / 8.0 * 2.0**-6 if e == 0 else (1.0 + m / 8.0) * 2.0 ** (e - 7))
        got[code] = -value if sign else value
    return got


def round_e4m3(y: np.ndarray) -> np.ndarray:
    """The nearest E4M3 value, ties to the even mantissa. |y| <= 448."""
    _, e = np.frexp(y)
    step = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.rint(y / step) * step  # rint: ties to even


def mx_encode(x: np.ndarray, model: str) -> tuple[np.ndarray, np.ndarray]:
    """float64 [..., d] (values of the model dtype) -> the codes' values [..., d] and the scales' bytes [..., d / 32]."""
    f = x.reshape(*x.shape[:-1], -1, GROUP)
    fine = np.isfinite(f)
    top = LARGEST[model]
    f = np.where(fine, np.clip(f, -top, top), np.nan)
    most = np.where(fine, np.abs(f), 0.0).max(-1)
    exps = np.arange(0, 256)
    # The least exponent whose 448 covers the group.
    covers = most[..., None] <= 448.0 * np.ldexp(1.0, exps - 127)
    scale = covers.argmax(-1)
    codes = np.where(fine, round_e4m3(np.where(fine, f, 0.0) * np.ldexp(1.0, 127 - scale)[..., None]), np.nan)
    return codes.reshape(x.shape), scale.astype(np.uint8)


def mx_decode(codes: np.ndarray, scales: np.ndarray) -> np.ndarray:
    """Code values [..., d] and scale bytes [..., d / 32] -> what they stand for."""
    f = codes.reshape(*codes.shape[:-1], -1, GROUP)
    return (f * np.ldexp(1.0, scales.astype(np.int64) - 127)[..., None]).reshape(codes.shape)


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float) -> tuple[np.ndarray, float, np.ndarray, float]:
    """One query row [d] over keys and values [t, d]: out [d], lse, and for bounds on the error sum p |v| [d] and the largest
    scale * sum |q| |k|."""
    if k.shape[0] == 0:
        return np.zeros(q.shape[-1]), -np.inf, np.zeros(q.shape[-1]), 0.0
    s = k @ q * scale
    m = s.max()
    p = np.exp(s - m)
    total = p.sum()
    w = p / total
    return w @ v, float(m + np.log(total)), w @ np.abs(v), float((np.abs(k) @ np.abs(q)).max() * scale)


def shared_decode(q: np.ndarray, prefix: tuple | None, own: list, scale: float) -> tuple[np.ndarray, np.ndarray, np.ndarray, np.ndarray]:
    """q [B, n_q, d]; prefix (keys, values) [h, P, d] or None; own[b] (keys, values) [h, len, d]. Each of `attend`'s results,
    [B, n_q, ...]."""
    b, n_q, d = q.shape
    got = [np.zeros((b, n_q, d)), np.zeros((b, n_q)), np.zeros((b, n_q, d)), np.zeros((b, n_q))]
    for i in range(b):
        n_kv = own[i][0].shape[0]
        for j in range(n_q):
            h = j // (n_q // n_kv)
            k, v = (x[h] for x in own[i])
            if prefix is not None:
                k, v = np.concatenate([prefix[0][h], k]), np.concatenate([prefix[1][h], v])
            for to, x in zip(got, attend(q[i, j], k, v, scale)):
                to[i, j] = x
    return tuple(got)
