"""A layer's forward over a bounded cache in 64 bits: new tokens normalised and rotated, a chunk of them attended, the weights that rows
get, and which rows an eviction leaves. numpy, from the definitions; nothing of the product is imported."""

from __future__ import annotations

import numpy as np


def rotate(x: np.ndarray, weight: np.ndarray | None, eps: float, cos: np.ndarray | None, sin: np.ndarray | None) -> np.ndarray:
    """x [..., T, d], weight [d], cos / sin [T, r]: normalised over the channels, the first r of them turned in pairs r / 2 apart."""
    y = x.astype(np.float64)
    if weight is not None:
        y = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps) * weight
    if cos is None or cos.shape[-1] == 0:
        return y
    half = cos.shape[-1] // 2
    z = y.copy()
    for i in range(half):
        a, b = y[..., i], y[..., i + half]
        z[..., i] = a * cos[:, i] - b * sin[:, i]
        z[..., i + half] = b * cos[:, i + half] + a * sin[:, i + half]
    return z


def scores(q: np.ndarray, k: np.ndarray, n: int, scale: float) -> np.ndarray:
    """q [T, d], k [len, d], the last n rows the chunk's own: [T, len], -inf where token t does not attend: it does rows 0 .. len - n + t, and none from
    token n on."""
    t, i = np.arange(q.shape[0])[:, None], np.arange(k.shape[0])[None]
    seen = (i <= k.shape[0] - n + t) & (t < n)
    with np.errstate(invalid="ignore"):
        return np.where(seen, q @ k.T * scale, -np.inf)


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, n: int, scale: float, there: np.ndarray | None = None) -> tuple[np.ndarray, ...]:
    """(out [T, d], lse [T], and for bounds on the error sum p |v| [T, d] and the largest scale * sum |q| |k| of a token [T]). there [len]: rows that can be
    attended."""
    s = scores(q, k, n, scale)
    if there is not None:
        s[:, ~there] = -np.inf
    m = s.max(-1, initial=-np.inf, keepdims=True)
    p = np.where(np.isneginf(s), 0.0, np.exp(s - np.where(np.isneginf(m), 0.0, m)))
    total = p.sum(-1, keepdims=True)
    some = total > 0
    w = p / np.where(some, total, 1.0)
    with np.errstate(divide="ignore"):
        lse = np.where(some, m + np.log(total), -np.inf)[:, 0]
    size = (np.abs(q) @ np.abs(k).T * scale).max(-1, initial=0.0)
    return w @ v, lse, w @ np.abs(v), size


def weigh(q: np.ndarray, k: np.ndarray, lse: np.ndarray, n: int, scale: float) -> np.ndarray:
    """q [g, T, d], k [len, d], lse [g, T]: each row's weights summed, [len]."""
    got = np.zeros(k.shape[0])
    for x, l in zip(q, lse):
        s = scores(x, k, n, scale)
        live = ~np.isneginf(l)
        got += np.where(np.isneginf(s[live]), 0.0, np.exp(s[live] - l[live, None])).sum(0)
    return got


def evict(sums: np.ndarray, positions: np.ndarray, keep: int, sinks: int, recent: int) -> tuple[np.ndarray, np.ndarray]:
    """One head's rows: (destinations, sources) of those that move."""
    n = len(sums)
    if n <= keep:
        return np.zeros(0, np.int64), np.zeros(0, np.int64)
    newest = int(positions.max())
    held = [int(p) < sinks or int(p) > newest - recent for p in positions]
    value = [0.0 if h or np.isnan(s) else -float(s) for h, s in zip(held, sums)]
    order = sorted(range(n), key=lambda i: (not held[i], bool(np.isnan(sums[i])) and not held[i], value[i], i))
    kept = sorted(order[:keep])
    at = set(kept)
    return np.array([i for i in range(keep) if i not in at], np.int64), np.array([i for i in kept if i >= keep], np.int64)
