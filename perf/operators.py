"""The 8-bit cache and the shared prefix: what their calls cost, at sizes that a decoding program meets.

A cache's rows are written as tokens arrive, as E4M3 codes with a power-of-two scale for every 32 channels of a row (`write`),
read back in the model's dtype for a forward of several tokens (`read`), and attended by one token of each sequence:
of one sequence over its own rows (`decode`), or of a batch whose sequences share a prefix that is stored
once and have rows of their own behind it (`shared`). `step` is a decode step's pair of calls: the new token's rows, then
the attention over them. Shapes are the 1B and 8B ones of the benchmark (32 query heads over 8 KV heads, head_dim 64 in
float16 or 128 in bfloat16) and, for drawn cases, sizes around them.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
GROUP = 32  # channels that share a scale
LARGEST = {torch.float16: 61440.0, torch.bfloat16: 1.875 * 2.0**127}  # the largest value of four significant bits


def _case(name: str, kind: str, dtype: str, d: int, *, h: int = 8, g: int = 4, seqs: int = 1, prefix: int = 0, rows: int = 0, ragged: bool = False,
          prefix8: bool = False, rows8: bool = True) -> dict:
    """prefix: tokens shared by all sequences; rows: tokens of its own that a sequence has (the most of them, where ragged), or
    that are written or read; prefix8 / rows8: held in 8 bits."""
    return {"name": name, "kind": kind, "dtype": dtype, "d": d, "h": h, "g": g, "seqs": seqs, "prefix": prefix, "rows": rows, "ragged": ragged,
            "prefix8": prefix8, "rows8": rows8}


def listed() -> list[dict]:
    return [
        # One decode step's token into one layer's 8-bit cache: the smallest call, all launch and latency.
        _case("write_token", "write", "bf16", 128, rows=1),
        # A 32K prompt's keys and values of one 1B-shaped layer, as a prefill hands them over.
        _case("write_32k", "write", "f16", 64, rows=32768),
        # A batch's questions behind a shared prefix, written at each sequence's own place.
        _case("write_batch", "write", "bf16", 128, seqs=24, rows=203, ragged=True),
        # What a turn's forward reads back of a chat of 4K tokens, and of a 128K context.
        _case("read_4k", "read", "f16", 64, rows=4099),
        _case("read_128k", "read", "bf16", 128, rows=131072),
        # One token over an 8-bit cache: a short chat, and a dense layer of the 128K context.
        _case("decode_4k", "decode", "f16", 64, rows=4099),
        _case("decode_128k", "decode", "bf16", 128, rows=131072),
        # Four samples of one short prompt, just begun: latency of a small batch.
        _case("shared_1k_4", "shared", "f16", 64, seqs=4, prefix=1021, rows=19, ragged=True, rows8=False),
        # Sixteen samples of a 32K prompt, a few hundred tokens on; one of them has none yet.
        _case("shared_32k_16", "shared", "bf16", 128, seqs=16, prefix=32768, rows=384, ragged=True, rows8=False),
        # Sixty-four samples of it: the batch where the matrix products weigh as much as the reads.
        _case("shared_32k_64", "shared", "bf16", 128, seqs=64, prefix=32768, rows=300, ragged=True, rows8=False),
        # A 128K document in 8 bits, thirty-two questions about it in 8 bits too.
        _case("shared_128k_32", "shared", "bf16", 128, seqs=32, prefix=131072, rows=700, ragged=True, prefix8=True),
        # A whole step of a 1B-shaped layer: each sequence's token written, then attended with the rest.
        _case("step_16k_8", "step", "f16", 64, seqs=8, prefix=16411, rows=257, prefix8=True),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("write", "read", "decode", "shared", "shared", "step"))
    dtype, d = rng.choice((("f16", 64), ("bf16", 128), ("bf16", 64), ("f16", 128)))
    h, g = rng.choice((1, 2, 4, 8, 8)), rng.choice((1, 2, 3, 4, 4, 5, 7, 8, 16))
    c = _case("", kind, dtype, d, h=h, g=g)
    del c["name"]
    budget = 131072 * 8 * 128 // (h * d)  # rows of the largest listed cache
    if kind in ("write", "read"):
        c["seqs"] = rng.choice((1, 1, _log(rng, 2, 64)))
        c["rows"] = _log(rng, 1, max(1, min(131072, budget // (2 * c["seqs"]))))
        c["ragged"] = kind == "write" and c["seqs"] > 1 and rng.random() < 0.5
        return c
    if kind == "decode":
        c["seqs"] = rng.choice((1, 1, _log(rng, 2, 32)))
        c["rows"] = _log(rng, 1, max(1, min(131072, budget // c["seqs"])))
        c["ragged"] = c["seqs"] > 1 and rng.random() < 0.5
        return c
    c["seqs"] = _log(rng, 2, 64)
    work = 131072 * 32 * 32 * 128 // (h * g * d * c["seqs"])  # tokens at the largest listed number of products
    c["prefix"] = _log(rng, 1, max(1, min(131072, budget // 2, work // 2)))
    c["rows"] = _log(rng, 1, max(1, min(2048, budget // (2 * c["seqs"]))))
    c["ragged"] = kind == "shared"
    c["prefix8"], c["rows8"] = rng.random() < 0.5, kind == "step" or rng.random() < 0.5
    return c


# -- inputs -----------------------------------------------------------------------------------------


def _gen(seed: int, salt: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed((seed * 1_000_003 + salt) % (1 << 62))


def _kv(case: dict, seed: int, salt: int, seqs: int, n: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values [seqs, h, n, d]: normal, with a few loud channels among the keys', as rotated keys have them."""
    gen, t = _gen(seed, salt), TYPES[case["dtype"]]
    shape = (seqs, case["h"], n, case["d"])
    loud = 0.4 + 0.8 * torch.rand((1, case["h"], 1, case["d"]), device=DEV, generator=gen)
    loud = torch.where(torch.rand(loud.shape, device=DEV, generator=gen) < 0.05, loud * 6.0, loud)
    keys = torch.randn(shape, device=DEV, generator=gen, dtype=t).mul_(loud.to(t))
    return keys, torch.randn(shape, device=DEV, generator=gen, dtype=t).mul_(0.7)


def _power(e: torch.Tensor) -> torch.Tensor:
    """2^e in 32 bits for whole -126 <= e <= 127, from its bits: torch's pow and ldexp may be a last place off."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """[..., d] -> codes (float8_e4m3fn, [..., d]) and scale exponents (uint8, [..., d / 32], biased by 127): the least power of
    two under which the group's largest magnitude is at most 448."""
    f = x.float().unflatten(-1, (-1, GROUP))
    fine = f.isfinite()
    f = torch.where(fine, f.clamp(-LARGEST[x.dtype], LARGEST[x.dtype]), float("nan"))
    most = torch.where(fine, f.abs(), 0.0).amax(-1)
    m, e = torch.frexp(most)  # most = m 2^e, 0.5 <= m < 1
    biased = torch.where(most > 0, e - 9 + 127 + (m > 0.875).int(), 0).clamp_min(0)
    codes = (f * _power(127 - biased).unsqueeze(-1)).to(torch.float8_e4m3fn)
    return codes.flatten(-2), biased.to(torch.uint8)


def _values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What codes and scales stand for, in 32 bits."""
    f = _power((scales.int() - 126).clamp_min(-126)) * torch.where(scales > 0, 0.5, 0.25).float()  # 2^(scale - 127), the least of them below the normal range
    return (codes.float().unflatten(-1, (-1, GROUP)) * f.unsqueeze(-1)).flatten(-2)


def _store(pair: tuple[torch.Tensor, torch.Tensor], eight: bool) -> dict:
    """A cache's rows as a program holds them: keys and values, or codes [2, seqs, h, n, d] and their scales."""
    if not eight:
        return {"keys": pair[0], "values": pair[1]}
    parts = [_quantise(x) for x in pair]
    return {"codes": torch.stack([c.view(torch.uint8) for c, _ in parts]).view(torch.float8_e4m3fn), "scales": torch.stack([s for _, s in parts])}


def _lengths(case: dict, seed: int) -> torch.Tensor:
    """Rows that each sequence has: up to `rows`, one sequence at the most and, in a batch of more than eight, one without any."""
    n, seqs = case["rows"], case["seqs"]
    if not case["ragged"]:
        return torch.full((seqs,), n, dtype=torch.int32, device=DEV)
    got = torch.randint(0, n + 1, (seqs,), device=DEV, generator=_gen(seed, 77), dtype=torch.int32)
    got[seqs // 2] = n
    if seqs > 8:
        got[seqs // 3] = 0
    return got


def prepare(case: dict, seed: int) -> dict:
    t, kind, seqs, n = TYPES[case["dtype"]], case["kind"], case["seqs"], case["rows"]
    h, d = case["h"], case["d"]
    state = {"case": case, "dtype": t}
    if kind == "write":
        # The cache has room ahead of and behind the rows: zeros there, which a call leaves as they are.
        state["new"] = _kv(case, seed, 1, seqs, n)
        room = n + 64
        state["codes"] = torch.zeros((2, seqs, h, room, d), dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
        state["scales"] = torch.zeros((2, seqs, h, room, d // GROUP), dtype=torch.uint8, device=DEV)
        state["starts"] = torch.randint(0, 64, (seqs,), device=DEV, generator=_gen(seed, 3), dtype=torch.int32) if case["ragged"] else None
        return state
    state["rows"] = _store(_kv(case, seed, 1, seqs, n), case["rows8"])
    if kind == "read":
        return state
    q = torch.randn((seqs, h * case["g"], d), device=DEV, generator=_gen(seed, 2))
    state["q"] = (q * 1.5).to(t)
    state["lengths"] = _lengths(case, seed)
    if case["prefix"]:
        state["prefix"] = _store(_kv(case, seed, 4, 1, case["prefix"]), case["prefix8"])
    if kind == "step":
        state["new"] = _kv(case, seed, 5, seqs, 1)
    return state


# -- one pass ---------------------------------------------------------------------------------------


def run(state: dict):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    if kind == "write":
        _write(state["codes"], state["scales"], state["new"], state["starts"])
        return {"codes": state["codes"], "scales": state["scales"]}
    if kind == "read":
        return list(_values(state["rows"]["codes"], state["rows"]["scales"]).to(state["dtype"]).unbind(0))
    if kind == "step":
        # The token that is the last of each sequence's rows.
        rows = state["rows"]
        last = state["case"]["rows"] - 1
        for i, x in enumerate(state["new"]):
            codes, scales = _quantise(x)
            rows["codes"].view(torch.uint8)[i, :, :, last : last + 1] = codes.view(torch.uint8)
            rows["scales"][i, :, :, last : last + 1] = scales
    return _attend(state)


def _write(codes: torch.Tensor, scales: torch.Tensor, new: tuple, starts: torch.Tensor | None) -> None:
    seqs, _, n, _ = new[0].shape
    raw = codes.view(torch.uint8)
    for i, x in enumerate(new):
        c, s = _quantise(x)
        if starts is None:
            raw[i, :, :, :n] = c.view(torch.uint8)
            scales[i, :, :, :n] = s
        else:
            at = starts.long()[:, None] + torch.arange(n, device=DEV)  # [seqs, n]
            b = torch.arange(seqs, device=DEV)[:, None]
            raw[i].transpose(1, 2)[b, at] = c.view(torch.uint8).transpose(1, 2)
            scales[i].transpose(1, 2)[b, at] = s.transpose(1, 2)


def _dense(store: dict) -> tuple[torch.Tensor, torch.Tensor]:
    if "codes" in store:
        k, v = _values(store["codes"], store["scales"]).unbind(0)
        return k, v
    return store["keys"].float(), store["values"].float()


def _attend(state: dict):
    """Softmax over the prefix's rows and each sequence's own, in 32 bits."""
    case = state["case"]
    h, g, seqs, d = case["h"], case["g"], case["seqs"], case["d"]
    q = state["q"].float().view(seqs, h, g, d) * d**-0.5
    k, v = _dense(state["rows"])  # [seqs, h, n, d]
    live = torch.arange(k.shape[2], device=DEV) < state["lengths"][:, None]
    s = (q @ k.transpose(-1, -2)).masked_fill(~live[:, None, None], float("-inf"))
    m = s.amax(-1)
    if case["prefix"]:
        pk, pv = (x[0] for x in _dense(state["prefix"]))  # [h, P, d]
        ps = (q.transpose(0, 1).reshape(h, seqs * g, d) @ pk.transpose(-1, -2)).view(h, seqs, g, -1)
        m = torch.maximum(m, ps.amax(-1).transpose(0, 1))
    m = m.clamp_min(torch.finfo(torch.float32).min)  # a sequence without any rows
    p = (s - m.unsqueeze(-1)).exp()
    total, out = p.sum(-1), p @ v
    if case["prefix"]:
        pp = (ps - m.transpose(0, 1).unsqueeze(-1)).exp()
        total = total + pp.sum(-1).transpose(0, 1)
        out = out + (pp.view(h, seqs * g, -1) @ pv).view(h, seqs, g, d).transpose(0, 1)
    out = torch.where(total.unsqueeze(-1) > 0, out / total.unsqueeze(-1), 0.0)
    return [out.reshape(seqs, h * g, d).to(state["dtype"]), (m + total.log()).reshape(seqs, h * g)]


def _run_own(state: dict):
    from lazykv_amd import kernels

    def rows(store: dict):
        if "codes" in store:
            return kernels.mx_rows(store["codes"], store["scales"], state["dtype"])
        return kernels.dense_rows(store["keys"], store["values"])

    case, kind = state["case"], state["case"]["kind"]
    if kind == "write":
        kernels.append_rows(kernels.mx_rows(state["codes"], state["scales"], state["dtype"]), *state["new"], starts=state["starts"])
        return {"codes": state["codes"], "scales": state["scales"]}
    if kind == "read":
        return list(kernels.read_rows(rows(state["rows"]), 0, case["rows"]))
    mine = rows(state["rows"])
    if kind == "step":
        kernels.append_rows(mine, *state["new"], start=case["rows"] - 1)
    return list(kernels.shared_decode(
        state["q"], scale=case["d"] ** -0.5, own=mine, lengths=state["lengths"], max_own=case["rows"],
        prefix=rows(state["prefix"]) if case["prefix"] else None, prefix_tokens=case["prefix"],
    ))


# -- what a pass cannot do without, and what it gives in 64 bits ------------------------------------


def work(case: dict) -> dict:
    h, g, d, seqs, n = case["h"], case["g"], case["d"], case["seqs"], case["rows"]
    eight, model = d + d // GROUP, 2 * d
    if case["kind"] in ("write", "read"):
        values = 2 * seqs * h * n
        return {"bytes": values * (eight + model), "flops": 0.0 if case["kind"] == "read" else 2.0 * values * d}
    live = n * (0.5 if case["ragged"] else 1.0) * seqs  # on average
    moved = 2 * h * (case["prefix"] * (eight if case["prefix8"] else model) + live * (eight if case["rows8"] else model))
    if case["kind"] == "step":
        moved += 2 * h * seqs * model  # the new token's rows read; written, they are among those counted
    moved += seqs * h * g * (4 * d + 4)
    return {"bytes": float(moved), "flops": 4.0 * h * g * d * (seqs * case["prefix"] + live)}


def _power64(e: torch.Tensor) -> torch.Tensor:
    return ((e.long() + 1023) << 52).view(torch.float64)


def _round_e4m3(y: torch.Tensor) -> torch.Tensor:
    """Float64 to the nearest E4M3 value, ties to even: steps of 2^(e - 3) from 2^-6 up, of 2^-9 below."""
    _, e = torch.frexp(y)
    step = _power64((e - 1).clamp_min(-6) - 3)
    return torch.round(y / step) * step


def _exact_codes(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes' values and scales' exponents of [..., d] in 64 bits: the exponent found by trying, not from the number's bits."""
    y = x.double().unflatten(-1, (-1, GROUP)).clamp(-LARGEST[x.dtype], LARGEST[x.dtype])
    most = y.abs().amax(-1)
    e = torch.ceil(torch.log2(most / 448.0)).clamp(-127, 127)
    e = torch.where(most > 448.0 * _power64(e), e + 1, e)
    e = torch.where(most <= 448.0 * _power64(e - 1), e - 1, e).clamp(-127, 127)
    e = torch.where(most > 0, e, -127.0)
    return _round_e4m3(y * _power64(-e).unsqueeze(-1)).flatten(-2), e


def _exact_dense(store: dict) -> tuple[torch.Tensor, torch.Tensor]:
    if "keys" in store:
        return store["keys"].double(), store["values"].double()
    f = _power64(store["scales"].long() - 127).repeat_interleave(GROUP, -1)
    v = store["codes"].double() * f
    return v[0], v[1]


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    kind = case["kind"]
    if kind == "write":
        codes, scales = state["codes"].double(), state["scales"].clone()
        seqs, _, n, _ = state["new"][0].shape
        at = state["starts"].tolist() if state["starts"] is not None else [0] * seqs
        for i, x in enumerate(state["new"]):
            c, e = _exact_codes(x)
            for b, a in enumerate(at):
                codes[i, b, :, a : a + n] = c[b]
                scales[i, b, :, a : a + n] = (e[b] + 127).to(torch.uint8)
        return {"codes": codes, "scales": scales}
    if kind == "read":
        return list(_exact_dense(state["rows"]))
    h, g, d, seqs, n = case["h"], case["g"], case["d"], case["seqs"], case["rows"]
    k, v = _exact_dense(state["rows"])
    if kind == "step":
        for x, to in zip(state["new"], (k, v)):
            c, e = _exact_codes(x)
            to[:, :, n - 1 : n] = c * _power64(e).repeat_interleave(GROUP, -1)
    pk, pv = (x[0] for x in _exact_dense(state["prefix"])) if case["prefix"] else (None, None)
    lengths = state["lengths"].tolist()
    out = torch.zeros((seqs, h, g, d), dtype=torch.float64, device=DEV)
    lse = torch.full((seqs, h, g), float("-inf"), dtype=torch.float64, device=DEV)
    q = state["q"].double().view(seqs, h, g, d)
    for b in range(seqs):
        for j in range(h):
            kk, vv = k[b, j, : lengths[b]], v[b, j, : lengths[b]]
            if pk is not None:
                kk, vv = torch.cat([pk[j], kk]), torch.cat([pv[j], vv])
            if kk.shape[0]:
                s = (q[b, j] @ kk.T) / math.sqrt(d)
                lse[b, j] = torch.logsumexp(s, -1)
                out[b, j] = torch.softmax(s, -1) @ vv
    return [out.view(seqs, h * g, d), lse.view(seqs, h * g)]
