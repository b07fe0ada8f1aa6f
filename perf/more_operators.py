"""A layer's forward over a bounded, paged cache: what its calls cost, at sizes that a serving program meets.

New tokens' queries and keys are normalised a head at a time and rotated, and keys and values written to their rows (`rotate`); a chunk of new
tokens of each sequence attends the rows before and among it (`attend`), one token of each being a decode step; the weights
that rows get are summed up (`weigh`); and where a cache has more rows than it may keep, those with the largest sums stay
(`evict`). Rows lie in pages of a pool or one after the other, in the model's dtype or as E4M3 codes with a power-of-two scale for every
32 channels. Shapes are the 1B and 8B ones of the benchmark (32 query heads over 8 KV heads, head_dim 64 in float16 or 128 in
bfloat16) and, for drawn cases, sizes around them.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}
GROUP = 32  # channels that share a scale
LARGEST = {torch.float16: 61440.0, torch.bfloat16: 1.875 * 2.0**127}  # the largest value of four significant bits
EPS = 1e-6


def _case(name: str, kind: str, dtype: str, d: int, *, h: int = 8, g: int = 4, seqs: int = 1, new: int = 1, past: int = 0, ragged: bool = False,
          page: int = 0, eight: bool = False, norm: bool = False, rot: int = 0, keep: int = 0, sinks: int = 0, recent: int = 0) -> dict:
    """new: tokens of a sequence in the call; past: rows that it has before them (the most of each, where ragged); page: tokens of a page, 0 for rows that
    lie one after the other; eight: rows in 8 bits; norm: queries and keys are normalised; rot: channels that turn; keep, sinks, recent:
    rows that an eviction leaves, and of them the first and the newest tokens that stay whatever their sums."""
    return {"name": name, "kind": kind, "dtype": dtype, "d": d, "h": h, "g": g, "seqs": seqs, "new": new, "past": past, "ragged": ragged, "page": page,
            "eight": eight, "norm": norm, "rot": rot, "keep": keep, "sinks": sinks, "recent": recent}


def listed() -> list[dict]:
    return [
        # One decode step's token of one sequence: the smallest call, all launch and latency.
        _case("rotate_token", "rotate", "bf16", 128, past=4099, page=16, norm=True, rot=128),
        # A chunk of an 8B-shaped prefill into pages.
        _case("rotate_chunk", "rotate", "bf16", 128, new=4099, past=8192, page=64, norm=True, rot=128),
        # A batch's questions, without norms, each at its own place of an 8-bit cache, and read back for their forward.
        _case("rotate_batch_8bit", "rotate", "f16", 64, seqs=24, new=203, past=61, ragged=True, eight=True, rot=64),
        # A decode step of sixteen sequences of a serving batch, of very different lengths.
        _case("attend_decode_16", "attend", "bf16", 128, seqs=16, past=8191, ragged=True, page=16),
        # A user's turn behind a 32K context.
        _case("attend_turn", "attend", "bf16", 128, new=203, past=32768, page=64),
        # A prompt from nothing, of a 1B-shaped layer.
        _case("attend_prompt", "attend", "f16", 64, new=4099),
        # A chunk of a long prefill: the largest call, bound by its products.
        _case("attend_chunk_32k", "attend", "bf16", 128, new=2048, past=32768, page=64),
        # Short questions of four sequences over 8-bit documents.
        _case("attend_questions_8bit", "attend", "bf16", 128, seqs=4, new=64, past=16411, ragged=True, page=128, eight=True),
        # What one decode token adds to the sums of a chat of 4K tokens.
        _case("weigh_token", "weigh", "f16", 64, past=4098, page=16),
        # What a chunk of a prefill adds to them.
        _case("weigh_chunk", "weigh", "bf16", 128, new=1024, past=15360, page=64),
        # A decode step of sixteen sequences, each one row over its budget.
        _case("evict_step", "evict", "bf16", 128, seqs=16, past=2049, page=16, keep=2048, sinks=4, recent=256),
        # A 128K prompt cut to a quarter.
        _case("evict_128k", "evict", "bf16", 128, past=131072, keep=32768, page=64, sinks=4, recent=4096),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng: random.Random) -> dict:
    kind = rng.choice(("rotate", "attend", "attend", "weigh", "evict"))
    dtype, d = rng.choice((("f16", 64), ("bf16", 128), ("bf16", 64), ("f16", 128)))
    c = _case("", kind, dtype, d, h=rng.choice((1, 2, 4, 8, 8)), g=rng.choice((1, 2, 3, 4, 4, 5, 7, 8, 16)), page=rng.choice((0, 16, 32, 48, 64, 128, 256)),
              eight=rng.random() < 0.3)
    del c["name"]
    c["seqs"] = rng.choice((1, 1, _log(rng, 2, 32)))
    c["ragged"] = c["seqs"] > 1 and rng.random() < 0.7
    budget = 131072 * 8 * 128 // (c["h"] * d * c["seqs"])  # rows of the largest listed cache
    if kind == "evict":
        c["past"] = _log(rng, 17, max(17, min(131072, budget)))
        c["keep"] = _log(rng, 1, c["past"])
        c["recent"] = rng.randrange(0, c["keep"] // 2 + 1)
        c["sinks"] = min(rng.choice((0, 1, 4)), c["keep"] - c["recent"])
        return c
    if kind == "rotate":
        c["new"] = _log(rng, 1, max(1, min(4099, 4099 * 8 * 6 * 128 // (c["seqs"] * c["h"] * (c["g"] + 2) * d))))
        c["past"] = rng.randrange(0, max(1, min(16384, budget // 8)))
        c["norm"] = rng.random() < 0.5
        c["rot"] = rng.choice((d, d, d, d // 2, d // 4 * 3, 16))
        return c
    c["new"] = rng.choice((1, _log(rng, 1, 64), _log(rng, 1, 2048)))
    heads = c["seqs"] * c["h"] * c["g"]
    c["new"] = min(c["new"], math.isqrt((1 << 30) // heads))  # scores: half of the largest listed case's at the most
    c["past"] = _log(rng, 1, max(1, min(65536, budget // 2, (1 << 30) // (heads * c["new"]) - c["new"])))
    return c


# -- inputs -----------------------------------------------------------------------------------------


def _gen(seed: int, salt: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed((seed * 1_000_003 + salt) % (1 << 62))


def _kv(shape: tuple, t: torch.dtype, seed: int, salt: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values [.., h, n, d]: normal, with a few loud channels among the keys', as rotated keys have them."""
    gen = _gen(seed, salt)
    loud = 0.4 + 0.8 * torch.rand((1, shape[1], 1, shape[3]), device=DEV, generator=gen)
    loud = torch.where(torch.rand(loud.shape, device=DEV, generator=gen) < 0.05, loud * 6.0, loud)
    keys = torch.randn(shape, device=DEV, generator=gen, dtype=t).mul_(loud.to(t))
    return keys, torch.randn(shape, device=DEV, generator=gen, dtype=t).mul_(0.7)


def _power(e: torch.Tensor) -> torch.Tensor:
    """2^e in 32 bits for whole -126 <= e <= 127, from its bits."""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """[..., d] -> codes (float8_e4m3fn, [..., d]) and scale exponents (uint8, [..., d / 32], biased by 127): the least power of
    two under which the group's largest magnitude is at most 448."""
    f = x.float().unflatten(-1, (-1, GROUP)).clamp(-LARGEST[x.dtype], LARGEST[x.dtype])
    most = f.abs().amax(-1)
    m, e = torch.frexp(most)  # most = m 2^e, 0.5 <= m < 1
    biased = torch.where(most > 0, e - 9 + 127 + (m > 0.875).int(), 0).clamp_min(0)
    codes = (f * _power(127 - biased).unsqueeze(-1)).to(torch.float8_e4m3fn)
    return codes.flatten(-2), biased.to(torch.uint8)


def _values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What codes and scales stand for, in 32 bits."""
    f = _power((scales.int() - 126).clamp_min(-126)) * torch.where(scales > 0, 0.5, 0.25).float()
    return (codes.float().unflatten(-1, (-1, GROUP)) * f.unsqueeze(-1)).flatten(-2)


def _cache(case: dict, seed: int) -> dict:
    """A cache's rows as a program holds them: keys and values [sequences or pages, h, n, d], or codes [2, ..] and scales; where in pages, each
    sequence's pages of the pool in its own order."""
    t, seqs, n = TYPES[case["dtype"]], case["seqs"], case["past"] + case["new"]
    store: dict = {"pages": None}
    if case["page"]:
        each = -(-n // case["page"])
        order = torch.randperm(seqs * each + 3, device=DEV, generator=_gen(seed, 9))
        store["pages"] = order[: seqs * each].view(seqs, each).int()
        shape = (seqs * each + 3, case["h"], case["page"], case["d"])
    else:
        shape = (seqs, case["h"], n, case["d"])
    pair = _kv(shape, t, seed, 1)
    if case["eight"]:
        parts = [_quantise(x) for x in pair]
        store["codes"] = torch.stack([c.view(torch.uint8) for c, _ in parts]).view(torch.float8_e4m3fn)
        store["scales"] = torch.stack([s for _, s in parts])
    else:
        store["keys"], store["values"] = pair
    return store


def _counts(case: dict, seed: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(tokens of the call that each sequence has, rows that it has with them): all, or up to that, one sequence at the most and, of more than four, one
    without any."""
    new, past, seqs = case["new"], case["past"], case["seqs"]
    if not case["ragged"]:
        return torch.full((seqs,), new, dtype=torch.int32, device=DEV), torch.full((seqs,), past + new, dtype=torch.int32, device=DEV)
    gen = _gen(seed, 77)
    count = torch.randint(1, new + 1, (seqs,), device=DEV, generator=gen, dtype=torch.int32)
    before = torch.randint(0, past + 1, (seqs,), device=DEV, generator=gen, dtype=torch.int32)
    count[seqs // 2], before[seqs // 2] = new, past
    if seqs > 4:
        count[seqs // 3], before[seqs // 3] = 0, 0
    return count, before + count


def prepare(case: dict, seed: int) -> dict:
    t, seqs, h, g, d, n = TYPES[case["dtype"]], case["seqs"], case["h"], case["g"], case["d"], case["new"]
    state = {"case": case, "dtype": t, "scale": d**-0.5}
    if case["kind"] == "evict":
        state["store"] = _cache(dict(case, new=0), seed)
        gen, m = _gen(seed, 21), case["past"]
        # Sums as attention leaves them: few large ones, many small ones, some rows that were never looked at.
        sums = torch.randn((seqs, h, m), device=DEV, generator=gen).mul_(2.0).exp_()
        state["sums"] = torch.where(torch.rand(sums.shape, device=DEV, generator=gen) < 0.1, 0.0, sums)
        # The tokens that rows hold: in order, but for rows that an earlier eviction moved to the front.
        at = torch.arange(m, device=DEV)
        moved = at // 2 + torch.where(at % 2 > 0, m // 4, 0)
        state["positions"] = torch.where(at < m // 2, moved, at + m // 4).int().expand(seqs, h, m).contiguous()
        state["lengths"] = _counts(dict(case, new=0), seed)[1] if not case["ragged"] else torch.randint(0, m + 1, (seqs,), device=DEV, generator=gen, dtype=torch.int32)
        if case["ragged"]:
            state["lengths"][seqs // 2] = m
        state["out"] = (torch.zeros_like(state["sums"]), torch.zeros_like(state["positions"]))
        return state
    state["store"] = _cache(case, seed)
    state["counts"], state["lengths"] = _counts(case, seed)
    if case["kind"] == "rotate":
        # What a fused projection gives, seen as heads; the tables are as a model's rotary embedding gives them, of each token's position.
        qkv = torch.randn((seqs, n, h * (g + 2), d), device=DEV, generator=_gen(seed, 2), dtype=t)
        qkv.mul_(torch.where(torch.rand((1, 1, h * (g + 2), d), device=DEV, generator=_gen(seed, 3)) < 0.05, 5.0, 0.8).to(t))
        state["q"], state["k"], state["v"] = (x.transpose(1, 2) for x in qkv.split((h * g, h, h), 2))
        state["starts"] = state["lengths"] - state["counts"]
        at = state["starts"][:, None].double() + torch.arange(n, device=DEV)
        rate = 500000.0 ** (-torch.arange(0, case["rot"], 2, device=DEV, dtype=torch.float64) / case["rot"])
        angle = (at.unsqueeze(-1) * rate).repeat(1, 1, 2)
        state["cos"], state["sin"] = angle.cos().to(t), angle.sin().to(t)
        if case["norm"]:
            state["wq"], state["wk"] = (torch.randn((2, d), device=DEV, generator=_gen(seed, 4)) * 0.2 + 1.0).to(t).unbind(0)
        else:
            state["wq"] = state["wk"] = None
        return state
    q = torch.randn((seqs, n, h * g, d), device=DEV, generator=_gen(seed, 2))
    state["q"] = (q * 1.5).to(t).transpose(1, 2)
    if case["kind"] == "weigh":
        state["lse"] = _attend(state)[1]
        m = case["past"] + n
        state["sums"] = torch.randn((seqs, h, m), device=DEV, generator=_gen(seed, 5)).exp_()
        state["out"] = torch.zeros_like(state["sums"])
        state["positions"] = torch.full((seqs, h, m), -1, dtype=torch.int32, device=DEV)
        state["seen"] = state["lengths"] - state["counts"] + 1000  # as many were evicted before
    return state


# -- one pass ---------------------------------------------------------------------------------------


def run(state: dict):
    if own:
        return _run_own(state)
    kind = state["case"]["kind"]
    return _rotate(state) if kind == "rotate" else _attend(state) if kind == "attend" else _weigh(state) if kind == "weigh" else _evict(state)


def _dense(store: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """Each sequence's keys and values one after the other, [seqs, h, n, d] in 32 bits."""
    pair = _values(store["codes"], store["scales"]).unbind(0) if "codes" in store else (store["keys"].float(), store["values"].float())
    if store["pages"] is None:
        return pair
    return tuple(x[store["pages"].long()].transpose(1, 2).flatten(2, 3) for x in pair)


def _turned(x: torch.Tensor, w: torch.Tensor | None, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
    r = cos.shape[-1]
    a, b = x[..., : r // 2], x[..., r // 2 : r]
    turned = x[..., :r] * cos.float().unsqueeze(1) + torch.cat([-b, a], -1) * sin.float().unsqueeze(1)
    return torch.cat([turned, x[..., r:]], -1)


def _rotate(state: dict):
    t, store, case = state["dtype"], state["store"], state["case"]
    q = _turned(state["q"], state["wq"], state["cos"], state["sin"]).to(t)
    k = _turned(state["k"], state["wk"], state["cos"], state["sin"]).to(t)
    # Token t of sequence b: its row, and the page or sequence that holds it; tokens behind a sequence's count go nowhere.
    new = torch.arange(case["new"], device=DEV)
    b, s = (new < state["counts"][:, None]).nonzero(as_tuple=True)
    at = state["starts"].long()[b] + s
    if store["pages"] is None:
        where = b
    else:
        where, at = store["pages"][b, at // case["page"]].long(), at % case["page"]
    for i, x in enumerate((k, state["v"])):
        x = x.transpose(1, 2)[b, s]  # [tokens, h, d]
        if "codes" in store:
            codes, scales = _quantise(x)
            store["codes"].view(torch.uint8)[i].transpose(1, 2)[where, at] = codes.view(torch.uint8)
            store["scales"][i].transpose(1, 2)[where, at] = scales
        else:
            store["values" if i else "keys"].transpose(1, 2)[where, at] = x
    if "codes" in store:  # read back, for the forward that wrote them
        return [q, *_values(store["codes"], store["scales"]).to(t).unbind(0)]
    return [q, store["keys"], store["values"]]


def _scores(state: dict, k: torch.Tensor) -> torch.Tensor:
    """[seqs, h, g * new, n] in 32 bits, what a token does not attend at -inf."""
    seqs, n_q, new, d = state["q"].shape
    q = state["q"].float().reshape(seqs, k.shape[1], -1, d) * state["scale"]
    t = torch.arange(new, device=DEV)
    past = (state["lengths"] - state["counts"])[:, None]
    limit = torch.where(t < state["counts"][:, None], past + t + 1, 0).repeat(1, n_q // k.shape[1])  # [seqs, g * new]
    seen = torch.arange(k.shape[2], device=DEV) < limit.unsqueeze(-1)
    return (q @ k.transpose(-1, -2)).masked_fill_(~seen.unsqueeze(1), float("-inf"))


def _attend(state: dict):
    """Softmax over each token's rows, in 32 bits."""
    k, v = _dense(state["store"])
    s = _scores(state, k)
    m = s.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = s.sub_(m).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.where(total > 0, (p @ v) / total, 0.0)
    return [out.view(state["q"].shape).to(state["dtype"]), (m + total.log()).view(state["q"].shape[:3])]


def _weigh(state: dict):
    """Each row's weights summed over the tokens and the heads of its group."""
    case, k = state["case"], _dense(state["store"])[0]
    s = _scores(state, k)
    lse = state["lse"].reshape(*s.shape[:3], 1)
    got = s.sub_(lse.masked_fill(lse == float("-inf"), 0.0)).exp_().sum(2)[..., : case["past"] + case["new"]]
    i = torch.arange(got.shape[2], device=DEV)
    length, past = (x[:, None, None] for x in (state["lengths"], state["lengths"] - state["counts"]))
    state["out"].copy_(torch.where(i < past, state["sums"] + got, torch.where(i < length, got, state["out"])))
    at = state["seen"][:, None, None] + i - past
    state["positions"].copy_(torch.where((i >= past) & (i < length), at, state["positions"]))
    return [state["out"], state["positions"]]


def _evict(state: dict):
    """The `keep` rows of the largest sums, ties to the lowest row, the first and the newest tokens before all; those of them that lie behind row `keep` go,
    in their order, to the rows before it that are not kept."""
    case, store = state["case"], state["store"]
    keep, m = case["keep"], state["sums"].shape[2]
    i = torch.arange(m, device=DEV)
    live = (i < state["lengths"][:, None, None]).expand_as(state["sums"])
    newest = torch.where(live, state["positions"], -1).amax(-1, keepdim=True)
    held = live & ((state["positions"] < case["sinks"]) | (state["positions"] > newest - case["recent"]))
    rank = torch.where(held, float("inf"), torch.where(live, state["sums"], float("-inf")))
    chosen = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :keep]
    kept = torch.zeros_like(live).scatter_(-1, chosen, True) & live
    from_ = (kept & (i >= keep)).nonzero(as_tuple=True)
    holes = (~kept & (i < keep) & (i < state["lengths"][:, None, None])).nonzero(as_tuple=True)
    (b, j, src), dst = from_, holes[2]  # as many of both, of each head in their order
    left = i < state["lengths"].clamp_max(keep)[:, None, None]
    for to, of in zip(state["out"], (state["sums"], state["positions"])):
        to.copy_(torch.where(left, of, to))
        to[b, j, dst] = of[b, j, src]
    to, of = (b, b) if store["pages"] is None else (store["pages"][b, x // case["page"]].long() for x in (dst, src))
    if store["pages"] is not None:
        src, dst = src % case["page"], dst % case["page"]
    for name in ("codes", "scales") if "codes" in store else ("keys", "values"):
        x = store[name].view(torch.uint8) if name == "codes" else store[name]
        if x.dim() == 5:
            x[:, to, j, dst] = x[:, of, j, src]
        else:
            x[to, j, dst] = x[of, j, src]
    return [*(store[x] for x in (("codes", "scales") if "codes" in store else ("keys", "values"))), *state["out"]]


def _run_own(state: dict):
    from lazykv_amd import kernels

    store, case, kind = state["store"], state["case"], state["case"]["kind"]
    if "codes" in store:
        rows = kernels.mx_rows(store["codes"], store["scales"], state["dtype"])
    else:
        rows = kernels.dense_rows(store["keys"], store["values"])
    pages, most = store["pages"], case["past"] + case["new"]
    if kind == "rotate":
        q = kernels.rotate_append(rows, state["q"], state["k"], state["v"], cos=state["cos"], sin=state["sin"], q_weight=state["wq"], k_weight=state["wk"], eps=EPS,
                                  starts=state["starts"], counts=state["counts"], pages=pages)
        return [q, *(kernels.read_rows(rows, 0, rows.tokens) if "codes" in store else (store["keys"], store["values"]))]
    if kind == "attend":
        return list(kernels.chunk_attend(state["q"], rows, scale=state["scale"], lengths=state["lengths"], counts=state["counts"], max_tokens=most, pages=pages))
    if kind == "weigh":
        kernels.weigh_rows(state["q"], state["lse"], rows, scale=state["scale"], lengths=state["lengths"], counts=state["counts"], max_tokens=most, pages=pages,
                           sums=state["sums"], out=state["out"], positions=state["positions"], seen=state["seen"])
        return [state["out"], state["positions"]]
    kernels.evict_rows(rows, state["sums"], state["positions"], keep=case["keep"], sinks=case["sinks"], recent=case["recent"], lengths=state["lengths"],
                       max_tokens=case["past"], pages=pages, out=state["out"])
    return [*(store[x] for x in (("codes", "scales") if "codes" in store else ("keys", "values"))), *state["out"]]


# -- what a pass cannot do without, and what it gives in 64 bits ------------------------------------


def work(case: dict) -> dict:
    h, g, d, seqs, new, past = (case[x] for x in ("h", "g", "d", "seqs", "new", "past"))
    row = d + d // GROUP if case["eight"] else 2 * d
    tokens = seqs * (1.0 + (new - 1) * 0.5 if case["ragged"] else new)  # on average
    before = seqs * past * (0.5 if case["ragged"] else 1.0)
    if case["kind"] == "rotate":
        tables = 4 * case["rot"] * seqs * new
        moved = seqs * new * h * g * 4 * d + tokens * h * 2 * (2 * d + row) + tables
        if case["eight"]:
            moved += 2 * seqs * (new + past) * h * (row + 2 * d)
        return {"bytes": moved, "flops": 6.0 * (tokens * h + seqs * new * h * g) * d}
    if case["kind"] == "evict":
        left = case["keep"] * before / past
        share = max(0.0, 1.0 - case["keep"] / past)  # of the rows that stay, those behind `keep`
        return {"bytes": before * h * 8 + left * h * 8 + 2 * 2 * left * share * h * row, "flops": before * h}
    pairs = tokens * (before / seqs + (1 + tokens / seqs) / 2)  # of a token and a row that it attends
    if case["kind"] == "attend":
        return {"bytes": 2 * h * row * (before + tokens) + seqs * new * h * g * (4 * d + 4), "flops": 4.0 * h * g * d * pairs}
    return {"bytes": h * row * (before + tokens) + h * 4 * (2 * before + 2 * tokens) + seqs * new * h * g * (2 * d + 4), "flops": 2.0 * h * g * d * pairs}


def _power64(e: torch.Tensor) -> torch.Tensor:
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_coded(x: torch.Tensor, t: torch.dtype) -> torch.Tensor:
    """What a row [.., d] of 64-bit values of type `t` is held as in 8 bits: the scale found by trying, codes to the nearest value of four bits, ties to
    even, in steps of 2^-9 at the least."""
    y = x.unflatten(-1, (-1, GROUP)).clamp(-LARGEST[t], LARGEST[t])
    most = y.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(most / 448.0)).clamp(-127, 127)
    e = torch.where(most > 448.0 * _power64(e), e + 1, e)
    e = torch.where(most <= 448.0 * _power64(e - 1), e - 1, e).clamp(-127, 127)
    scale = _power64(torch.where(most > 0, e, -127.0))
    y = y / scale
    step = _power64((torch.frexp(y)[1] - 1).clamp_min(-6) - 3)
    return (torch.round(y / step) * step * scale).flatten(-2)


def _exact_rows(store: dict) -> list[torch.Tensor]:
    if "keys" in store:
        return [store["keys"].double(), store["values"].double()]
    return list((store["codes"].double() * _power64(store["scales"].long() - 127).repeat_interleave(GROUP, -1)).unbind(0))


def _exact_rotate(state: dict):
    case, store, t = state["case"], state["store"], state["dtype"]
    rows = _exact_rows(store)
    half = case["rot"] // 2
    cos, sin = state["cos"].double(), state["sin"].double()

    def turn(x: torch.Tensor, w: torch.Tensor | None) -> torch.Tensor:
        y = x.double()
        if w is not None:
            y = y / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS) * w.double()
        z = y.clone()
        z[..., :half] = y[..., :half] * cos[:, None, :, :half] - y[..., half : 2 * half] * sin[:, None, :, :half]
        z[..., half : 2 * half] = y[..., half : 2 * half] * cos[:, None, :, half:] + y[..., :half] * sin[:, None, :, half:]
        return z

    k, v = turn(state["k"], state["wk"]), state["v"].double()
    if case["eight"]:
        k, v = _exact_coded(k.to(t).double(), t), _exact_coded(v, t)
    counts, starts = state["counts"].tolist(), state["starts"].tolist()
    for b, n in enumerate(counts):
        if store["pages"] is None:
            for of, to in zip((k, v), rows):
                to[b, :, starts[b] : starts[b] + n] = of[b, :, :n]
            continue
        pages = store["pages"][b].tolist()
        done = 0
        while done < n:  # a page at a time
            at = starts[b] + done
            some = min(n - done, case["page"] - at % case["page"])
            for of, to in zip((k, v), rows):
                to[pages[at // case["page"]], :, at % case["page"] : at % case["page"] + some] = of[b, :, done : done + some]
            done += some
    return [turn(state["q"], state["wq"]), *rows]


def _exact_sequence(state: dict, b: int, rows: list[torch.Tensor]) -> list[torch.Tensor]:
    """Sequence b's keys and values [h, length, d], page by page."""
    n, store = int(state["lengths"][b]), state["store"]
    if store["pages"] is None:
        return [x[b, :, :n] for x in rows]
    return [torch.cat([x[p] for p in store["pages"][b].tolist()], 1)[:, :n] for x in rows]


def exact(case: dict, seed: int):
    state = prepare(case, seed)
    store, kind = state["store"], case["kind"]
    if kind == "rotate":
        return _exact_rotate(state)
    if kind == "evict":
        return _exact_evict(state)
    h, g, seqs, new = case["h"], case["g"], case["seqs"], case["new"]
    rows = _exact_rows(store)
    out = torch.zeros((seqs, h * g, new, case["d"]), dtype=torch.float64, device=DEV)
    lse = torch.full((seqs, h * g, new), float("-inf"), dtype=torch.float64, device=DEV)
    sums, positions = state.get("out"), state.get("positions")
    sums = sums.double() if kind == "weigh" else None
    for b, n in enumerate(state["counts"].tolist()):
        k, v = _exact_sequence(state, b, rows)
        past = k.shape[1] - n
        hidden = torch.ones((n, k.shape[1]), dtype=torch.bool, device=DEV).triu(past + 1)
        for j in range(h):
            got = torch.zeros(k.shape[1], dtype=torch.float64, device=DEV)
            for i in range(j * g, (j + 1) * g):
                s = (state["q"][b, i, :n].double() @ k[j].T / math.sqrt(case["d"])).masked_fill_(hidden, float("-inf"))
                if kind == "attend":
                    lse[b, i, :n] = torch.logsumexp(s, -1)
                    out[b, i, :n] = torch.softmax(s, -1) @ v[j]
                else:
                    got += (s - state["lse"][b, i, :n, None].double()).exp().sum(0)
            if kind == "weigh":
                got[:past] += state["sums"][b, j, :past].double()
                sums[b, j, : k.shape[1]] = got
                positions[b, j, past : past + n] = int(state["seen"][b]) + torch.arange(n, dtype=torch.int32, device=DEV)
    return [out, lse] if kind == "attend" else [sums, positions]


def _exact_evict(state: dict):
    """A head's rows after the other's, sorted by (whether they stay whatever their sums, the sums, the row) on the host."""
    case, store, keep = state["case"], state["store"], state["case"]["keep"]
    names = ("codes", "scales") if "codes" in store else ("keys", "values")
    held = [store[x].view(torch.uint8) if x == "codes" else store[x] for x in names]
    table = None if store["pages"] is None else store["pages"].cpu().numpy()
    out = [x.cpu().numpy() for x in state["out"]]
    every = [x.cpu().numpy() for x in (state["sums"], state["positions"])]
    for b, n in enumerate(state["lengths"].tolist()):
        for j in range(case["h"] if n else 0):
            sums, at = (x[b, j, :n].copy() for x in every)
            stays = (at < case["sinks"]) | (at > at.max() - case["recent"])
            order = np.lexsort((np.arange(n), np.where(stays, 0.0, -sums.astype(np.float64)), ~stays))
            kept = np.sort(order[:keep])
            of = kept[kept >= keep]
            to = np.setdiff1d(np.arange(min(keep, n)), kept)
            sums[to], at[to] = sums[of], at[of]
            out[0][b, j, : min(n, keep)], out[1][b, j, : min(n, keep)] = sums[:keep], at[:keep]
            if not len(of):
                continue
            (tp, ti), (sp, si) = ((np.full_like(x, b), x) if table is None else (table[b][x // case["page"]], x % case["page"]) for x in (to, of))
            tp, ti, sp, si = (torch.from_numpy(np.ascontiguousarray(x)).long().to(DEV) for x in (tp, ti, sp, si))
            for x in held:
                if x.dim() == 5:
                    x[:, tp, j, ti] = x[:, sp, j, si]
                else:
                    x[tp, j, ti] = x[sp, j, si]
    return [*(store[x] for x in names), *(torch.from_numpy(x).to(DEV) for x in out)]
