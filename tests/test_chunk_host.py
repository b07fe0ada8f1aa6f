"""What the calls of a layer's forward over a bounded cache do on the host (CPU): the arithmetic of pages, scratch, and checks that come before any launch."""

from __future__ import annotations

import ctypes

import pytest


@pytest.mark.parametrize("sixteens", [1, 2, 3, 5, 7, 8, 12, 60, 63, 64, 65, 341, 1000, 1023, 1024])
def test_a_rows_page_is_found_by_one_multiplication(sixteens: int) -> None:
    """The kernels divide a row's group of sixteen by a page's as (group * ceil(2^36 / sixteens)) >> 36: exact for every group below 2^26 (rows below 2^30), within
    64 bits. The error of the factor is less than sixteens / 2^36, so that of the quotient less than 2^26 * 2^10 / 2^36 = 1 of a step: the borders decide."""
    magic = ((1 << 36) + sixteens - 1) // sixteens
    top = 1 << 26
    assert (top - 1) * magic < 1 << 64
    quotients = sorted({0, 1, 2, top // sixteens // 2, (top - 1) // sixteens - 1, (top - 1) // sixteens, *range(0, top // sixteens, max(1, top // sixteens // 997))})
    for quotient in quotients:
        for group in (quotient * sixteens, quotient * sixteens + sixteens - 1, quotient * sixteens + sixteens // 2):
            if 0 <= group < top:
                assert (group * magic) >> 36 == group // sixteens


def _chunk(n_seqs: int, n_q: int, n_kv: int, d: int, t: int, most: int):  # noqa: ANN202
    from lazykv_amd import _lib

    return _lib.ChunkDesc(n_seqs, n_q, n_kv, d, t, 0.1, 0, most, n_q * t * d, t * d, d)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize(("n_q", "n_kv"), [(1, 1), (4, 1), (32, 8), (40, 1), (128, 128)])
def test_scratch_is_bounded(n_q: int, n_kv: int, d: int) -> None:
    """Partial results of attention are for at most 1,024 workgroups of 128 query rows: rows are divided as 512 workgroups would share them, a sequence of several parts has
    fewer than twice as many as its rows make whole ones, and one of a single part writes the output. Sums by parts are for at most 2,048 workgroups of 256 rows."""
    from lazykv_amd import _lib

    lib = _lib.lib()
    for n_seqs in (1, 3, 16, 257):
        for t in (0, 1, 2, 7, 9, 33, 203, 2048):
            for most in (0, 1, 127, 4099, 131072, 1 << 30):
                if n_seqs * n_q * t > 1 << 26:
                    continue
                desc = ctypes.byref(_chunk(n_seqs, n_q, n_kv, d, t, most))
                assert lib.lkv_chunk_attend_workspace_bytes(desc) <= 1024 * 128 * (d + 2) * 4 + 16, (n_seqs, t, most)
                assert lib.lkv_weigh_rows_workspace_bytes(desc) <= 2048 * 256 * 4, (n_seqs, t, most)


CHUNK = {"desc": {"n_seqs": 2, "n_q": 8, "n_kv": 2, "head_dim": 64, "new_tokens": 3, "scale": 0.1, "tokens": 0, "max_tokens": 64}, "strides": (1536, 192, 64), "q": 4096, "dtype": 0,
         "rows": {"seqs": 9, "tokens": 16, "dtype": 0, "k": 4096, "v": 1 << 20, "seq_stride": 2048, "head_stride": 1024}, "pages": {"table": 4096, "seq_stride": 4, "n_pages": 4},
         "out": 4096, "lse": 4096, "ws": 4096, "ws_bytes": 1 << 30}


def _call(fn: str, change: dict) -> str:
    """A call with one thing wrong; the refusal's message. Nothing it is given is memory: a refusal comes before any use of it."""
    from lazykv_amd import _lib

    case = {k: ({**v, **(change.get(k) or {})} if isinstance(v, dict) else change.get(k, v)) for k, v in CHUNK.items()}
    lib = _lib.lib()
    r, p = case["rows"], case["pages"]
    rows = _lib.KVRows(r["k"], r["v"], r.get("k_scale"), r.get("v_scale"), r["seq_stride"], r["head_stride"], r["tokens"], r["seqs"], r["dtype"], 0)
    pages = _lib.Pages(p["table"], p["seq_stride"], p["n_pages"]) if change.get("pages", 1) is not None else None
    refs = ctypes.byref(rows), (None if pages is None else ctypes.byref(pages))
    d = case["desc"]
    desc = _lib.ChunkDesc(d["n_seqs"], d["n_q"], d["n_kv"], d["head_dim"], d["new_tokens"], d["scale"], d["tokens"], d["max_tokens"], *case["strides"])
    two = _lib.Pair(128, 64)
    if fn == "attend":
        rc = lib.lkv_chunk_attend(0, ctypes.byref(desc), case["q"], case["dtype"], *refs, None, None, case["out"], 0, case["lse"], case["ws"], case["ws_bytes"])
    elif fn == "weigh":
        rc = lib.lkv_weigh_rows(0, ctypes.byref(desc), case["q"], case["dtype"], case["lse"], *refs, None, None, None, None, case["out"], two, None, None, None, case["ws"],
                                case["ws_bytes"])
    elif fn == "evict":
        e = {"keep": 8, "sinks": 0, "recent": 0, **change.get("evict", {})}
        ev = _lib.EvictDesc(d["n_seqs"], d["n_kv"], d["head_dim"], case["dtype"], e["keep"], e["sinks"], e["recent"], d["tokens"], d["max_tokens"])
        rc = lib.lkv_evict_rows(0, ctypes.byref(ev), *refs, None, case["lse"], two, case["lse"], two, case["out"], two, case["out"], two, case["ws"], case["ws_bytes"])
    else:
        x = {"rotary": 64, "table": 0, "weight": 0, "eps": 0.0, "start": 0, "cos": 4096, **change.get("rotate", {})}
        st = case["strides"]
        ro = _lib.RotateDesc(d["n_seqs"], d["n_q"], d["n_kv"], d["head_dim"], d["new_tokens"], case["dtype"], x["rotary"], x["table"], x["weight"], x["eps"], *st, *st, *st, *st, 0)
        rc = lib.lkv_rotate_append(0, ctypes.byref(ro), case["q"], case["q"], case["q"], x["cos"], x["cos"], case["q"], case["q"], case["out"], *refs, None, x["start"], None)
    assert rc == -1, rc
    return lib.lkv_last_error().decode()


EVERY = ("attend", "weigh", "evict", "rotate")


@pytest.mark.parametrize(("fns", "change", "says"), [
    (EVERY, {"desc": {"head_dim": 96}}, "head_dim 96"),
    (EVERY, {"desc": {"n_seqs": -1}}, "bad shape"),
    (EVERY, {"desc": {"n_kv": 0}}, "bad shape"),
    (EVERY, {"dtype": 2}, "dtype"),
    (EVERY, {"rows": {"k": 0}}, "NULL"),
    (EVERY, {"rows": {"k": 4104}}, "16 bytes"),
    (EVERY, {"rows": {"tokens": 24}}, "multiple of 16"),
    (EVERY, {"rows": {"tokens": 0}}, "multiple of 16"),
    (EVERY, {"rows": {"tokens": 32768}}, "16384"),
    (EVERY, {"rows": {"seqs": 0}}, "without pages"),
    (EVERY, {"rows": {"seq_stride": 2056}}, "multiples of 32"),
    (EVERY, {"rows": {"dtype": 1}}, "under a call"),
    (EVERY, {"rows": {"dtype": 4}}, "scales"),
    (EVERY, {"pages": {"n_pages": -1}}, "page table"),
    (EVERY, {"pages": {"table": 0}}, "page table"),
    (EVERY, {"pages": {"n_pages": 1 << 27}}, "at most"),
    (EVERY, {"pages": None}, "rows of 9 sequences"),
    (("attend", "weigh", "evict"), {"desc": {"max_tokens": 65}}, "over 64"),
    (("attend", "weigh", "evict"), {"desc": {"max_tokens": -1}}, "bad extent"),
    (("attend", "weigh", "evict"), {"desc": {"tokens": -1}}, "bad extent"),
    (("evict",), {"ws": 0}, "workspace"),
    (("evict",), {"ws_bytes": 8}, "workspace"),
    (("evict",), {"ws": 4104}, "workspace"),
    (("attend", "weigh"), {"desc": {"n_q": 9}}, "bad shape"),
    (("attend", "weigh"), {"desc": {"new_tokens": -1}}, "bad shape"),
    (("attend", "weigh"), {"desc": {"new_tokens": 1 << 23}}, "query rows"),
    (("attend", "weigh"), {"desc": {"scale": 0.0}}, "scale"),
    (("attend", "weigh"), {"desc": {"scale": float("inf")}}, "scale"),
    (("attend", "weigh"), {"strides": (1536, 192, 60)}, "multiples of 8"),
    (("attend", "weigh"), {"q": 4104}, "16 bytes"),
    (("attend", "weigh"), {"q": 0}, "NULL"),
    (("evict",), {"evict": {"keep": 0}}, "that are kept"),
    (("evict",), {"evict": {"sinks": 5, "recent": 4}}, "that are kept"),
    (("evict",), {"evict": {"recent": -1}}, "that are kept"),
    (("rotate",), {"rotate": {"rotary": 24}}, "multiple of 16"),
    (("rotate",), {"rotate": {"rotary": 80}}, "at most 64"),
    (("rotate",), {"rotate": {"cos": 0}}, "tables"),
    (("rotate",), {"rotate": {"table": 1}}, "tables of dtype"),
    (("rotate",), {"rotate": {"weight": 1}}, "weights of dtype"),
    (("rotate",), {"rotate": {"eps": -1.0}}, "eps"),
    (("rotate",), {"rotate": {"eps": 1e-40}}, "eps"),
    (("weigh",), {"desc": {"scale": 1e-39}}, "reciprocal"),
    (("rotate",), {"rotate": {"start": 62}}, "exceed"),
    (("rotate",), {"desc": {"n_q": 1 << 20, "new_tokens": 1 << 11}, "rows": {"tokens": 16384}}, "in one call"),
    (("rotate",), {"desc": {"n_q": 1, "n_kv": 1, "n_seqs": 1 << 14, "new_tokens": 1 << 10}, "rows": {"tokens": 16384}}, "in one call"),
    (("attend", "weigh"), {"desc": {"n_seqs": 1 << 30, "new_tokens": 0}}, "query rows"),
    (("evict",), {"desc": {"n_seqs": 1 << 30, "n_kv": 1 << 30}}, "in one call"),
    (("attend",), {"desc": {"n_seqs": 1 << 25, "n_q": 2, "new_tokens": 1}}, "in one call"),
    (("weigh",), {"desc": {"n_seqs": 1 << 25, "n_q": 2, "new_tokens": 1}}, "in one call"),
    (("evict",), {"desc": {"n_seqs": 1 << 10, "n_kv": 8, "max_tokens": 1 << 24}, "rows": {"tokens": 16384}, "pages": {"n_pages": 1024}, "ws_bytes": 1 << 60}, "in one call"),
    (("rotate",), {"strides": (1536, 192, 60)}, "multiples of 8"),
    (("rotate",), {"strides": (0, 192, 64)}, "share an address"),
    (("rotate", "evict"), {"rows": {"seq_stride": 1024}}, "share an address"),
    (("rotate", "evict"), {"rows": {"v": 4096}}, "share an address"),
])
def test_calls_are_refused_before_any_launch(fns: tuple, change: dict, says: str) -> None:
    for fn in fns:
        assert says in _call(fn, change), (fn, _call(fn, change))


def test_tensors_on_the_host_are_refused() -> None:
    import torch

    from lazykv_amd import kernels

    with pytest.raises(RuntimeError, match="no CPU path"):
        kernels.evict_rows(None, torch.zeros((1, 1, 8)), torch.zeros((1, 1, 8), dtype=torch.int32), keep=4, tokens=8)


@pytest.fixture
def kernels(monkeypatch: pytest.MonkeyPatch):  # noqa: ANN201
    """The calls' checks over tensors on the host. Nothing is launched: a call that comes so far fails the test."""
    from lazykv_amd import _lib, kernels

    monkeypatch.setattr(_lib, "require_cuda", lambda *_: None)
    monkeypatch.setattr(kernels, "_launch", lambda _, fn, *args: pytest.fail(f"{fn} was launched"))
    return kernels


def test_queries_without_heads_are_refused(kernels) -> None:  # noqa: ANN001
    """Their keys and values would be new rows: returning without them would lose them."""
    import torch

    rows = kernels.dense_rows(*torch.zeros((2, 2, 2, 16, 64), dtype=torch.bfloat16))
    q, k = torch.zeros((2, 0, 3, 64), dtype=torch.bfloat16), torch.zeros((2, 2, 3, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="without heads"):
        kernels.rotate_append(rows, q, k, k)
    with pytest.raises(ValueError, match="does not match"):
        kernels.chunk_attend(q, rows, scale=0.1, tokens=9)


@pytest.mark.parametrize("scale", [1e-39, 1e-38, 2.0**-121])
def test_accounts_of_scales_whose_reciprocal_times_an_lse_is_not_finite_are_refused(scale: float) -> None:
    """Few query rows' scores start from -lse / scale: at 1e-38 an lse of 4.2 (64 rows alike) is past float32's range there, and every weight would be 0."""
    assert "reciprocal" in _call("weigh", {"desc": {"scale": scale}})


def _pool(eight: bool, n_bytes: int):  # noqa: ANN202
    """(a buffer of bytes, (sequences, h, tokens, d), rows at its start): two sequences of two heads, 16 rows of 64 channels."""
    import torch

    from lazykv_amd import kernels

    pool = torch.zeros(n_bytes, dtype=torch.uint8)
    if eight:
        return pool, kernels.mx_rows(pool[:8192].view(2, 2, 2, 16, 64), pool[8192:8448].view(2, 2, 2, 16, 2), torch.bfloat16)
    return pool, kernels.dense_rows(*pool[:16384].view(torch.bfloat16).view(2, 2, 2, 16, 64))


@pytest.mark.parametrize(("eight", "at"), [(False, 0), (False, 8192), (False, 16128), (True, 0), (True, 4096), (True, 8064), (True, 8192), (True, 8320)])
def test_what_lies_among_a_caches_rows_is_refused(kernels, eight: bool, at: int) -> None:  # noqa: ANN001
    """A pool of bytes cut into a cache and what calls write: what is cut from keys, values, their codes or their scales, or reaches into them, is refused."""
    import torch

    pool, rows = _pool(eight, 1 << 16)
    cut = lambda dtype, *shape: pool[at:].view(dtype)[: torch.Size(shape).numel()].view(shape)  # noqa: E731
    q, k = torch.zeros((2, 4, 3, 64), dtype=torch.bfloat16), torch.zeros((2, 2, 3, 64), dtype=torch.bfloat16)
    lse, sums, positions = torch.zeros((2, 4, 3)), torch.zeros((2, 2, 16)), torch.zeros((2, 2, 16), dtype=torch.int32)
    with pytest.raises(ValueError, match="must not lie among"):
        kernels.rotate_append(rows, q, k, k, out=cut(torch.bfloat16, 2, 4, 3, 64))
    kw = dict(scale=0.1, tokens=16)
    for out in ({"out": cut(torch.bfloat16, 2, 4, 3, 64)}, {"lse": cut(torch.float32, 2, 4, 3)}):
        with pytest.raises(ValueError, match="must not lie among"):
            kernels.chunk_attend(q, rows, **kw, **out)
    for out in ({"out": cut(torch.float32, 2, 2, 16)}, {"sums": cut(torch.float32, 2, 2, 16)}, {"positions": cut(torch.int32, 2, 2, 16)}):
        with pytest.raises(ValueError, match="must not lie among"):
            kernels.weigh_rows(q, lse, rows, **kw, **out)
    for args, out in (((cut(torch.float32, 2, 2, 16), positions), None), ((sums, cut(torch.int32, 2, 2, 16)), None), ((sums, positions), (cut(torch.float32, 2, 2, 8), positions)),
                      ((sums, positions), (sums, cut(torch.int32, 2, 2, 8)))):
        with pytest.raises(ValueError, match="share addresses"):
            kernels.evict_rows(rows, *args, keep=8, tokens=16, out=out)


@pytest.mark.parametrize("eight", [False, True])
def test_what_lies_beside_a_caches_rows_is_launched(monkeypatch: pytest.MonkeyPatch, kernels, eight: bool) -> None:  # noqa: ANN001
    import torch

    launched = []
    monkeypatch.setattr(kernels, "_launch", lambda _, fn, *args: launched.append(args) or 0)
    pool, rows = _pool(eight, 1 << 16)
    at = 8448 if eight else 16384
    cut = lambda dtype, *shape: pool[at:].view(dtype)[: torch.Size(shape).numel()].view(shape)  # noqa: E731
    q, k = torch.zeros((2, 4, 3, 64), dtype=torch.bfloat16), torch.zeros((2, 2, 3, 64), dtype=torch.bfloat16)
    lse, sums, positions = torch.zeros((2, 4, 3)), torch.zeros((2, 2, 16)), torch.zeros((2, 2, 16), dtype=torch.int32)
    kernels.rotate_append(rows, q, k, k, out=cut(torch.bfloat16, 2, 4, 3, 64))
    kernels.chunk_attend(q, rows, scale=0.1, tokens=16, out=cut(torch.bfloat16, 2, 4, 3, 64))
    kernels.weigh_rows(q, lse, rows, scale=0.1, tokens=16, sums=cut(torch.float32, 2, 2, 16), positions=positions)
    kernels.evict_rows(rows, sums, cut(torch.int32, 2, 2, 16), keep=8, tokens=16)
    assert len(launched) == 4


@pytest.mark.parametrize(("eight", "at"), [(False, 0), (False, 8192), (True, 0), (True, 4096), (True, 8192), (True, 8320)])
def test_new_tokens_that_lie_among_a_caches_rows_are_copied_first(monkeypatch: pytest.MonkeyPatch, kernels, eight: bool, at: int) -> None:  # noqa: ANN001
    """Their bytes are the cache's, in its dtype or not: the launch gets others."""
    import torch

    launched = []
    monkeypatch.setattr(kernels, "_launch", lambda _, fn, *args: launched.append(args) or 0)
    pool, rows = _pool(eight, 1 << 16)
    lo = pool.data_ptr()
    hi = lo + (8448 if eight else 16384)
    mine = pool[at:].view(torch.bfloat16)[: 2 * 2 * 3 * 64].view(2, 2, 3, 64)
    other = torch.zeros((2, 2, 3, 64), dtype=torch.bfloat16)
    kernels.append_rows(rows, mine, other)
    kernels.append_rows(rows, other, mine)
    kernels.rotate_append(rows, mine, other, other)
    kernels.rotate_append(rows, other, mine, other)
    kernels.rotate_append(rows, other, other, mine)
    assert len(launched) == 5
    for args in launched:
        addresses = [x for x in args[1:4] if isinstance(x, int) and x > 1 << 20]
        assert len(addresses) >= 2 and not any(lo <= x < hi for x in addresses), (lo, hi, addresses)


def test_numbers_that_lie_among_what_a_call_writes_are_copied_first(monkeypatch: pytest.MonkeyPatch, kernels) -> None:  # noqa: ANN001
    """Lengths, counts, page tables and the tokens seen are read by workgroups that others are ahead of: where one buffer holds them and a call's outputs, the launch
    gets copies, with their values, and elsewhere the tensors themselves."""
    import torch

    launched = []

    def launch(_: int, fn, *args) -> int:  # noqa: ANN001, ANN002
        flat = [y for x in args for y in ((x.table,) if isinstance(x, _lib.Pages) else (x,)) if isinstance(y, int) and y > 1 << 20]
        launched.append({y: ctypes.c_int32.from_address(y).value for y in flat})
        return 0

    from lazykv_amd import _lib

    monkeypatch.setattr(kernels, "_launch", launch)
    rows = kernels.dense_rows(*torch.zeros((2, 4, 2, 16, 64), dtype=torch.bfloat16))
    q, k = torch.zeros((2, 4, 3, 64), dtype=torch.bfloat16), torch.zeros((2, 2, 3, 64), dtype=torch.bfloat16)
    lse, sums = torch.zeros((2, 4, 3)), torch.zeros((2, 2, 16))
    state = torch.zeros(4096, dtype=torch.int32)
    far = torch.zeros(16, dtype=torch.int32)
    for one, (name, n) in enumerate((("counts", 2), ("pages", 2), ("lengths", 2), ("seen", 2))):
        for among in (True, False):
            mine = (state[6:8] if among else far[:n]).copy_(torch.tensor([one + 1, 2]))
            lo = state.data_ptr()
            kw = {"lengths": torch.tensor([9, 9], dtype=torch.int32), "pages": torch.tensor([[0], [1]], dtype=torch.int32), name: mine.view(2, 1) if name == "pages" else mine}
            calls = [lambda: kernels.weigh_rows(q, lse, rows, scale=0.1, sums=sums, positions=state[:64].view(2, 2, 16), **kw)]  # noqa: B023
            chunk = {x: y for x, y in kw.items() if x != "seen"}
            if name != "seen":
                calls.append(lambda: kernels.chunk_attend(q, rows, scale=0.1, out=state[:768].view(torch.bfloat16).view(2, 4, 3, 64), **chunk))  # noqa: B023
                calls.append(lambda: kernels.chunk_attend(q, rows, scale=0.1, lse=state[:24].view(torch.float32).view(2, 4, 3), **chunk))  # noqa: B023
                moved = {"starts" if x == "lengths" else x: y for x, y in chunk.items()}
                calls.append(lambda: kernels.rotate_append(rows, q, k, k, out=state[:768].view(torch.bfloat16).view(2, 4, 3, 64), **moved))  # noqa: B023
            if name in ("pages", "lengths"):
                calls.append(lambda: kernels.evict_rows(rows, sums, state[:64].view(2, 2, 16), keep=4, **{x: kw[x] for x in ("pages", "lengths")}))  # noqa: B023
            for call in calls:
                launched.clear()
                call()
                (got,) = launched
                there = [x for x in got if lo + 24 <= x < lo + 32]
                assert not there and (one + 1 in got.values()), (name, among)
                assert among or mine.data_ptr() in got, name


def test_a_page_table_among_rows_that_an_eviction_moves_is_copied_first(monkeypatch: pytest.MonkeyPatch, kernels) -> None:  # noqa: ANN001
    import torch

    tables = []
    monkeypatch.setattr(kernels, "_launch", lambda _, fn, *args: tables.extend(x.table for x in args if hasattr(x, "table")) or 0)
    pool = torch.zeros((2, 4, 2, 16, 64), dtype=torch.bfloat16)
    rows = kernels.dense_rows(pool[0], pool[1])
    table = pool.view(torch.int32).flatten()[32:34].view(2, 1)
    kernels.evict_rows(rows, torch.zeros((2, 2, 16)), torch.zeros((2, 2, 16), dtype=torch.int32), keep=4, tokens=16, pages=table)
    assert len(tables) == 1 and tables[0] != table.data_ptr()


@pytest.mark.parametrize(("n_q", "tokens"), [(1 << 29, 1), ((1 << 28) + 16, 1), (1 << 22, 511)])
def test_rotations_of_more_threads_than_a_launch_has_are_refused(n_q: int, tokens: int) -> None:
    """Few tokens of many heads: sixteen heads a workgroup of up to 256 threads, 2^24 of which are 2^32 threads."""
    change = {"desc": {"n_seqs": 1, "n_q": n_q, "n_kv": 1, "new_tokens": tokens}, "strides": (n_q * 64 * tokens, 64 * tokens, 64),
              "rows": {"tokens": 1024, "v": 1 << 40, "seq_stride": 1 << 16, "head_stride": 1 << 16}}
    assert "in one call" in _call("rotate", change)
