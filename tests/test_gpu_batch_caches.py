"""The 8-bit cache and the batch over a shared prefix, under a transformers Llama stack on the GPU.

The 8-bit cache's model attends what the cache holds, so its reference is the same model over a dense cache whose rows are
the 64-bit oracle's codes read back; the batch's reference is each sequence alone over a dense cache that holds the prefix and its
own tokens. Both sides run the same float16 model; their attention sums in another order and rounds its weights to float16,
so log-probabilities agree within 2e-2, as between the tiers."""

from __future__ import annotations

import copy

import numpy as np
import pytest
import torch

from lazykv_amd.cache import Decoded
from oracle import reference as R
from oracle import rows as O

pytestmark = pytest.mark.gpu

TOL = 2e-2


@pytest.fixture(scope="module")
def tiny():  # noqa: ANN201
    from transformers import LlamaConfig, LlamaForCausalLM

    from lazykv_amd.attention import IMPLEMENTATION_NAME, install

    install()
    torch.manual_seed(0)
    cfg = LlamaConfig(hidden_size=256, intermediate_size=512, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                      vocab_size=512, max_position_embeddings=4096)
    with torch.device("cuda"):
        model = LlamaForCausalLM(copy.deepcopy(cfg))
    model.set_attn_implementation(IMPLEMENTATION_NAME)
    return cfg, model.to(dtype=torch.float16).eval()


def _ids(seed: int, *shape: int) -> torch.Tensor:
    return torch.randint(0, 512, shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def _forward(model, cache, ids: torch.Tensor, **kw) -> torch.Tensor:  # noqa: ANN001, ANN003
    with torch.inference_mode():
        out = model(input_ids=ids, past_key_values=cache, use_cache=True, **kw)
    return torch.log_softmax(out.logits.float(), -1)


def _coded(x: torch.Tensor) -> torch.Tensor:
    values = O.mx_decode(*O.mx_encode(x.double().cpu().numpy(), "f16"))
    return torch.from_numpy(values).to(x.dtype).to(x.device)


def _rounded_cache(layers: int, cap: int):  # noqa: ANN202
    """A dense cache that holds what the 8-bit cache holds, in the model dtype."""
    from lazykv_amd.cache import DenseLayer, FullGPUCache

    class Rounded(DenseLayer):
        def _write(self, k, v, a, b):  # noqa: ANN001, ANN202
            super()._write(_coded(k), _coded(v), a, b)

    class RoundedCache(FullGPUCache):
        layer_type = Rounded

    return RoundedCache(layers, cap)


@pytest.mark.parametrize("chunk", [7, 64, 1])
def test_8_bit_cache_decodes_like_a_dense_cache_of_its_rows(tiny, chunk: int) -> None:  # noqa: ANN001
    """Prefill in chunks (of one token too: the decode path), then 20 tokens, then a turn and 5 more."""
    from lazykv_amd.cache import MXFP8Cache

    cfg, model = tiny
    prompt = 100 if chunk > 1 else 9
    ids = _ids(1, 1, prompt + 20 + 12 + 5)
    mx, ref = MXFP8Cache(cfg.num_hidden_layers, 256), _rounded_cache(cfg.num_hidden_layers, 256)
    spans = [(a, min(prompt, a + chunk)) for a in range(0, prompt, chunk)] + [(i, i + 1) for i in range(prompt, prompt + 20)]
    spans += [(prompt + 20, prompt + 32)] + [(i, i + 1) for i in range(prompt + 32, prompt + 37)]
    for a, b in spans:
        got, want = _forward(model, mx, ids[:, a:b]), _forward(model, ref, ids[:, a:b])
        assert float((got - want).abs().max()) < TOL, (a, b)
    n = ids.shape[1]
    for ours, dense in zip(mx.layers, ref.layers):
        assert ours.get_seq_length() == n
        k, v = ours.dense()
        # The first layer's rows come from the same hidden states: the same codes.
        if ours is mx.layers[0]:
            assert torch.equal(k, dense.keys[:, :, :n]) and torch.equal(v, dense.values[:, :, :n])
    s, full = mx.stats(), ref.stats()
    assert s.seq_len == n and s.gpu_resident_kv_bytes * 64 == full.gpu_resident_kv_bytes * 33
    assert s.gpu_allocated_kv_bytes == sum(layer.codes.numel() + layer.scales.numel() for layer in mx.layers)


def test_8_bit_cache_truncates_and_resets(tiny) -> None:  # noqa: ANN001
    from lazykv_amd.cache import MXFP8Cache

    cfg, model = tiny
    ids = _ids(2, 1, 40)
    cache = MXFP8Cache(cfg.num_hidden_layers, 64)
    _forward(model, cache, ids[:, :30])
    first = _forward(model, cache, ids[:, 30:31])
    cache.truncate(30)
    _forward(model, cache, ids[:, 35:36])
    cache.truncate(30)
    assert torch.equal(first, _forward(model, cache, ids[:, 30:31]))
    with pytest.raises(RuntimeError, match="full"):
        _forward(model, cache, _ids(3, 1, 40))


def _follow(cache, ref) -> None:  # noqa: ANN001
    """Has `ref`'s tiers attend the blocks that `cache`'s choose, which must be their own choice up to near ties: the two hold queries
    and keys that differ by roundings, and a swap at a tie moves an output by any amount. With Delta the largest difference of
    the two bounds (64 bits) and e the float32 bound's error, a block that `cache` chooses has a bound of at least its K-th - e
    there, so of at least the K-th - e - 2 Delta in `ref` (the K-th largest moves by Delta at most)."""
    chosen = {}
    ours = cache.select

    def bound(tier, query):  # noqa: ANN001, ANN202
        n, _ = tier.candidates()
        lo, hi = (x.double().cpu().numpy().reshape(tier.h, -1, tier.d)[:, 1:n] for x in (tier.kmin, tier.kmax))
        q = query.double().cpu().numpy().reshape(-1, tier.d)
        return R.quest_bound(q, lo, hi), float(np.abs(q).max() * np.maximum(np.abs(lo), np.abs(hi)).sum(-1).max()) * 2.0**-19

    def record(layer, query, *args):  # noqa: ANN001, ANN002, ANN202
        tier = cache.tiers.get(layer)
        if tier is not None:
            chosen[layer] = (tier.rank(query).clone(), bound(tier, query))
        return ours(layer, query, *args)

    def follow(layer, query, key=None, value=None, scaling=None):  # noqa: ANN001, ANN202
        tier = ref.tiers.get(layer)
        if tier is None:
            return None
        idx, (theirs, _) = chosen[layer]
        own, err = bound(tier, query)
        for j in range(tier.h):
            assert R.selection_ok(idx[j].cpu().numpy() - 1, own[j], tier.k, abs_err=err + 2 * float(np.abs(theirs - own).max()))[0], (layer, j)
        out, lse = tier.decode(query, scaling, idx=idx)
        return Decoded(out.view(1, -1, 1, tier.d), lse.view(1, -1))

    cache.select, ref.select = record, follow


def test_8_bit_dense_layers_of_a_tiered_cache(tiny) -> None:  # noqa: ANN001
    """A tier whose dense layers stay in 8 bits, from a layer-major prefill and from a prefilled cache: the same tier either way as
    from dense layers of those rows, and the same decode."""
    from lazykv_amd.cache import MXFP8Cache
    from lazykv_amd.tiered import TieredCache
    from lazykv_amd.tiered_prefill import tiered_prefill

    cfg, model = tiny
    prompt, bs, k = 200, 8, 6
    ids = _ids(4, 1, prompt + 12)
    for chunk in (64, 199):  # the second leaves a last chunk of one token
        got = tiered_prefill(model, ids[:, :prompt], chunk, k, bs, 512, dense_layers=1, dense_quant="mxfp8", fetch="resident")
        assert isinstance(got.cache.full, MXFP8Cache) and got.cache.full.layers[0].get_seq_length() == prompt
        ref = _rounded_cache(cfg.num_hidden_layers, 512)
        # The reference: the same prefill over rounded dense rows in the first layer only.
        for layer in ref.layers[1:]:
            layer._write = super(type(layer), layer)._write
        for a in range(0, prompt, chunk):
            _forward(model, ref, ids[:, a : min(prompt, a + chunk)])
        tier = TieredCache(ref, k, bs, 512, dense_layers=1, fetch="resident")
        _follow(got.cache, tier)
        for i in range(prompt, prompt + 12):
            a, b = (_forward(model, c, ids[:, i : i + 1], **c.model_kwargs()) for c in (got.cache, tier))
            assert float((a - b).abs().max()) < TOL, i
    mx = MXFP8Cache(cfg.num_hidden_layers, 512)
    _forward(model, mx, ids[:, :prompt])
    tier = TieredCache(mx, k, bs, 512, dense_layers=1, fetch="resident")
    keys, values = mx.layers[1].dense()
    assert torch.equal(tier.tiers[1].store[3, :, 0], keys[0, :, 3 * bs : 4 * bs]) and torch.equal(tier.tiers[1].store[3, :, 1], values[0, :, 3 * bs : 4 * bs])
    _forward(model, tier, ids[:, prompt : prompt + 1], **tier.model_kwargs())


def _alone(model, cfg, prefix: torch.Tensor, own: list[torch.Tensor]) -> list[torch.Tensor]:  # noqa: ANN001
    """Each sequence over a dense cache of its own: log-probabilities of every own token."""
    from lazykv_amd.cache import FullGPUCache

    got = []
    for ids in own:
        cache = FullGPUCache(cfg.num_hidden_layers, 512)
        _forward(model, cache, prefix)
        got.append(torch.cat([_forward(model, cache, ids[None, i : i + 1])[0] for i in range(len(ids))]) if len(ids) else None)
    return got


@pytest.mark.parametrize(("seqs", "prompt"), [(1, 50), (3, 130), (20, 77)])
def test_a_batch_decodes_like_its_sequences_alone(tiny, seqs: int, prompt: int) -> None:  # noqa: ANN001
    from lazykv_amd.cache import FullGPUCache, SharedPrefixCache

    cfg, model = tiny
    prefix, own = _ids(5, 1, prompt), _ids(6, seqs, 10)
    full = FullGPUCache(cfg.num_hidden_layers, 512)
    _forward(model, full, prefix)
    cache = SharedPrefixCache(full, seqs, 16)
    got = [_forward(model, cache, own[:, i : i + 1], **cache.model_kwargs())[:, 0] for i in range(10)]
    want = _alone(model, cfg, prefix, list(own))
    for b in range(seqs):
        assert float((torch.stack([x[b] for x in got]) - want[b]).abs().max()) < TOL, b
    assert cache.get_seq_length() == prompt + 10 and cache.lengths() == [10] * seqs
    assert full.layers[0].get_seq_length() == prompt  # the prefix is not written to
    s = cache.stats()
    own_bytes = 3 * 2 * seqs * 2 * 16 * 64 * 2
    assert s.gpu_allocated_kv_bytes == full.stats().gpu_allocated_kv_bytes + own_bytes
    assert s.gpu_resident_kv_bytes == full.stats().gpu_resident_kv_bytes + own_bytes * 10 // 16


@pytest.mark.parametrize("prefix_quant", [False, True])
@pytest.mark.parametrize("quant", [None, "mxfp8"])
def test_questions_of_different_lengths_about_one_document(tiny, prefix_quant: bool, quant: str | None) -> None:  # noqa: ANN001
    """Questions padded on the right, cut to their lengths, answered token by token; then one sequence leaves and another goes on
    twice. Against each sequence alone over a dense cache of the rows that the batch holds."""
    from lazykv_amd.cache import FullGPUCache, MXFP8Cache, SharedPrefixCache

    cfg, model = tiny
    prompt, lens = 90, [5, 12, 1, 8]
    prefix, questions, answers = _ids(7, 1, prompt), _ids(8, 4, 12), _ids(9, 4, 6)
    full = (MXFP8Cache if prefix_quant else FullGPUCache)(cfg.num_hidden_layers, 256)
    _forward(model, full, prefix)
    cache = SharedPrefixCache(full, 4, 32, quant=quant)
    got = _forward(model, cache, questions, position_ids=cache.positions(12), **cache.model_kwargs())
    first = [got[b, n - 1] for b, n in enumerate(lens)]
    cache.truncate(lens)
    assert cache.lengths() == lens and cache.get_seq_length() == prompt + 12
    rows = [[x] for x in first]
    for i in range(3):
        step = _forward(model, cache, answers[:, i : i + 1], position_ids=cache.positions(), **cache.model_kwargs())
        for b in range(4):
            rows[b].append(step[b, 0])
    order = [3, 1, 3]
    cache.keep(order)
    assert cache.lengths() == [lens[b] + 3 for b in order]
    rows = [list(rows[b]) for b in order]
    for i in range(3, 6):
        step = _forward(model, cache, answers[order, i : i + 1], position_ids=cache.positions(), **cache.model_kwargs())
        for j in range(3):
            rows[j].append(step[j, 0])

    class Mixed(FullGPUCache):  # a dense cache that rounds the prefix's rows, the own ones, or both as the batch's caches do
        pass

    for j, b in enumerate(order):
        alone = Mixed(cfg.num_hidden_layers, 256)
        for layer in alone.layers:
            def write(k, v, a, e, layer=layer, plain=layer._write):  # noqa: ANN001, ANN202
                rounded = prefix_quant if a < prompt else quant == "mxfp8"
                plain(*((_coded(k), _coded(v)) if rounded else (k, v)), a, e)
            layer._write = write
        _forward(model, alone, prefix)
        want = [_forward(model, alone, questions[b : b + 1, : lens[b]])[0, -1]]
        want += [_forward(model, alone, answers[b : b + 1, i : i + 1])[0, 0] for i in range(6)]
        assert float((torch.stack(rows[j]) - torch.stack(want)).abs().max()) < TOL, b
    assert torch.equal(torch.stack(rows[0]), torch.stack(rows[2]))  # the same sequence twice


def test_a_batch_alternates_questions_and_answers(tiny) -> None:  # noqa: ANN001
    """A second forward of several tokens behind ragged answers."""
    from lazykv_amd.cache import FullGPUCache, SharedPrefixCache

    cfg, model = tiny
    prefix, ids = _ids(10, 1, 33), _ids(11, 2, 20)
    full = FullGPUCache(cfg.num_hidden_layers, 128)
    _forward(model, full, prefix)
    cache = SharedPrefixCache(full, 2, 40)
    _forward(model, cache, ids[:, :6], **cache.model_kwargs())
    cache.truncate([6, 2])
    got = _forward(model, cache, ids[:, 6:11], position_ids=cache.positions(5), **cache.model_kwargs())
    last = _forward(model, cache, ids[:, 11:12], position_ids=cache.positions(), **cache.model_kwargs())
    for b, n in enumerate((6, 2)):
        alone = FullGPUCache(cfg.num_hidden_layers, 128)
        _forward(model, alone, prefix)
        _forward(model, alone, ids[b : b + 1, :n])
        want = _forward(model, alone, ids[b : b + 1, 6:11])
        assert float((got[b] - want[0]).abs().max()) < TOL
        assert float((last[b] - _forward(model, alone, ids[b : b + 1, 11:12])[0]).abs().max()) < TOL


def test_decode_steps_never_wait_for_the_device(tiny) -> None:  # noqa: ANN001
    from lazykv_amd.cache import FullGPUCache, SharedPrefixCache

    cfg, model = tiny
    full = FullGPUCache(cfg.num_hidden_layers, 128)
    _forward(model, full, _ids(12, 1, 40))
    cache = SharedPrefixCache(full, 3, 16, quant="mxfp8")
    ids, pos = _ids(13, 3, 1), torch.full((3, 1), 40, device="cuda")
    cache.layers[0].prefix_rows  # made when the cache was
    _forward(model, cache, ids, position_ids=pos, **cache.model_kwargs())
    torch.cuda.synchronize()
    q = torch.randn((3, 4, 1, 64), device="cuda").half()
    kv = torch.randn((2, 3, 2, 1, 64), device="cuda").half()
    torch.cuda.set_sync_debug_mode("error")
    try:
        for layer in range(cfg.num_hidden_layers):
            cache.update(kv[0], kv[1], layer)
            got = cache.select(layer, q)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    torch.cuda.synchronize()
    assert got.out.shape == (3, 4, 1, 64) and got.lse.shape == (3, 4) and bool(got.out.isfinite().all())


def test_refusals(tiny) -> None:  # noqa: ANN001
    from lazykv_amd import snapshot
    from lazykv_amd.attention import attend, lazykv_attention_forward
    from lazykv_amd.cache import FullGPUCache, MXFP8Cache, MXFP8Layer, SharedPrefixCache
    from lazykv_amd.selection import QuestView
    from lazykv_amd.tiered import TieredCache
    from lazykv_amd.tiered_prefill import tiered_prefill

    cfg, model = tiny
    full = FullGPUCache(cfg.num_hidden_layers, 64)
    with pytest.raises(ValueError, match="prefilled"):
        SharedPrefixCache(full, 2, 8)
    _forward(model, full, _ids(14, 1, 20))
    for bad in (dict(n_seqs=0, max_new=4), dict(n_seqs=2, max_new=0), dict(n_seqs=2, max_new=4, quant="int4")):
        with pytest.raises(ValueError):
            SharedPrefixCache(full, **bad)
    cache = SharedPrefixCache(full, 2, 3)
    with pytest.raises(ValueError, match="2 sequences"):
        _forward(model, cache, _ids(15, 3, 1), **cache.model_kwargs())
    with pytest.raises(RuntimeError, match="full"):
        _forward(model, cache, _ids(15, 2, 4), **cache.model_kwargs())
    for cut in (1, [0], [0, 1]):
        with pytest.raises(ValueError, match="cut"):
            cache.truncate(cut)
    for keep in ([], [2], [-1]):
        with pytest.raises(ValueError):
            cache.keep(keep)
    cache.update(torch.zeros((2, 2, 1, 64), dtype=torch.float16, device="cuda"), torch.zeros((2, 2, 1, 64), dtype=torch.float16, device="cuda"), 0)
    with pytest.raises(RuntimeError, match="between forwards"):
        cache.truncate(0)
    q = torch.zeros((2, 4, 1, 64), dtype=torch.float16, device="cuda")
    kv = torch.zeros((2, 2, 5, 64), dtype=torch.float16, device="cuda")
    with pytest.raises(RuntimeError, match="batch size 1"):
        lazykv_attention_forward(model, q, kv, kv, None)
    mx = MXFP8Cache(cfg.num_hidden_layers, 64)
    _forward(model, mx, _ids(16, 1, 20))
    with pytest.raises(ValueError, match="8-bit"):
        QuestView(mx, 1, 4, dense_layers=1)
    k, v = mx.layers[0].update(kv[:1, :, :1], kv[:1, :, :1])
    with pytest.raises(ValueError, match="one token"):
        attend(q[:1].expand(1, 4, 2, 64), k, v, None)
    with pytest.raises(ValueError, match="head_dim"):
        MXFP8Layer(8).update(kv[:1, :, :, :32], kv[:1, :, :, :32])
    with pytest.raises(ValueError, match="float16 or bfloat16"):
        MXFP8Layer(8).update(kv[:1].float(), kv[:1].float())
    with pytest.raises(ValueError, match="precision"):
        tiered_prefill(model, _ids(17, 1, 40), 16, 2, 8, 64, dense_layers=1, dense_quant="int8")
    mx.truncate(20)
    tier = TieredCache(mx, 1, 4, 64, dense_layers=1, fetch="resident")
    with pytest.raises(ValueError, match="8-bit dense"):
        snapshot.save(tier, torch.zeros(512), "/nonexistent/x.lkv")


def test_eight_bit_layers_hold_rows_independent_of_how_they_came() -> None:
    from lazykv_amd.cache import MXFP8Layer

    gen = torch.Generator(device="cuda").manual_seed(1)
    kv = torch.randn((2, 1, 4, 50, 128), device="cuda", generator=gen).bfloat16()
    a, b = MXFP8Layer(64), MXFP8Layer(64)
    a.update(kv[0], kv[1])
    for i in range(50):
        b.update(kv[0, :, :, i : i + 1], kv[1, :, :, i : i + 1])
    assert torch.equal(a.codes.view(torch.uint8), b.codes.view(torch.uint8)) and torch.equal(a.scales, b.scales)
    want = [O.mx_decode(*O.mx_encode(x.double().cpu().numpy(), "bf16")) for x in kv]
    for x, y in zip(a.dense(), want):
        assert np.array_equal(x.double().cpu().numpy(), y)


def test_a_forward_without_the_selector_is_refused(tiny) -> None:  # noqa: ANN001
    """With another attention function too, which would attend the new token alone."""
    from lazykv_amd.attention import IMPLEMENTATION_NAME
    from lazykv_amd.cache import FullGPUCache, SharedPrefixCache

    cfg, model = tiny
    full = FullGPUCache(cfg.num_hidden_layers, 64)
    _forward(model, full, _ids(20, 1, 20))
    cache = SharedPrefixCache(full, 1, 8)
    model.set_attn_implementation("sdpa")
    try:
        with pytest.raises(RuntimeError, match="model_kwargs"):
            _forward(model, cache, _ids(21, 1, 1), position_ids=cache.positions())
    finally:
        model.set_attn_implementation(IMPLEMENTATION_NAME)
    cache.reset()
    assert bool(_forward(model, cache, _ids(21, 1, 1), **cache.model_kwargs()).isfinite().all()) and cache.lengths() == [1]


def test_a_prefix_that_was_cut_and_one_that_is_not_dense_are_refused(tiny) -> None:  # noqa: ANN001
    from lazykv_amd.cache import FullGPUCache, SharedPrefixCache
    from lazykv_amd.tiered import TieredCache

    cfg, model = tiny
    full = FullGPUCache(cfg.num_hidden_layers, 64)
    _forward(model, full, _ids(22, 1, 20))
    cache = SharedPrefixCache(full, 2, 8)
    full.truncate(19)
    with pytest.raises(RuntimeError, match="cut to 19"):
        _forward(model, cache, _ids(23, 2, 1), **cache.model_kwargs())
    _forward(model, full, _ids(24, 1, 1))
    tier = TieredCache(full, 1, 4, 64, dense_layers=1, fetch="resident")
    with pytest.raises(ValueError, match="densely"):
        SharedPrefixCache(tier, 2, 8)


@pytest.mark.parametrize("quant", [None, "mxfp8"])
def test_a_batch_is_reset_and_reordered_as_transformers_caches_are(tiny, quant: str | None) -> None:  # noqa: ANN001
    from lazykv_amd.cache import FullGPUCache, SharedPrefixCache

    cfg, model = tiny
    full = FullGPUCache(cfg.num_hidden_layers, 64)
    _forward(model, full, _ids(25, 1, 33))
    cache = SharedPrefixCache(full, 3, 8, quant=quant)
    ids, order = _ids(26, 3, 2), torch.tensor([2, 0, 2], device="cuda")
    first = _forward(model, cache, ids[:, :1], **cache.model_kwargs())
    cache.reorder_cache(order)
    got = _forward(model, cache, ids[:, 1:], **cache.model_kwargs())
    cache.reset()
    assert cache.lengths() == [0, 0, 0] and cache.get_seq_length() == 33
    assert torch.equal(_forward(model, cache, ids[:, :1], **cache.model_kwargs()), first)
    cache.reset()
    _forward(model, cache, ids[order][:, :1], **cache.model_kwargs())
    assert torch.equal(_forward(model, cache, ids[:, 1:], **cache.model_kwargs()), got)
    cache.batch_select_indices(torch.tensor([1], device="cuda"))
    assert cache.lengths() == [2] and cache.n_seqs == 1
    for layer in cache.layers:
        for call in (layer.reset, lambda layer=layer: layer.reorder_cache(order)):
            with pytest.raises(RuntimeError, match="through its SharedPrefixCache"):
                call()
