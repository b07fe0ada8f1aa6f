"""The 8-bit cache and the batch over a shared prefix at the edges of what their documentation allows, on the GPU."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tiny():  # noqa: ANN201
    from transformers import LlamaConfig, LlamaForCausalLM

    from lazykv_amd.attention import IMPLEMENTATION_NAME, install

    install()
    torch.manual_seed(0)
    cfg = LlamaConfig(hidden_size=256, intermediate_size=512, num_hidden_layers=3, num_attention_heads=4, num_key_value_heads=2, head_dim=64,
                      vocab_size=512, max_position_embeddings=4096)
    with torch.device("cuda"):
        model = LlamaForCausalLM(cfg)
    model.set_attn_implementation(IMPLEMENTATION_NAME)
    return model.to(dtype=torch.float16).eval()


def _ids(seed: int, *shape: int) -> torch.Tensor:
    return torch.randint(0, 512, shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def _forward(model, cache, ids: torch.Tensor, **kw) -> torch.Tensor:  # noqa: ANN001, ANN003
    with torch.inference_mode():
        return model(input_ids=ids, past_key_values=cache, use_cache=True, **kw).logits


def _prefilled(model, tokens: int, cap: int = 256, seed: int = 1):  # noqa: ANN001, ANN202
    from lazykv_amd.cache import FullGPUCache

    full = FullGPUCache(3, cap)
    _forward(model, full, _ids(seed, 1, tokens))
    return full


def test_gradients_are_refused_not_dropped(tiny) -> None:  # noqa: ANN001
    """Inputs, caches and outputs that autograd follows, in both modes; under no_grad, and without a gradient, the calls go on."""
    import torch.autograd.forward_ad as fwd

    from lazykv_amd import kernels
    from lazykv_amd.cache import MXFP8Cache, SharedPrefixCache

    gen = torch.Generator(device="cuda").manual_seed(2)
    kv = torch.randn((2, 1, 2, 5, 64), device="cuda", generator=gen).half()
    q = torch.randn((1, 4, 64), device="cuda", generator=gen).half()
    leaf = lambda x: x.clone().requires_grad_()  # noqa: E731
    codes, scales = kernels.mx_empty(1, 2, 5, 64, "cuda")
    rows = kernels.mx_rows(codes, scales, torch.float16)
    dense = kernels.dense_rows(kv[0], kv[1])
    followed = leaf(kv)
    calls = [
        lambda: kernels.append_rows(rows, leaf(kv[0]), kv[1]), lambda: kernels.append_rows(rows, kv[0], leaf(kv[1])),
        lambda: kernels.append_rows(kernels.dense_rows(followed[0], followed[1]), kv[0], kv[1]),
        lambda: kernels.read_rows(rows, 0, 5, out=(leaf(kv[0]), kv[1].clone())),
        lambda: kernels.shared_decode(leaf(q), scale=0.1, own=dense, own_tokens=5),
        lambda: kernels.shared_decode(q, scale=0.1, prefix=kernels.dense_rows(followed[0], followed[1]), prefix_tokens=5),
        lambda: kernels.shared_decode(q, scale=0.1, own=dense, own_tokens=5, out=leaf(q)),
    ]
    for call in calls:
        with pytest.raises(RuntimeError, match="no gradient"):
            call()
        with torch.no_grad():
            call()
    with fwd.dual_level():
        kernels.append_rows(rows, kv[0], kv[1])
        with pytest.raises(RuntimeError, match="tangents"):
            kernels.append_rows(rows, fwd.make_dual(kv[0].clone(), kv[1].clone()), kv[1])
        with pytest.raises(RuntimeError, match="tangents"):
            kernels.shared_decode(fwd.make_dual(q.clone(), q.clone()), scale=0.1, own=dense, own_tokens=5)
    # A model whose weights have gradients.
    mx = MXFP8Cache(3, 64)
    with pytest.raises(RuntimeError, match="no gradient"):
        tiny(input_ids=_ids(3, 1, 9), past_key_values=mx, use_cache=True)
    batch = SharedPrefixCache(_prefilled(tiny, 20), 2, 8)
    with pytest.raises(RuntimeError, match="no gradient"):
        tiny(input_ids=_ids(3, 2, 1), past_key_values=batch, use_cache=True, **batch.model_kwargs())


def test_writes_are_seen_by_graphs_that_saved_what_they_change() -> None:
    """A backward pass that needs a tensor as it was fails, as after any write in place, instead of going on with other values."""
    from lazykv_amd import kernels

    gen = torch.Generator(device="cuda").manual_seed(4)
    w = torch.randn((1, 2, 5, 64), device="cuda", generator=gen).half().requires_grad_()
    new = torch.ones((1, 2, 5, 64), device="cuda").half()
    q = torch.ones((1, 4, 64), device="cuda").half()
    store = torch.zeros((2, 1, 2, 5, 64), device="cuda").half()
    codes, scales = kernels.mx_empty(1, 2, 5, 64, "cuda")
    mx = kernels.mx_rows(codes, scales, torch.float16)
    out = (torch.zeros_like(store[0]), torch.zeros_like(store[0]))
    got, lse = torch.ones((1, 4, 64), device="cuda").half(), torch.ones((1, 4), device="cuda")
    for saved, write in (
        (store[0], lambda: kernels.append_rows(kernels.dense_rows(store[0], store[1]), new, new)),
        (out[1], lambda: kernels.read_rows(mx, 0, 5, out=out)),
        (got, lambda: kernels.shared_decode(q, scale=1.0, own=mx, own_tokens=5, out=got, lse=lse)),
    ):
        y = (w[:, :1, :4] * saved.view(1, -1, 4, 64)[:, :1]).sum() if saved is got else (w * saved).sum()
        with torch.no_grad():
            write()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()


@pytest.mark.parametrize("cut", ["reset", "truncate", "layer"])
def test_a_prefix_that_was_cut_and_filled_again_is_noticed(tiny, cut: str) -> None:  # noqa: ANN001
    """Another prompt of the same length in the prefix's place: the batch would answer about the wrong one."""
    from lazykv_amd.cache import SharedPrefixCache

    full = _prefilled(tiny, 30)
    batch = SharedPrefixCache(full, 2, 8)
    _forward(tiny, batch, _ids(5, 2, 1), **batch.model_kwargs())
    if cut == "reset":
        for layer in full.layers:
            layer.reset()
        _forward(tiny, full, _ids(6, 1, 30))
    elif cut == "truncate":
        full.truncate(29)
        _forward(tiny, full, _ids(6, 1, 1))
    else:
        full.layers[2].truncate(0)
        with torch.inference_mode():
            full.layers[2].store(*(torch.zeros((1, 2, 30, 64), device="cuda").half() for _ in range(2)))
    assert full.get_seq_length() == 30
    with pytest.raises(RuntimeError, match="the prefix was cut"):
        _forward(tiny, batch, _ids(5, 2, 1), **batch.model_kwargs())
    fresh = SharedPrefixCache(full, 2, 8)  # a batch over what is there now
    assert bool(_forward(tiny, fresh, _ids(5, 2, 1), **fresh.model_kwargs()).isfinite().all())


def test_a_prefix_may_grow_and_be_cut_back(tiny) -> None:  # noqa: ANN001
    """Tokens behind the batch's prefix come and go without a change to it, also under a second batch over more of them."""
    from lazykv_amd.cache import SharedPrefixCache

    full, ids = _prefilled(tiny, 30), _ids(7, 2, 2)
    batch = SharedPrefixCache(full, 2, 8)
    _forward(tiny, batch, ids[:, :1], **batch.model_kwargs())
    want = _forward(tiny, batch, ids[:, 1:], **batch.model_kwargs())
    batch.truncate(1)
    _forward(tiny, full, _ids(8, 1, 5))
    longer = SharedPrefixCache(full, 2, 8)
    full.truncate(30)
    assert torch.equal(_forward(tiny, batch, ids[:, 1:], **batch.model_kwargs()), want)
    with pytest.raises(RuntimeError, match="cut to 30"):
        _forward(tiny, longer, ids[:, :1], **longer.model_kwargs())


class _Stop(Exception):
    pass


def _stop_at(model, layer: int, after: bool):  # noqa: ANN001, ANN202
    """A forward that raises at a layer: before its attention has begun, or after it."""
    def hook(*args: object) -> None:
        raise _Stop

    module = model.model.layers[layer].self_attn
    return module.register_forward_hook(hook) if after else module.register_forward_pre_hook(hook)


@pytest.mark.parametrize("n", [1, 3])
@pytest.mark.parametrize(("layer", "after"), [(0, False), (0, True), (1, False), (2, False), (2, True)])
def test_a_forward_that_raised_is_rolled_back(tiny, layer: int, after: bool, n: int) -> None:  # noqa: ANN001
    """Behind ragged lengths, one token or several; the batch then goes on as if that forward had not been. Without the rollback
    another forward is refused where it would leave layers with tokens of both."""
    from lazykv_amd.cache import SharedPrefixCache

    batch = SharedPrefixCache(_prefilled(tiny, 25), 3, 32, quant="mxfp8")
    _forward(tiny, batch, _ids(9, 3, 4), **batch.model_kwargs())
    batch.truncate([4, 1, 2])
    _forward(tiny, batch, _ids(10, 3, 1), position_ids=batch.positions(), **batch.model_kwargs())
    call = dict(position_ids=batch.positions(n), **batch.model_kwargs())
    want = _forward(tiny, batch, _ids(11, 3, n), **call)
    batch.truncate([5, 2, 3])
    hook = _stop_at(tiny, layer, after)
    try:
        with pytest.raises(_Stop):
            _forward(tiny, batch, _ids(12, 3, n), **call)
    finally:
        hook.remove()
    if (layer, after) not in ((0, False), (2, True)):  # nothing written yet, everything attended
        with pytest.raises(RuntimeError, match="rollback"):
            batch.truncate([5, 2, 3])
        with pytest.raises(RuntimeError, match="rollback"):
            _forward(tiny, batch, _ids(12, 3, n), **call)
    batch.rollback()
    if (layer, after) == (2, True):  # ended: taken back as any other
        batch.truncate([5, 2, 3])
    assert batch.lengths() == [5, 2, 3] and batch.get_seq_length() == 30
    assert torch.equal(_forward(tiny, batch, _ids(11, 3, n), **call), want)
    batch.rollback()  # of nothing
    assert batch.lengths() == [5 + n, 2 + n, 3 + n]


@pytest.mark.parametrize("by_length", [False, True])
def test_a_layers_attention_that_raised_is_rolled_back(tiny, by_length: bool) -> None:  # noqa: ANN001
    """The last layer's tokens written, its attention refused: every layer has them, and none is left after the rollback, or after
    lengths without them are set."""
    from lazykv_amd.cache import SharedPrefixCache

    batch = SharedPrefixCache(_prefilled(tiny, 25), 2, 8)
    kv = torch.randn((2, 2, 2, 1, 64), device="cuda").half()
    q = torch.randn((2, 4, 1, 64), device="cuda").half()
    for layer in range(3):
        batch.update(kv[0], kv[1], layer)
        if layer < 2:
            batch.select(layer, q)
    with pytest.raises(ValueError, match="sequences"):
        batch.select(2, q[:1])
    if by_length:
        batch.truncate(0)
    else:
        batch.rollback()
    assert batch.lengths() == [0, 0]
    assert bool(_forward(tiny, batch, _ids(13, 2, 1), **batch.model_kwargs()).isfinite().all()) and batch.lengths() == [1, 1]


@pytest.mark.parametrize("ragged", [False, True])
def test_the_documented_loop_never_waits_for_the_device(tiny, ragged: bool) -> None:  # noqa: ANN001
    """Whole forwards of one token, with the positions that the cache gives."""
    from lazykv_amd.cache import SharedPrefixCache

    batch = SharedPrefixCache(_prefilled(tiny, 40), 3, 16)
    _forward(tiny, batch, _ids(14, 3, 4), position_ids=batch.positions(4), **batch.model_kwargs())
    batch.truncate([4, 2, 3] if ragged else 3)
    ids = _ids(15, 3, 1)
    _forward(tiny, batch, ids, position_ids=batch.positions(), **batch.model_kwargs())
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        for _ in range(3):
            ids = _forward(tiny, batch, ids, position_ids=batch.positions(), **batch.model_kwargs())[:, -1:].argmax(-1)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    lengths = [8, 6, 7] if ragged else [7, 7, 7]
    assert batch.lengths() == lengths
    for n in (1, 5):
        got = batch.positions(n)
        assert got.dtype == torch.int64 and got.is_contiguous()
        assert got.tolist() == [[40 + m + t for t in range(n)] for m in lengths]


def test_a_forward_of_several_tokens_leaves_no_buffer(tiny) -> None:  # noqa: ANN001
    """The prefix's copy in the model dtype is counted while a forward holds it, and goes with its last layer, or with a rollback."""
    from lazykv_amd.cache import SharedPrefixCache

    batch = SharedPrefixCache(_prefilled(tiny, 200), 2, 32)
    call = dict(position_ids=batch.positions(3), **batch.model_kwargs())
    own = 3 * 2 * 2 * 2 * 32 * 64 * 2  # layers, keys and values, sequences, heads, tokens, channels, bytes
    full = batch.full.stats().gpu_allocated_kv_bytes
    seen = []
    hook = tiny.model.layers[0].register_forward_hook(lambda *a: seen.append(batch.stats().gpu_allocated_kv_bytes))
    try:
        _forward(tiny, batch, _ids(16, 2, 3), **call)
        assert seen == [full + own // 3 + 2 * 2 * 256 * 64 * 2]  # the other layers hold nothing yet
        assert batch.stats().gpu_allocated_kv_bytes == full + own
    finally:
        hook.remove()
    hook = _stop_at(tiny, 1, True)
    try:
        with pytest.raises(_Stop):
            _forward(tiny, batch, _ids(16, 2, 3), **call)
    finally:
        hook.remove()
    assert batch.stats().gpu_allocated_kv_bytes > full + own
    batch.rollback()
    assert batch.stats().gpu_allocated_kv_bytes == full + own


def test_layers_of_different_shapes_share_no_buffer() -> None:
    """Layers whose head_dim, dtype or heads differ, each against its tokens in 64 bits: softmax weights of 3 + 2 (causal) rows; float16 /
    bfloat16 outputs of torch's attention, within 4 half steps of the largest value."""
    from lazykv_amd.cache import FullGPUCache, SharedPrefixCache

    gen = torch.Generator(device="cuda").manual_seed(17)
    shapes = [(2, 64, torch.float16), (2, 128, torch.float16), (2, 128, torch.bfloat16), (1, 128, torch.bfloat16), (2, 64, torch.float16)]
    full = FullGPUCache(len(shapes), 16)
    made = []
    for layer, (h, d, t) in zip(full.layers, shapes):
        kv = torch.randn((2, 1, h, 3, d), device="cuda", generator=gen).to(t)
        layer.store(kv[0], kv[1])
        made.append((kv, torch.randn((2, 2, h, 2, d), device="cuda", generator=gen).to(t), torch.randn((2, 2 * h, 2, d), device="cuda", generator=gen).to(t)))
    batch = SharedPrefixCache(full, 2, 8)
    for i, (kv, new, q) in enumerate(made):
        batch.update(new[0], new[1], i)
        got = batch.select(i, q).out.double().cpu().view(q.shape)
        for b in range(2):
            for j in range(q.shape[1]):
                k, v = (torch.cat([kv[w, 0, j // 2], new[w, b, j // 2]]).double().cpu() for w in range(2))
                for t in range(2):
                    p = torch.softmax(k[: 4 + t] @ q[b, j, t].double().cpu() * q.shape[3] ** -0.5, 0)
                    tol = 4 * torch.finfo(q.dtype).eps / 2 * float(v.abs().max())
                    assert float((got[b, j, t] - p @ v[: 4 + t]).abs().max()) <= tol, (i, b, j, t)
