"""Attention by rules and over a paged cache on the CPU: against the definition in 64 bits, refusals, and the layers."""

import numpy as np
import pytest
import torch

import keras_b200 as keras
from keras_b200.kernels import dispatch
from keras_b200.ops import attention_rules
from tests import attention_definition as definition


@pytest.fixture(autouse=True)
def _no_kernels(monkeypatch):
    """These are the plain forms' tests, wherever they run."""
    monkeypatch.setattr(dispatch, "enabled", lambda t: False)


def _inputs(B, T, S, H, K, D, dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    make = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).to(dtype)  # noqa: E731
    return make(B, T, H, D, scale=2.0), make(B, S, K, D), make(B, S, K, D), make(B, T, H, D)


SLOPES = [0.5, 0.1, 0.03, 0.7]
RULES = {
    "cap": dict(attn_logits_soft_cap=3.0),
    "slopes": dict(distance_slopes=SLOPES, is_causal=True),
    "window": dict(sliding_window=3),
    "window_causal": dict(sliding_window=4, is_causal=True, attn_logits_soft_cap=2.0),
    "prefix": dict(prefix_lengths=[0, 4, 40], is_causal=True),
    "segments": dict(segment_ids=torch.tensor([[0, 0, 0, 1, 1, 2, 2, 2, -1], [3, 1, 3, 1, 3, 1, 3, 1, 3], [-1] * 9], dtype=torch.int32), is_causal=True),
    "all": dict(attn_logits_soft_cap=2.0, distance_slopes=SLOPES, sliding_window=5, prefix_lengths=torch.tensor([2, 0, 9]), is_causal=True,
                segment_ids=torch.tensor([[0] * 5 + [1] * 4, [0] * 9, [0, 1] * 4 + [-3]])),
}


def _definition(q, k, v, do, rules, scale=None):
    B, T, S = q.shape[0], q.shape[1], k.shape[1]
    seg = rules.get("segment_ids")
    seg = None if seg is None else seg if isinstance(seg, tuple) else (seg, seg)
    prefix = rules.get("prefix_lengths")
    seen = definition.visible(T, S, B, rules.get("is_causal", False), rules.get("sliding_window"), None if prefix is None else torch.as_tensor(prefix), seg)
    return definition.attention(q, k, v, seen, rules.get("attn_logits_soft_cap"), rules.get("distance_slopes"), scale, do)


@pytest.mark.parametrize("name", sorted(RULES))
def test_rules_and_their_gradients_are_the_definition(name):
    q, k, v, do = _inputs(3, 9, 9, 4, 2, 8)
    found = _definition(q, k, v, do, RULES[name])
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = keras.ops.dot_product_attention(*leaves, **RULES[name])
    definition.check("out", out, found)
    for n, g in zip(("dq", "dk", "dv"), torch.autograd.grad(out, leaves, do)):
        definition.check(n, g, found)


def test_rows_and_keys_of_different_lengths_and_rows_that_see_nothing():
    q, k, v, do = _inputs(2, 5, 7, 4, 4, 8)
    rules = dict(segment_ids=(torch.tensor([[0, 1, 2, -1, 5], [0] * 5]), torch.tensor([[0, 0, 1, 1, -1, 3, 3], [1] * 7])))
    found = _definition(q, k, v, do, rules)
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    out = keras.ops.dot_product_attention(*leaves, **rules)
    definition.check("out", out, found)
    assert not out[1].any() and not out[0, 2:].any() and out[0, :2].all()
    grads = torch.autograd.grad(out, leaves, do)
    for n, g in zip(("dq", "dk", "dv"), grads):
        definition.check(n, g, found)
    assert not grads[1][1].any()


def wide_ids():
    """Ids that int32 does not tell apart, and what they stand for."""
    small = torch.tensor([[0, 0, 0, 1, 1, 2, 2, 0, -1], [3, 1, 3, 1, 3, 1, 3, 1, 3], [0, 1, 2, -1, 4, 5, 6, 7, 8]])
    return {"hashes": torch.where(small < 0, small, small * 2 ** 33 + 2 ** 40 + 5), "padding": torch.where(small < 0, -2 ** 50 + small, 2 ** 62 - small),
            "uint32": torch.where(small < 0, torch.arange(27).reshape(3, 9) + 100, small + 2 ** 31 + 3).to(torch.uint32)}, small


@pytest.mark.parametrize("name", ["hashes", "padding", "uint32"])
@pytest.mark.parametrize("pair", [False, True])
def test_segment_ids_beyond_int32(name, pair):
    wide, small = wide_ids()
    if name == "uint32":  # has no padding: an id of its own in its place, which sees itself
        small = torch.where(small < 0, torch.arange(27).reshape(3, 9) + 100, small)
    q, k, v, do = _inputs(3, 9, 9, 4, 2, 8)
    given = (wide[name], wide[name].clone()) if pair else wide[name]
    found = _definition(q, k, v, do, dict(segment_ids=small))
    definition.check("out", keras.ops.dot_product_attention(q, k, v, segment_ids=given), found)


def test_segment_ids_of_64_bits_that_may_be_none_are_refused():
    q, k, v, _ = _inputs(1, 9, 9, 4, 2, 8)
    with pytest.raises(ValueError, match="integer type"):
        keras.ops.dot_product_attention(q, k, v, segment_ids=torch.zeros(1, 9, dtype=torch.uint64))


def test_gradients_agree_with_differences():
    g = torch.Generator().manual_seed(3)
    leaves = [torch.randn(1, 6, h, 4, generator=g, dtype=torch.float64, requires_grad=True) for h in (4, 2, 2)]
    rules = attention_rules.make(*leaves, 0.5, True, 2.0, SLOPES, 4, torch.tensor([[0, 0, 1, 1, 0, -1]]), [2])
    assert torch.autograd.gradcheck(lambda *t: attention_rules.plain(*t, rules), leaves)  # the entry takes 64 bits as 32


def test_rules_together_with_a_mask_and_a_bias():
    q, k, v, _ = _inputs(1, 6, 6, 4, 4, 8)
    mask = torch.rand(1, 1, 6, 6, generator=torch.Generator().manual_seed(1)) > 0.4
    bias = torch.randn(1, 4, 6, 6, generator=torch.Generator().manual_seed(2))
    out = keras.ops.dot_product_attention(q, k, v, bias=bias, mask=mask, sliding_window=3)
    i = torch.arange(6)
    seen = mask & ((i[:, None] - i[None]).abs() < 3)
    x = (q.transpose(1, 2) @ k.permute(0, 2, 3, 1)) / 8 ** 0.5 + bias
    p = torch.softmax(x.masked_fill(~seen, -1e30), -1) * seen
    torch.testing.assert_close(out, (p @ v.transpose(1, 2)).transpose(1, 2), rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("T,S", [(0, 4), (3, 0), (1, 1)])
def test_empty_and_single_lengths(T, S):
    q, k, v, _ = _inputs(2, T, S, 4, 2, 8)
    out = keras.ops.dot_product_attention(q, k, v, sliding_window=2)
    assert out.shape == (2, T, 4, 8)
    if S == 0:
        assert not out.any()


@pytest.mark.parametrize("given,words", [
    (dict(distance_slopes=[0.1]), "one number a query head"),
    (dict(distance_slopes=torch.zeros(4, requires_grad=True)), "constants"),
    (dict(sliding_window=0), "positive integer"),
    (dict(sliding_window=2.0), "positive integer"),
    (dict(prefix_lengths=[1, 1, 1]), "is_causal"),
    (dict(prefix_lengths=[1.0, 1.0, 1.0], is_causal=True), "integer type"),
    (dict(prefix_lengths=[1], is_causal=True), "shape"),
    (dict(segment_ids=torch.zeros(3, 9)), "integer type"),
    (dict(segment_ids=torch.zeros(3, 8, dtype=torch.int32)), "shape"),
    (dict(segment_ids=(torch.zeros(3, 9, dtype=torch.int32),)), "tuple"),
    (dict(sliding_window=2, attn_logits_soft_cap=0.0), "positive"),
    (dict(sliding_window=2, attn_logits_soft_cap=float("nan")), "finite"),
    (dict(sliding_window=2, flash_attention=True, bias=torch.zeros(1, 1, 9, 9)), "bias"),
])
def test_refused_rules(given, words):
    q, k, v, _ = _inputs(3, 9, 9, 4, 2, 8)
    with pytest.raises(ValueError, match=words):
        keras.ops.dot_product_attention(q, k, v, **given)


def test_refused_shapes():
    q, k, v, _ = _inputs(3, 9, 9, 4, 3, 8)
    with pytest.raises(ValueError, match="multiple"):
        keras.ops.dot_product_attention(q, k, v, sliding_window=2)
    q, k, v, _ = _inputs(3, 9, 8, 4, 2, 8)
    with pytest.raises(ValueError, match="tuple"):
        keras.ops.dot_product_attention(q, k, v, segment_ids=torch.zeros(3, 9, dtype=torch.int32))


# ------------------------------------------------------------------------------------------------ the paged cache
def _cached(lengths, T, page, K=2, D=8, B=None, seed=0, room=None):
    """Whole sequences, and a cache that holds all but their last T tokens."""
    B = len(lengths)
    S = max(lengths) + T if room is None else room
    q, k, v, _ = _inputs(B, S, S, 4, K, D, seed=seed)
    pool_k, pool_v, pages = definition.pool_of(torch.stack([torch.cat([k[b, :n], torch.full((S - n, K, D), float("nan"))]) for b, n in enumerate(lengths)]),
                                               torch.stack([torch.cat([v[b, :n], torch.full((S - n, K, D), float("nan"))]) for b, n in enumerate(lengths)]), page)
    new = [torch.stack([t[b, n:n + T] for b, n in enumerate(lengths)]) for t in (q, k, v)]
    return (q, k, v), new, {"key": pool_k, "value": pool_v, "pages": pages, "lengths": torch.tensor(lengths, dtype=torch.int32)}


@pytest.mark.parametrize("rules", [{}, dict(attn_logits_soft_cap=2.0, distance_slopes=SLOPES), dict(sliding_window=3)], ids=["plain", "cap_slopes", "window"])
@pytest.mark.parametrize("page", [1, 4, 16])
@pytest.mark.parametrize("T", [1, 3])
def test_a_cached_call_is_the_end_of_the_whole_sequence(rules, page, T):
    lengths = [0, 7, 12]
    (q, k, v), new, cache = _cached(lengths, T, page)
    before = {n: cache[n].clone() for n in ("key", "value")}
    out = keras.ops.dot_product_attention(*new, cache=cache, **rules)
    written = set()
    for b, n in enumerate(lengths):
        whole = [t[b:b + 1, : n + T] for t in (q, k, v)]
        found = _definition(*whole, None, dict(rules, is_causal=True))
        value, bound = found["out"]
        definition.check("out", out[b:b + 1], {"out": (value[:, n:], bound[:, n:])})
        for t in range(T):
            page_no, at = int(cache["pages"][b, (n + t) // page]), (n + t) % page
            written.add((page_no, at))
            assert torch.equal(cache["key"][page_no, at], new[1][b, t]) and torch.equal(cache["value"][page_no, at], new[2][b, t])
    for name in ("key", "value"):  # nothing else was written
        for i in range(cache[name].shape[0]):
            for j in range(page):
                if (i, j) not in written:
                    assert torch.equal(cache[name][i, j].nan_to_num(), before[name][i, j].nan_to_num())


def test_idle_sequences_write_nothing_and_are_zero():
    _, new, cache = _cached([5, 5], 3, 4)
    cache["lengths"][1] = -1
    before = cache["key"].clone()
    out = keras.ops.dot_product_attention(*new, cache=cache)
    assert out[0].all() and not out[1].any()
    assert torch.equal(cache["key"][cache["pages"][1].long()].nan_to_num(), before[cache["pages"][1].long()].nan_to_num())


@pytest.mark.parametrize("break_it", ["page_high", "page_negative", "table_end"])
def test_missing_pages_are_an_error_on_the_cpu(break_it):
    _, new, cache = _cached([5, 5], 1, 4)
    if break_it == "page_high":
        cache["pages"][0, 0] = cache["key"].shape[0]
    elif break_it == "page_negative":
        cache["pages"][0, 1] = -7
    else:
        cache["lengths"][1] = cache["pages"].shape[1] * 4
    with pytest.raises(ValueError, match="no page"):
        keras.ops.dot_product_attention(*new, cache=cache)


@pytest.mark.parametrize("change,words", [
    (lambda c: c.pop("pages"), "dict of"),
    (lambda c: c.update(lengths=c["lengths"].long()), "int32"),
    (lambda c: c.update(pages=c["pages"].long()), "int32"),
    (lambda c: c.update(pages=c["pages"][:1]), "int32 of"),
    (lambda c: c.update(lengths=[5, 5]), "tensor"),
    (lambda c: c.update(key=c["key"].half()), "type"),
    (lambda c: c.update(key=c["key"][..., :4]), "pools"),
    (lambda c: c.update(value=c["value"].requires_grad_(True)), "gradients"),
])
def test_refused_caches(change, words):
    _, new, cache = _cached([5, 5], 1, 4)
    change(cache)
    with pytest.raises(ValueError, match=words):
        keras.ops.dot_product_attention(*new, cache=cache)


def test_refused_together_with_a_cache():
    _, new, cache = _cached([5, 5], 1, 4)
    for extra in (dict(mask=torch.ones(1, 1, 1, 1)), dict(segment_ids=torch.zeros(2, 1, dtype=torch.int32)), dict(prefix_lengths=[1, 1])):
        with pytest.raises(ValueError, match="cache takes no"):
            keras.ops.dot_product_attention(*new, cache=cache, **extra)


@pytest.mark.parametrize("which", [0, 1, 2])
def test_refused_devices_with_a_cache(which):
    """An operand of another device than the rest's: its address means nothing to a kernel."""
    _, new, cache = _cached([5, 5], 1, 4)
    new[which] = new[which].to("meta")
    with pytest.raises(ValueError, match="device"):
        keras.ops.dot_product_attention(*new, cache=cache)


# ------------------------------------------------------------------------------------------------ layers
def _layer(kind, **more):
    if kind == "mha":
        return keras.layers.MultiHeadAttention(4, 8, **more)
    return keras.layers.GroupedQueryAttention(8, 4, 2, **more)


@pytest.mark.parametrize("kind", ["mha", "gqa"])
def test_layers_follow_their_rules(kind):
    layer = _layer(kind, attn_logits_soft_cap=1.5, distance_slopes=SLOPES, sliding_window=4)
    x = torch.randn(2, 9, 16, generator=torch.Generator().manual_seed(0))
    seg = torch.tensor([[0] * 4 + [1] * 5, [0] * 8 + [-1]])
    got = layer(x, x, use_causal_mask=True, segment_ids=seg, prefix_lengths=torch.tensor([2, 0]))
    q, k, v = layer.query_dense(x), layer.key_dense(x), layer.value_dense(x)
    rules = dict(attn_logits_soft_cap=1.5, distance_slopes=SLOPES, sliding_window=4, segment_ids=seg, prefix_lengths=torch.tensor([2, 0]), is_causal=True)
    want = layer.output_dense(keras.ops.dot_product_attention(q, k, v, **rules))
    torch.testing.assert_close(got, want)
    again = type(layer).from_config(layer.get_config())
    again.build(x.shape, x.shape)
    again.set_weights(layer.get_weights())
    torch.testing.assert_close(again(x, x, use_causal_mask=True, segment_ids=seg, prefix_lengths=torch.tensor([2, 0])), got)


@pytest.mark.parametrize("kind", ["mha", "gqa"])
def test_a_layers_configuration_without_rules_is_what_it_was(kind):
    config = _layer(kind).get_config()
    assert not {"attn_logits_soft_cap", "distance_slopes"} & set(config) and config.get("sliding_window") is None


@pytest.mark.parametrize("kind", ["mha", "gqa"])
def test_layers_with_masks_beside_their_rules(kind):
    layer = _layer(kind, distance_slopes=SLOPES)
    x = torch.randn(2, 6, 16, generator=torch.Generator().manual_seed(0))
    keep = torch.tensor([[True] * 6, [True] * 4 + [False] * 2])
    got = layer(x, x, value_mask=keep, use_causal_mask=True)
    q, k, v = layer.query_dense(x), layer.key_dense(x), layer.value_dense(x)
    want = layer.output_dense(keras.ops.dot_product_attention(q, k, v, distance_slopes=SLOPES, is_causal=True, mask=keep[:, None, None]))
    torch.testing.assert_close(got, want)


class _Decoder(keras.Model):
    """Two blocks whose attention may read a cache."""

    def __init__(self, vocab, dim, **rules):
        super().__init__()
        self.embed = keras.layers.Embedding(vocab, dim)
        self.norms = [keras.layers.RMSNormalization() for _ in range(2)]
        self.attend = [keras.layers.GroupedQueryAttention(8, 4, 2, **rules) for _ in range(2)]
        self.head = keras.layers.Dense(vocab)

    def call(self, tokens, caches=None):
        x = self.embed(tokens)
        for i in range(2):
            h = self.norms[i](x)
            x = x + self.attend[i](h, h, use_causal_mask=True, cache=None if caches is None else caches[i])
        return self.head(x)


def _generation(device, dtype, rtol):
    """Logits of whole sequences against those of a prompt and then single tokens through the cache."""
    model = _Decoder(50, 16, attn_logits_soft_cap=4.0, distance_slopes=SLOPES, sliding_window=6)
    tokens = torch.randint(0, 50, (3, 11), generator=torch.Generator().manual_seed(0)).to(device)
    whole = model(tokens)
    pages = torch.randperm(12, generator=torch.Generator().manual_seed(1)).reshape(3, 4).to(torch.int32).to(device)
    lengths = torch.zeros(3, dtype=torch.int32, device=device)
    caches = [{"key": torch.full((12, 4, 2, 8), float("nan"), dtype=dtype, device=device), "value": torch.full((12, 4, 2, 8), float("nan"), dtype=dtype, device=device),
               "pages": pages, "lengths": lengths} for _ in range(2)]
    parts = []
    for first, last in ((0, 5), (5, 6), (6, 7), (7, 9), (9, 10), (10, 11)):
        parts.append(model(tokens[:, first:last], caches=caches).detach())
        lengths += last - first
    torch.testing.assert_close(torch.cat(parts, 1).float(), whole.detach().float(), rtol=rtol, atol=rtol)


def test_a_model_generates_through_its_caches():
    # float32 sums of 16 to 50 terms through two blocks: some hundred roundings of 2^-24
    _generation("cpu", torch.float32, 1e-4)


@pytest.mark.parametrize("kind", ["mha", "gqa"])
def test_refused_layer_calls(kind):
    x = torch.zeros(1, 4, 16)
    with pytest.raises(ValueError, match="positive"):
        _layer(kind, attn_logits_soft_cap=-1.0)
    with pytest.raises(ValueError, match="one number a query head"):
        _layer(kind, distance_slopes=[1.0])
    with pytest.raises(ValueError, match="Dropout"):
        _layer(kind, attn_logits_soft_cap=3.0, dropout=0.1)
    with pytest.raises(ValueError, match="Dropout"):
        _layer(kind, dropout=0.1)(x, x, segment_ids=np.zeros((1, 4), "int32"))
    with pytest.raises(ValueError, match="scores"):
        _layer(kind, attn_logits_soft_cap=3.0)(x, x, return_attention_scores=True)
    _, _, cache = _cached([5], 1, 4)
    with pytest.raises(ValueError, match="cache"):
        _layer(kind)(x, x, cache=cache, attention_mask=np.ones((1, 4, 4), bool))
    layer = _layer("gqa")
    cache["key"], cache["value"] = cache["key"].half(), cache["value"].half()
    with pytest.raises(ValueError, match="type"):  # not a copy of the pools that would be written to and dropped
        layer(x, x, cache=cache)


def test_rules_in_a_functional_model_that_trains():
    x, s = keras.Input((8, 16)), keras.Input((8,), dtype="int32")
    y = keras.layers.GroupedQueryAttention(8, 4, 2, attn_logits_soft_cap=5.0)(x, x, use_causal_mask=True, segment_ids=s)
    model = keras.Model([x, s], keras.layers.Dense(3)(y))
    model.compile(optimizer="sgd", loss="mse")
    rng = np.random.default_rng(0)
    data = [rng.normal(size=(4, 8, 16)).astype("float32"), np.repeat([[0, 0, 0, 1, 1, 2, -1, -1]], 4, 0).astype("int32")]
    before = [w.copy() for w in model.get_weights()]
    model.train_on_batch(data, rng.normal(size=(4, 8, 3)).astype("float32"))
    assert all(np.isfinite(w).all() for w in model.get_weights()) and any((a != b).any() for a, b in zip(before, model.get_weights()))


def _slopes_model(kind, seed=0):
    keras.utils.set_random_seed(seed)
    x = keras.Input((8, 16))
    layer = _layer(kind, distance_slopes=SLOPES)
    model = keras.Model(x, keras.layers.Dense(3)(layer(x, x, use_causal_mask=True)))
    model.compile(optimizer="sgd", loss="mse")
    return model, layer


def _transform(how, model, layer, path):
    """A first call of the layer in a mode whose tensors do not outlive it."""
    x = torch.randn(2, 8, 16, generator=torch.Generator().manual_seed(5)).to(model.trainable_variables[0].value.device)
    if how == "export":
        model.export(str(path / "m"), format="torch_export", verbose=False)
    elif how == "func_grad":
        torch.func.grad(lambda z: layer(z, z, use_causal_mask=True).sum())(x)
    elif how == "vmap":
        torch.vmap(lambda z: layer(z[None], z[None], use_causal_mask=True))(x)
    elif how == "trace":
        for v in layer.trainable_variables:  # a trace holds weights as constants
            v._value.requires_grad_(False)
        torch.jit.trace(lambda z: layer(z, z, use_causal_mask=True), (x,), check_trace=False)
        for v in layer.trainable_variables:
            v._value.requires_grad_(True)
    else:
        with torch.inference_mode():
            layer(x, x, use_causal_mask=True)


TRANSFORMS = ["export", "func_grad", "vmap", "trace", "inference"]


def _trains_after(kind, how, path):
    rng = np.random.default_rng(0)
    x, y = rng.normal(size=(4, 8, 16)).astype("float32"), rng.normal(size=(4, 8, 3)).astype("float32")
    losses, weights, kept = [], [], []
    for first in (None, how):
        model, layer = _slopes_model(kind)
        if first is not None:
            _transform(first, model, layer, path)
        losses.append([float(model.train_on_batch(x, y)) for _ in range(3)])
        weights.append(model.get_weights())
        kept.append(list(layer._slopes_on.values()))
        assert type(model(x)) is torch.Tensor and np.isfinite(model.predict(x, verbose=0)).all()
    assert losses[0][0] > 0 and losses[0] == losses[1]
    assert all(np.array_equal(a, b) for a, b in zip(*weights))
    for t in kept[1]:
        assert type(t) is torch.Tensor and not t.is_inference() and not torch._C._functorch.is_functorch_wrapped_tensor(t)


@pytest.mark.parametrize("how", TRANSFORMS)
@pytest.mark.parametrize("kind", ["mha", "gqa"])
def test_slopes_of_a_transform_do_not_outlive_it(kind, how, tmp_path):
    """A layer that is first called under an export, a function transform, a trace or in inference mode trains as one that was not."""
    _trains_after(kind, how, tmp_path)


def test_an_exported_cap_takes_any_batch(tmp_path):
    """Which way a call takes goes by its sizes, and says nothing of those of an export."""
    x = keras.Input((8, 4, 16))
    model = keras.Model(x, keras.layers.Lambda(lambda t: keras.ops.dot_product_attention(t, t, t, attn_logits_soft_cap=3.0))(x))
    model.export(str(tmp_path / "m"), format="torch_export", verbose=False)
    program = torch.export.load(str(tmp_path / "m" / "serve.pt2")).module()
    for n in (1, 3, 6000):
        t = torch.randn(n, 8, 4, 16, generator=torch.Generator().manual_seed(n))
        torch.testing.assert_close(program(t), keras.ops.dot_product_attention(t, t, t, attn_logits_soft_cap=3.0))


@pytest.mark.parametrize("B,T,pays", [(1, 100, True), (2, 4096, False), (4, 4096, False), (5, 4096, True), (1, 100000, True)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_cap_alone_makes_no_matrices_beyond_the_memory(B, T, pays, dtype):
    """16 heads of 256, whose training is faster in the library's operations: not for few pairs, and not beyond 2^30 of them."""
    from keras_b200.kernels import attention_rules as kernels

    q = torch.empty(B, T, 16, 256, dtype=dtype, device="meta", requires_grad=True)
    assert kernels.cap_pays(q, q, q, False) is pays
