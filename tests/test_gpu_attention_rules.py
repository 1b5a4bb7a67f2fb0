"""The kernels of attention by rules and over a paged cache: against the definition in 64 bits, at the sizes, layouts and masks where they can go
wrong, recorded, on other streams, and as a model uses them."""

import pytest
import torch

import keras_b200 as keras
from keras_b200.kernels import attention, attention_cache, attention_rules, ops as kops
from tests import attention_definition as definition
from tests.test_attention_rules import SLOPES, TRANSFORMS, _Decoder, _generation, _layer, _trains_after

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def _names(v):
    return str(v).replace("torch.", "") if isinstance(v, torch.dtype) else None


def _inputs(B, T, S, H, K, D, dtype, seed=0, q_scale=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda *s, scale=1.0: (torch.randn(*s, generator=g, device="cuda") * scale).to(dtype)  # noqa: E731
    return make(B, T, H, D, scale=q_scale), make(B, S, K, D), make(B, S, K, D), make(B, T, H, D)


def _slopes(H):
    return [2.0 ** (-8.0 * (h + 1) / H) for h in range(H)]


def _definition(q, k, v, do, rules, scale=None):
    seg = rules.get("segment_ids")
    seg = None if seg is None else seg if isinstance(seg, tuple) else (seg, seg)
    seen = definition.visible(q.shape[1], k.shape[1], q.shape[0], rules.get("is_causal", False), rules.get("sliding_window"), rules.get("prefix_lengths"), seg)
    return definition.attention(q, k, v, seen, rules.get("attn_logits_soft_cap"), rules.get("distance_slopes"), scale, do)


def _run(q, k, v, do, rules):
    """Results and gradients, and that kernels made them; the result without gradients, whose rounding of the probabilities may differ, last."""
    before = kops.launch_count()
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = keras.ops.dot_product_attention(*leaves, **rules)
    grads = torch.autograd.grad(out, leaves, do)
    assert kops.launch_count() - before >= 3
    with torch.no_grad():
        alone = keras.ops.dot_product_attention(q, k, v, **rules)
    return (out.detach(), *grads, alone)


def _check(q, k, v, do, rules):
    found = _definition(q, k, v, do, rules)
    for name, got in zip(("out", "dq", "dk", "dv", "out"), _run(q, k, v, do, rules)):
        assert got.dtype == q.dtype
        definition.check(name, got, found)


def _ids(B, T, kind):
    g = torch.Generator().manual_seed(T)
    if kind == "documents":
        return torch.cumsum((torch.rand(B, T, generator=g) < 0.02).int(), 1).to(torch.int32).cuda()
    if kind == "padded":
        ids = torch.cumsum((torch.rand(B, T, generator=g) < 0.03).int(), 1).to(torch.int32)
        ids[0, T // 2:] = -1
        ids[-1] = -5
        return ids.cuda()
    return torch.randint(-1, 4, (B, T), generator=g, dtype=torch.int32).cuda()  # in no order


def _rules(name, B, T, H):
    return {
        "cap": lambda: dict(attn_logits_soft_cap=3.0),
        "cap_causal": lambda: dict(attn_logits_soft_cap=30.0, is_causal=True),
        "slopes": lambda: dict(distance_slopes=_slopes(H), is_causal=True),
        "slopes_both_ways": lambda: dict(distance_slopes=_slopes(H)),
        "window": lambda: dict(sliding_window=max(1, T // 3)),
        "window_causal": lambda: dict(sliding_window=max(1, T // 4), is_causal=True, attn_logits_soft_cap=5.0),
        "prefix": lambda: dict(prefix_lengths=torch.tensor([T // 2, 0, T + 9][:B], dtype=torch.int32, device="cuda"), is_causal=True),
        "documents": lambda: dict(segment_ids=_ids(B, T, "documents"), is_causal=True),
        "padded": lambda: dict(segment_ids=_ids(B, T, "padded"), attn_logits_soft_cap=10.0),
        "mixed": lambda: dict(segment_ids=_ids(B, T, "mixed"), is_causal=True),
        "all": lambda: dict(segment_ids=_ids(B, T, "documents"), is_causal=True, sliding_window=T // 2 + 1, distance_slopes=_slopes(H), attn_logits_soft_cap=4.0,
                            prefix_lengths=torch.tensor([T // 3, 1, 0][:B], dtype=torch.int32, device="cuda")),
    }[name]()


ALL = ["cap", "cap_causal", "slopes", "slopes_both_ways", "window", "window_causal", "prefix", "documents", "padded", "mixed", "all"]


@pytest.mark.parametrize("rule", ALL)
@pytest.mark.parametrize("dtype", DTYPES, ids=_names)
def test_rules(rule, dtype):
    B, T, H, K, D = 3, 300, 4, 2, 64
    _check(*_inputs(B, T, T, H, K, D, dtype), _rules(rule, B, T, H))


@pytest.mark.parametrize("prefix", [torch.tensor([-2 ** 31, 2 ** 31 - 1, -1], dtype=torch.int32), torch.tensor([-2 ** 40, 2 ** 40, -2 ** 63])], ids=["int32", "int64"])
@pytest.mark.parametrize("dtype", DTYPES, ids=_names)
def test_prefixes_at_the_ends_of_their_type(prefix, dtype):
    """Less than none is none, more than all is all, in each direction."""
    _check(*_inputs(3, 300, 300, 4, 2, 64, dtype), dict(prefix_lengths=prefix.cuda(), is_causal=True))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=_names)
def test_segment_ids_beyond_int32(dtype):
    """Rows and keys of their own lengths, in no order, and in a recorded step."""
    rows, keys = _ids(2, 150, "mixed"), _ids(2, 260, "mixed")
    args, small = _inputs(2, 150, 260, 4, 2, 64, dtype), (rows, keys)
    wide = tuple(torch.where(t < 0, -2 ** 40 + t, 2 ** 40 + t.long() * 2 ** 34) for t in small)
    want = _run(*args, dict(segment_ids=small))
    assert all(torch.equal(a, b) for a, b in zip(_run(*args, dict(segment_ids=wide)), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = keras.ops.dot_product_attention(*args[:3], segment_ids=wide)
    graph.replay()
    assert torch.equal(out, want[4])
    del graph


@pytest.mark.parametrize("D", [8, 24, 64, 72, 80, 96, 120, 128, 200, 256, 7, 33])
@pytest.mark.parametrize("dtype", DTYPES, ids=_names)
def test_head_sizes(D, dtype):
    B, T, H, K = 2, 150, 2, 1
    _check(*_inputs(B, T, T, H, K, D, dtype), dict(is_causal=True, attn_logits_soft_cap=6.0))


@pytest.mark.parametrize("T", [1, 2, 31, 64, 65, 127, 128, 129, 255, 257, 384, 640])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.bfloat16, 128), (torch.float32, 64)], ids=["bfloat16-64", "bfloat16-128", "float32-64"])
def test_lengths(T, dtype, D):
    _check(*_inputs(2, T, T, 2, 2, D, dtype), dict(is_causal=True, sliding_window=100, distance_slopes=_slopes(2)))


@pytest.mark.parametrize("T,S", [(1, 300), (300, 1), (130, 257), (257, 130), (64, 640)])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=_names)
def test_rows_and_keys_of_different_lengths(T, S, causal, dtype):
    ids = (_ids(2, T, "mixed"), _ids(2, S, "mixed"))
    _check(*_inputs(2, T, S, 4, 2, 64, dtype), dict(is_causal=causal, segment_ids=ids, attn_logits_soft_cap=8.0))


@pytest.mark.parametrize("H,K", [(1, 1), (6, 1), (8, 2), (12, 12), (7, 7), (14, 2)])
@pytest.mark.parametrize("D", [64, 128])
def test_heads_that_share_keys(H, K, D):
    _check(*_inputs(2, 200, 200, H, K, D, torch.bfloat16), dict(is_causal=True, distance_slopes=_slopes(H)))


@pytest.mark.parametrize("B,T,S,H,K", [(1, 700, 700, 8, 1), (1, 900, 900, 7, 7), (1, 50, 1500, 16, 2), (2, 1500, 50, 4, 2), (1, 130, 130, 12, 1)])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64), (torch.bfloat16, 200)], ids=str)
def test_gradients_of_few_key_heads_are_shared_out(B, T, S, H, K, dtype, D):
    """Blocks take parts of a key tile's walk over its query heads, whose sums are joined; some parts are empty, some begin within a head."""
    _check(*_inputs(B, T, S, H, K, D, dtype), dict(is_causal=True, sliding_window=400))


@pytest.mark.parametrize("reach", [0.4, 0.7, 0.9, 1.5])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=_names)
def test_every_form_of_the_cap(reach, dtype):
    """Scores up to so much of their cap: each form of its tanh, in whole tiles and in masked ones."""
    q, k, v, do = _inputs(1, 400, 400, 2, 2, 64, dtype)
    top = torch.einsum("bthd,bshd->bhts", q.float(), k.float()).abs().max().item() / 8.0
    _check(q, k, v, do, dict(is_causal=True, attn_logits_soft_cap=top / reach))


@pytest.mark.parametrize("layout", ["heads_first", "fused", "offset", "expanded", "sliced_heads", "backwards"])
@pytest.mark.parametrize("dtype", DTYPES, ids=_names)
def test_layouts(layout, dtype):
    B, T, H, D = 2, 140, 4, 64
    q, k, v, do = _inputs(B, T, T, H, H, D, dtype)
    if layout == "heads_first":
        q, k, v, do = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v, do))
    elif layout == "fused":
        packed = torch.cat([q, k, v], dim=2)
        q, k, v = packed.split(H, dim=2)
    elif layout == "offset":  # starts off every boundary of a vector
        def move(t):
            flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
            flat[1:] = t.reshape(-1)
            return flat[1:].view(t.shape)
        q, k, v, do = (move(t) for t in (q, k, v, do))
    elif layout == "expanded":
        k, v = k[:, :, :1].expand(B, T, H, D), v[:1].expand(B, T, H, D)
        do = do[:, :1].expand(B, T, H, D)
    elif layout == "sliced_heads":
        q, k, v = (torch.cat([t, t], dim=-1)[..., :D] for t in (q, k, v))
    else:
        k, v = (t.transpose(1, 3).contiguous().transpose(1, 3) for t in (k, v))  # the head dimension is not the unit one
    _check(q, k, v, do, dict(is_causal=True, attn_logits_soft_cap=5.0))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=_names)
def test_scores_beyond_the_cap_and_scales_of_any_sign(dtype):
    q, k, v, do = _inputs(1, 200, 200, 2, 2, 64, dtype, q_scale=12.0)
    _check(q, k, v, do, dict(attn_logits_soft_cap=1.5, is_causal=True))
    for scale in (-0.2, 0.0):
        found = _definition(q, k, v, do, dict(sliding_window=50), scale=scale)
        for name, got in zip(("out", "dq", "dk", "dv"), _run(q, k, v, do, dict(sliding_window=50, scale=scale))):
            definition.check(name, got, found)


@pytest.mark.parametrize("scale", [-0.2, -0.01, 0.0])
def test_a_cap_with_scales_of_any_sign(scale):
    """Whole tiles and masked ones: with a negative scale the largest score is that of the smallest product."""
    q, k, v, do = _inputs(1, 400, 400, 2, 2, 64, torch.bfloat16, q_scale=6.0)
    found = _definition(q, k, v, do, dict(attn_logits_soft_cap=30.0, is_causal=True), scale=scale)
    for name, got in zip(("out", "dq", "dk", "dv", "out"), _run(q, k, v, do, dict(attn_logits_soft_cap=30.0, is_causal=True, scale=scale))):
        definition.check(name, got, found)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=_names)
def test_saved_tensors_that_come_back_in_another_layout(dtype):
    """Hooks may keep what is saved elsewhere and hand it back contiguous: the gradients go by the tensors they get."""
    q, k, v, do = (t.transpose(1, 2).contiguous().transpose(1, 2) for t in _inputs(2, 150, 150, 4, 2, 64, dtype))
    rules = dict(is_causal=True, attn_logits_soft_cap=5.0)
    want = _run(q, k, v, do, rules)[1:4]
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    assert not leaves[0].is_contiguous()
    with torch.autograd.graph.save_on_cpu():
        out = keras.ops.dot_product_attention(*leaves, **rules)
    for a, b in zip(torch.autograd.grad(out, leaves, do), want):
        assert torch.equal(a, b)


def _gradients(q, k, v, do, rules):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    return torch.autograd.grad(keras.ops.dot_product_attention(*leaves, **rules), leaves, do)


@pytest.mark.parametrize("B,T,H,K,D", [(2, 300, 4, 4, 64), (1, 900, 8, 1, 128), (2, 200, 4, 2, 80)])
@pytest.mark.parametrize("cap", [None, 50.0])
def test_float16_gradients_keep_their_bits_at_every_size(B, T, H, K, D, cap):
    """A gradient of the result that is 2^16 times as small gives gradients that are, bit for bit, wherever those are still normal numbers.  (Its values are multiples of
    2^-14, so that it is exact itself and its numbers are normal too: of others the tensor cores' sums may be cut off elsewhere.)"""
    q, k, v, _ = _inputs(B, T, T, H, K, D, torch.float16)
    v = v * 64
    do = torch.randint(-8, 9, q.shape, generator=torch.Generator().manual_seed(1)).cuda().half() * 4
    rules = dict(is_causal=True, sliding_window=T, attn_logits_soft_cap=cap)
    for name, large, small in zip(("dq", "dk", "dv"), _gradients(q, k, v, do, rules), _gradients(q, k, v, do * 2.0 ** -16, rules)):
        assert torch.isfinite(large).all()
        normal = small.abs() > 2.0 ** -14  # 2^-14 itself is also what the numbers of half a step below it are rounded to
        assert name == "dv" or normal.float().mean() > 0.5
        assert torch.equal(small.double()[normal] * 2 ** 16, large.double()[normal]), name


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [300, 1024])
def test_float16_gradients_of_a_mean_loss(T, D):
    """As far off as two roundings, not as what float16 leaves of numbers far below 2^-14.  An element is rounded once, with an error of root mean square r; dS was
    rounded before its sum, an independent error of the same relative size in each term, whose sum is r again where the terms do not cancel, half as much more
    where they do (1.5 r in 64 bits with that rounding alone, one in all by root sum): 2 r bounds it.  The sequences' gradients differ by 10^4."""
    q, k, v, do = _inputs(2, T, T, 2, 2, D, torch.float16, q_scale=3.0)
    do = (do.float() * torch.tensor([1.0, 1e-4], device="cuda").view(2, 1, 1, 1)).half()
    rules = dict(is_causal=True, sliding_window=T)
    found = _definition(q, k, v, do, rules)
    for name, got in zip(("dq", "dk"), _gradients(q, k, v, do, rules)):
        exact = found[name][0]
        for b in range(2):
            rounding = (exact[b].half().double() - exact[b]).square().mean().sqrt()
            off = (got[b].double().cpu() - exact[b]).square().mean().sqrt()
            assert off <= 2 * rounding, (name, b, float(off / rounding))


def test_float16_gradients_of_recorded_steps():
    """Two recordings, replayed in turn with gradients of very different sizes: each finds its own largest norms again."""
    graphs = []
    for B, T, H, K in ((2, 200, 4, 2), (1, 300, 8, 1)):
        q, k, v, do = _inputs(B, T, T, H, K, 64, torch.float16)
        leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
        _gradients(q, k, v, do, dict(is_causal=True, attn_logits_soft_cap=9.0))  # a process's first launch of a kernel loads it, which no recording takes
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            made = torch.autograd.grad(keras.ops.dot_product_attention(*leaves, is_causal=True, attn_logits_soft_cap=9.0), leaves, do)
        graphs.append((graph, leaves, do, made))
    for factor in (1.0, 2.0 ** -10, 2.0 ** 6):
        for graph, leaves, do, _ in graphs:
            do.copy_(torch.randn(do.shape, generator=torch.Generator().manual_seed(3)).cuda().half() * factor)
            graph.replay()
        for graph, leaves, do, made in graphs:
            want = _gradients(*(t.detach() for t in leaves), do, dict(is_causal=True, attn_logits_soft_cap=9.0))
            assert all(torch.equal(a, b) for a, b in zip(made, want))
    del graph, graphs


def test_float16_gradients_beside_infinite_and_zero_ones():
    """What is infinite in one sequence, and zero in another, has no say in a third."""
    q, k, v, do = _inputs(3, 260, 260, 2, 1, 64, torch.float16)
    rules = dict(is_causal=True, sliding_window=100)
    want = _gradients(q, k, v, do, rules)
    do[0, 40, 1, 3], do[1] = float("inf"), 0
    v[0, 7] = float("nan")
    got = _gradients(q, k, v, do, rules)
    for a, b in zip(got, want):
        assert torch.equal(a[2], b[2]) and not a[1].any()
    v[2] = 0
    assert not _gradients(q, k, v, do, rules)[0][2].any()


@pytest.mark.parametrize("B,T,H,D,dtype,causal,forward,trained", [
    (2, 1024, 8, 64, torch.bfloat16, False, True, True), (2, 1024, 8, 128, torch.float16, True, True, True), (1, 64, 8, 256, torch.bfloat16, False, True, True),
    (1, 1024, 4, 64, torch.float32, True, False, False), (2, 1024, 8, 64, torch.float32, False, True, False), (2, 1024, 8, 64, torch.float32, True, True, True),
    (64, 64, 16, 64, torch.float32, False, True, True), (64, 64, 16, 128, torch.float32, True, False, False),
    (2, 1024, 8, 128, torch.float32, False, False, False), (2, 1024, 8, 128, torch.float32, True, True, True), (2, 1024, 8, 100, torch.bfloat16, True, True, False),
    (2, 1024, 8, 256, torch.float32, True, True, False), (2, 1024, 8, 256, torch.bfloat16, True, False, False), (2, 1024, 8, 160, torch.float16, False, False, False),
], ids=str)
def test_a_cap_alone_runs_where_it_is_faster(B, T, H, D, dtype, causal, forward, trained, monkeypatch):
    """The library's operations took such calls before there were kernels: where those are faster they still do."""
    q, k, v, do = _inputs(B, T, T, H, H, D, dtype)
    calls = _spy(monkeypatch)
    with torch.no_grad():
        out = keras.ops.dot_product_attention(q, k, v, is_causal=causal, attn_logits_soft_cap=20.0)
    assert bool(calls["forward"]) == forward
    calls["forward"] = 0
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    again = keras.ops.dot_product_attention(*leaves, is_causal=causal, attn_logits_soft_cap=20.0)
    grads = torch.autograd.grad(again, leaves, do)
    assert bool(calls["forward"]) == bool(calls["backward"]) == trained
    assert out.shape == again.shape == q.shape and out.dtype == dtype and all(torch.isfinite(t).all() for t in (out, again, *grads))


def _spy(monkeypatch):
    """How often the kernels' two directions run from here on."""
    calls = {"forward": 0, "backward": 0}
    for name in calls:
        def spied(*a, _name=name, _fn=getattr(attention_rules, name), **k):
            calls[_name] += 1
            return _fn(*a, **k)
        monkeypatch.setattr(attention_rules, name, spied)
    return calls


def _turned(t):
    """The same values, with the first and the last dimension's places in memory exchanged."""
    return t.transpose(0, -1).contiguous().transpose(0, -1) if t.ndim > 1 else torch.stack([t, t], 1)[:, 0]


@pytest.mark.parametrize("rule", ["cap_causal", "all"])
@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float16, 128), (torch.float32, 64), (torch.bfloat16, 200)], ids=str)
def test_every_saved_tensor_may_come_back_in_another_layout(rule, dtype, D):
    q, k, v, do = _inputs(3, 150, 150, 4, 2, D, dtype)
    rules = _rules(rule, 3, 150, 4)
    want = _run(q, k, v, do, rules)[1:4]
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, _turned):
        out = keras.ops.dot_product_attention(*leaves, **rules)
        got = torch.autograd.grad(out, leaves, do)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("change", [lambda t: t.half() if t.dtype == torch.float32 else t, lambda t: t[:1], lambda t: t.long() if t.dtype == torch.int32 else t, lambda t: t.cpu()],
                         ids=["type", "shape", "integers", "device"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=_names)
def test_saved_tensors_that_come_back_as_others_are_an_error(change, dtype):
    """Before a launch, which would read them as what they were."""
    q, k, v, do = _inputs(3, 20, 20, 4, 2, 64, dtype)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, change):
        out = keras.ops.dot_product_attention(*leaves, **_rules("all", 3, 20, 4))
        launches = kops.launch_count()
        with pytest.raises(RuntimeError, match="came back"):
            torch.autograd.grad(out, leaves, do)
    assert kops.launch_count() == launches


@pytest.fixture(autouse=True)
def _no_wait_ran_out():
    yield
    attention.check_errors()


@pytest.mark.parametrize("dtype,D", [(torch.bfloat16, 64), (torch.float32, 64), (torch.float16, 128)])
def test_results_repeat_bit_for_bit(dtype, D):
    args = _inputs(2, 500, 500, 4, 2, D, dtype), _rules("all", 2, 500, 4)
    first = _run(*args[0], args[1])
    for got in (_run(*args[0], args[1]) for _ in range(3)):
        assert all(torch.equal(a, b) for a, b in zip(first, got))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=_names)
def test_nan_and_infinity_reach_the_rows_that_see_them_alone(dtype):
    """Tiles that a row does not see are not looked at: what is wrong there stays there."""
    q, k, v, do = _inputs(2, 512, 512, 2, 2, 64, dtype)
    ids = torch.arange(512, device="cuda", dtype=torch.int32).div(256, rounding_mode="floor").expand(2, 512).contiguous()
    k[0, 300], v[1, 400] = float("nan"), float("inf")
    out = keras.ops.dot_product_attention(q, k, v, segment_ids=ids)
    assert torch.isfinite(out[:, :256]).all()
    assert torch.isnan(out[0, 256:]).all() and not torch.isfinite(out[1, 256:]).any()


def test_only_the_wanted_gradients():
    q, k, v, do = _inputs(2, 200, 200, 4, 2, 64, torch.bfloat16)
    rules = dict(is_causal=True, attn_logits_soft_cap=5.0)
    want = _run(q, k, v, do, rules)[1:]
    for wanted in ((0,), (1,), (2,), (0, 2), (1, 2)):
        leaves = [t.detach().requires_grad_(i in wanted) for i, t in enumerate((q, k, v))]
        out = keras.ops.dot_product_attention(*leaves, **rules)
        for i, g in zip(wanted, torch.autograd.grad(out, [leaves[i] for i in wanted], do)):
            assert torch.equal(g, want[i])


def test_the_same_tensor_as_query_key_and_value():
    x = _inputs(2, 150, 150, 4, 4, 64, torch.bfloat16)[0].requires_grad_(True)
    do = torch.randn_like(x)
    found = _definition(x, x, x, do, dict(sliding_window=20))
    total, bound = (sum(found[n][i] for n in ("dq", "dk", "dv")) for i in (0, 1))
    grad, = torch.autograd.grad(keras.ops.dot_product_attention(x, x, x, sliding_window=20), x, do)
    definition.check("sum", grad, {"sum": (total, bound + 3 * 2.0 ** -8 * sum(found[n][0].abs() for n in ("dq", "dk", "dv")))})  # two additions of bfloat16


def test_second_derivatives():
    q, k, v, do = _inputs(1, 20, 20, 2, 1, 8, torch.float32)
    rules = dict(is_causal=True, attn_logits_soft_cap=5.0, sliding_window=7)
    got = []
    for fused in (None, False):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = keras.ops.dot_product_attention(*leaves, flash_attention=fused, **rules)
        first = torch.autograd.grad(out, leaves, do, create_graph=True)
        got.append(torch.autograd.grad(sum((g * g).sum() for g in first), leaves))
    for a, b in zip(*got):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4)  # float32 sums of a few hundred terms of size one, squared


@pytest.mark.parametrize("rules", [dict(attn_logits_soft_cap=5.0), dict(sliding_window=7, is_causal=True)], ids=["cap", "window"])
def test_a_batch_of_gradients_at_once(rules):
    """A vectorized Jacobian hands the backward pass a tensor without an address of its own."""
    q, k, v, _ = _inputs(1, 20, 20, 2, 1, 8, torch.float32)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = keras.ops.dot_product_attention(*leaves, **rules)
    batch = torch.randn(3, *out.shape, generator=torch.Generator().manual_seed(1)).cuda()
    many = torch.autograd.grad(out, leaves, batch, is_grads_batched=True, retain_graph=True)
    one = [torch.autograd.grad(out, leaves, g, retain_graph=True) for g in batch]
    for i, got in enumerate(many):
        torch.testing.assert_close(got, torch.stack([g[i] for g in one]), rtol=1e-4, atol=1e-5)  # float32 sums of twenty terms of size one, twice
    many = torch.autograd.grad(out, leaves[:2], batch, is_grads_batched=True, create_graph=True)
    assert many[0].requires_grad and many[1].shape == (3, *k.shape)


def test_saved_rules_must_not_be_written_to():
    q, k, v, do = _inputs(1, 20, 20, 2, 1, 64, torch.bfloat16)
    ids = torch.zeros(1, 20, dtype=torch.int32, device="cuda")
    q.requires_grad_(True)
    out = keras.ops.dot_product_attention(q, k, v, segment_ids=ids)
    ids += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward(do)


@pytest.mark.parametrize("pair", [False, True])
def test_rules_that_were_made_in_inference_mode(pair):
    """A data pipeline may run in that mode: its masks do for training all the same."""
    q, k, v, do = _inputs(3, 50, 50, 4, 2, 64, torch.bfloat16)
    rules = dict(_rules("all", 3, 50, 4), distance_slopes=torch.tensor(_slopes(4), device="cuda"))
    want = _run(q, k, v, do, rules)
    with torch.inference_mode():
        rules = {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in rules.items()}
    assert rules["segment_ids"].is_inference() and rules["distance_slopes"].is_inference()
    if pair:
        rules["segment_ids"] = (rules["segment_ids"].clone(), rules["segment_ids"])
    assert all(torch.equal(a, b) for a, b in zip(_run(q, k, v, do, rules), want))


def test_another_stream_and_a_recorded_step():
    q, k, v, do = _inputs(2, 333, 333, 4, 2, 64, torch.bfloat16)
    rules = dict(_rules("all", 2, 333, 4), distance_slopes=torch.tensor(_slopes(4), device="cuda"))
    want = _run(q, k, v, do, rules)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _run(q, k, v, do, rules)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))

    leaves = [t.detach().clone().requires_grad_(True) for t in (q, k, v)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = keras.ops.dot_product_attention(*leaves, **rules)
        made = (out, *torch.autograd.grad(out, leaves, do))
    other = _inputs(2, 333, 333, 4, 2, 64, torch.bfloat16, seed=9)
    for new in ((q, k, v), other[:3]):
        with torch.no_grad():
            for leaf, t in zip(leaves, new):
                leaf.copy_(t)
        graph.replay()
        for a, b in zip(made, _run(*new, do, rules)):
            assert torch.equal(a, b)
    del graph


def test_the_cap_alone_on_a_trained_layer():
    """A capped layer trains on the kernels, its recorded step included."""
    keras.config.set_dtype_policy("mixed_bfloat16")
    x, s = keras.Input((64, 64)), keras.Input((64,), dtype="int32")
    layer = keras.layers.GroupedQueryAttention(64, 4, 2, attn_logits_soft_cap=5.0, distance_slopes=SLOPES)
    model = keras.Model([x, s], keras.layers.Dense(3)(layer(x, x, use_causal_mask=True, segment_ids=s)))
    model.compile(optimizer="adam", loss="mse")
    data = [torch.randn(4, 64, 64).numpy(), torch.zeros(4, 64, dtype=torch.int32).numpy()]
    before = kops.launch_count()
    for _ in range(6):
        loss = model.train_on_batch(data, torch.zeros(4, 64, 3).numpy())
    assert kops.launch_count() > before and loss == loss


@pytest.mark.parametrize("rules", [dict(sliding_window=4), dict(attn_logits_soft_cap=5.0)], ids=["window", "cap"])
def test_shared_key_heads_under_a_trace(rules):
    q, k, v, _ = _inputs(2, 9, 9, 4, 2, 8, torch.float32)
    traced = torch.jit.trace(lambda *t: keras.ops.dot_product_attention(*t, is_causal=True, **rules), (q, k, v), check_trace=False)
    want = _definition(q, k, v, None, dict(rules, is_causal=True))
    definition.check("out", traced(q, k, v), want)


@pytest.mark.parametrize("kind", ["mha", "gqa"])
@pytest.mark.parametrize("policy", ["float32", "mixed_bfloat16"])
def test_a_layer_with_a_cap_alone_runs_on_the_kernels_in_both_directions(kind, policy, monkeypatch):
    """Against the same weights with the kernels refused.  Sums of up to 64 products on values of size one, through three matrices: float32 some hundred roundings of
    2^-24; bfloat16 about eight of 2^-8 each way, of the whole gradient's size."""
    keras.config.set_dtype_policy(policy)
    x = torch.randn(4, 64, 64, generator=torch.Generator().manual_seed(0)).cuda()
    up = torch.randn(4, 64, 64, generator=torch.Generator().manual_seed(1)).cuda()
    found, weights = [], None
    for kernels in (True, False):
        keras.utils.set_random_seed(0)
        if not kernels:
            keras.config.disable_flash_attention()
        layer = _layer(kind, attn_logits_soft_cap=2.0)
        keras.config.enable_flash_attention()
        layer.build((4, 64, 64), (4, 64, 64))
        weights = weights or layer.get_weights()
        layer.set_weights(weights)
        calls = _spy(monkeypatch)
        out = layer(x, x, use_causal_mask=True)
        out.float().backward(up)
        assert calls == {"forward": int(kernels), "backward": int(kernels)}
        found.append([out.detach().float(), *(v.value.grad.float() for v in layer.trainable_variables)])
    for a, b in zip(*found):
        assert (a - b).norm() <= (1e-5 if policy == "float32" else 16 * 2.0 ** -8) * b.norm()


@pytest.mark.parametrize("how", TRANSFORMS)
@pytest.mark.parametrize("kind", ["mha", "gqa"])
def test_slopes_of_a_transform_do_not_outlive_it(kind, how, tmp_path, monkeypatch):
    """The kernels take the slopes' address and save them for the gradients: those of a trace, a transform or inference mode have none, or refuse."""
    calls = _spy(monkeypatch)
    _trains_after(kind, how, tmp_path)
    assert calls["backward"] >= 2 and calls["forward"] > calls["backward"]


# ------------------------------------------------------------------------------------------------ the paged cache
def _cached(lengths, T, page, H, K, D, dtype, seed=0, wide=None):
    B, S = len(lengths), max(max(lengths), 0) + T
    q, k, v, _ = _inputs(B, S, S, H, K, D, dtype, seed=seed)
    lens = [max(n, 0) for n in lengths]

    def old(t):
        return torch.stack([torch.cat([t[b, :n].cpu(), torch.full((S - n, K, D), float("nan"), dtype=dtype)]) for b, n in enumerate(lens)])

    pool_k, pool_v, pages = definition.pool_of(old(k), old(v), page, seed=seed, wide=wide)
    new = [torch.stack([t[b, n:n + T] for b, n in enumerate(lens)]) for t in (q, k, v)]
    return (q, k, v), new, {"key": pool_k.cuda(), "value": pool_v.cuda(), "pages": pages.cuda(), "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")}


def _check_cached(whole, new, cache, lengths, T, page, rules, skip=()):
    before = {n: cache[n].clone() for n in ("key", "value")}
    launches = kops.launch_count()
    out = keras.ops.dot_product_attention(*new, cache=cache, **rules)
    assert kops.launch_count() > launches
    pages = cache["pages"].cpu()
    for b, n in enumerate(lengths):
        if b in skip:
            continue
        part = [t[b:b + 1, : n + T] for t in whole]
        # the rows of the new tokens alone: the definition of all rows would be quadratic in the length
        i = torch.arange(n, n + T).view(1, T, 1) - torch.arange(n + T).view(1, 1, n + T)
        seen = (i >= 0) & (i < (rules.get("sliding_window") or 1 << 40))
        found = _late(part[0][:, n:], part[1], part[2], seen, rules, n)
        definition.check("out", out[b:b + 1], found)
        for t in range(T):
            to, at = int(pages[b, (n + t) // page]), (n + t) % page
            for name, fresh in (("key", new[1]), ("value", new[2])):
                assert torch.equal(cache[name][to, at], fresh[b, t])
                before[name][to, at] = fresh[b, t]
    for name in ("key", "value"):
        assert torch.equal(cache[name].nan_to_num(), before[name].nan_to_num())
    return out


def _late(q, k, v, seen, rules, n):
    """The definition for rows that begin at position n."""
    slopes = rules.get("distance_slopes")
    if slopes is None:
        return definition.attention(q, k, v, seen, rules.get("attn_logits_soft_cap"))
    T, S = q.shape[1], k.shape[1]
    full = torch.zeros(1, S, q.shape[2], q.shape[3], dtype=q.dtype)
    full[:, n:] = q.cpu()
    mask = torch.zeros(1, S, S, dtype=torch.bool)
    mask[:, n:] = seen
    value, bound = definition.attention(full, k, v, mask, rules.get("attn_logits_soft_cap"), slopes)["out"]
    return {"out": (value[:, n:], bound[:, n:])}


CACHE_RULES = {"plain": {}, "cap": dict(attn_logits_soft_cap=4.0), "window": dict(sliding_window=37), "one": dict(sliding_window=1)}


@pytest.mark.parametrize("rule", sorted(CACHE_RULES))
@pytest.mark.parametrize("dtype", DTYPES, ids=_names)
@pytest.mark.parametrize("T", [1, 5])
def test_cached_attention(rule, dtype, T):
    lengths = [0, 1, 31, 32, 33, 150, 700]
    data = _cached(lengths, T, 16, 8, 2, 64, dtype)
    _check_cached(*data, lengths, T, 16, CACHE_RULES[rule])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=_names)
@pytest.mark.parametrize("T", [1, 4])
def test_cached_attention_with_slopes(dtype, T):
    lengths = [5, 300]
    _check_cached(*_cached(lengths, T, 24, 4, 4, 64, dtype), lengths, T, 24, dict(distance_slopes=_slopes(4), attn_logits_soft_cap=8.0))


@pytest.mark.parametrize("H,K", [(1, 1), (12, 12), (7, 1), (32, 2), (32, 1), (28, 4)])
@pytest.mark.parametrize("T", [1, 3, 20])
def test_cached_heads_and_rows(H, K, T):
    lengths = [90, 0, 257]
    _check_cached(*_cached(lengths, T, 32, H, K, 128, torch.bfloat16), lengths, T, 32, dict(sliding_window=70))


@pytest.mark.parametrize("D", [8, 24, 64, 80, 96, 128, 256, 7, 33])
@pytest.mark.parametrize("dtype", DTYPES, ids=_names)
def test_cached_head_sizes(D, dtype):
    lengths = [75, 10]
    _check_cached(*_cached(lengths, 2, 16, 4, 2, D, dtype), lengths, 2, 16, {})


@pytest.mark.parametrize("page", [1, 3, 7, 16, 24, 64, 100, 128, 1000])
def test_page_sizes(page):
    lengths = [0, 99, 100, 511]
    _check_cached(*_cached(lengths, 2, page, 4, 2, 64, torch.bfloat16), lengths, 2, page, {})


@pytest.mark.parametrize("page", [3, 7, 16, 24, 64])
@pytest.mark.parametrize("T,window,D", [(1, 5, 64), (1, 16, 128), (5, 33, 64), (20, 9, 128), (2, 200, 80)])
@pytest.mark.parametrize("dtype", DTYPES, ids=_names)
def test_positions_before_a_window_may_hold_anything(page, T, window, D, dtype):
    """Their pages may belong to another sequence by now, or to nobody."""
    lengths = [30, 100, 515, 2, 64]
    whole, new, cache = _cached(lengths, T, page, 8, 2, D, dtype)
    pages = cache["pages"].cpu()
    for b, n in enumerate(lengths):
        for p in range(max(0, n + 1 - window)):
            for name in ("key", "value"):
                cache[name][int(pages[b, p // page]), p % page] = float("nan") if p % 2 else float("inf")
    _check_cached(whole, new, cache, lengths, T, page, dict(sliding_window=window))


@pytest.mark.parametrize("B,K,n,wide", [(1, 1, 20000, None), (1, 8, 5000, None), (2, 2, 3000, 4000), (200, 2, 40, None)])
def test_short_and_long_caches_split_over_many_blocks(B, K, n, wide):
    lengths = [n - 13 * (b % 3) for b in range(B)]
    _check_cached(*_cached(lengths, 1, 64, 2 * K, K, 64, torch.bfloat16, wide=wide), lengths, 1, 64, {})


@pytest.mark.parametrize("dtype,D", [(torch.float32, 64), (torch.float32, 128), (torch.bfloat16, 200), (torch.float16, 33)], ids=str)
@pytest.mark.parametrize("T", [1, 6])
def test_long_caches_of_other_types_and_sizes(dtype, D, T):
    """Few long sequences are shared out over the chip by the kernel of every type; one is idle, one short."""
    lengths = [6000, -1, 130]
    whole, new, cache = _cached(lengths, T, 24, 4, 2, D, dtype)
    out = _check_cached(whole, new, cache, lengths, T, 24, dict(attn_logits_soft_cap=9.0, sliding_window=5500), skip=(1,))
    assert (out[1] == 0).all()


def test_idle_sequences_and_missing_pages():
    lengths = [50, -1, 60, 70, 40]
    whole, new, cache = _cached(lengths, 2, 16, 4, 2, 64, torch.bfloat16)
    P = cache["key"].shape[0]
    cache["pages"][2, 1] = P          # no page of the pool, in the middle
    cache["pages"][3, 4] = -3         # the new tokens' own page
    cache["lengths"][4] = 16 * cache["pages"].shape[1] - 1   # the second token is behind the table's end
    cache["key"][cache["pages"][4].long()] = 0  # that sequence is longer than what was filled
    cache["value"][cache["pages"][4].long()] = 0
    before = {n: cache[n].clone() for n in ("key", "value")}
    out = keras.ops.dot_product_attention(*new, cache=cache)
    assert not out[1].any() and torch.isnan(out[2]).all() and torch.isnan(out[3]).all()
    assert torch.isfinite(out[4, 0]).all() and torch.isnan(out[4, 1]).all()
    definition.check("out", out[:1], _late(new[0][:1], whole[1][:1, :52], whole[2][:1, :52],
                                          (torch.arange(50, 52).view(1, 2, 1) >= torch.arange(52).view(1, 1, 52)), {}, 50))
    changed = (cache["key"].nan_to_num() != before["key"].nan_to_num()).flatten(2).any(2).nonzero().tolist()
    pages = cache["pages"].cpu()
    expected = {(int(pages[0, 3]), 2), (int(pages[0, 3]), 3), (int(pages[2, 3]), 12), (int(pages[2, 3]), 13), (int(pages[4, -1]), 15)}
    assert {tuple(c) for c in changed} == expected
    # within a window that does not reach the missing page its sequence is whole again
    out = keras.ops.dot_product_attention(*new, cache=cache, sliding_window=20)
    assert torch.isfinite(out[2]).all() and torch.isnan(out[3]).all()


@pytest.mark.parametrize("dtype", DTYPES, ids=_names)
@pytest.mark.parametrize("n", [64, 1000, 2 ** 31 - 9])
def test_lengths_behind_the_table(dtype, n):
    """Nothing is read or written there: the rows are NaN, at once, however long the sequence is said to be; others are as they were."""
    whole, new, cache = _cached([50, 20], 2, 16, 4, 2, 64, dtype, wide=4)
    cache["lengths"][0] = n
    before = {k: cache[k].clone() for k in ("key", "value")}
    out = keras.ops.dot_product_attention(*new, cache=cache)
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()
    changed = sum(int((cache[k] != before[k]).logical_and(~(cache[k].isnan() & before[k].isnan())).any(dim=(2, 3)).sum()) for k in before)
    assert changed <= 4  # the second sequence's two tokens


@pytest.mark.parametrize("which", [0, 1, 2])
def test_operands_of_the_host_are_refused(which):
    """Before a launch: a kernel would read the host's address."""
    _, new, cache = _cached([5, 9], 1, 16, 4, 2, 64, torch.bfloat16)
    before = {n: cache[n].clone() for n in ("key", "value")}
    new[which] = new[which].cpu()
    launches = kops.launch_count()
    with pytest.raises(ValueError, match="device"):
        keras.ops.dot_product_attention(*new, cache=cache)
    assert kops.launch_count() == launches
    assert all(torch.equal(cache[n].nan_to_num(), before[n].nan_to_num()) for n in before)


def test_a_cache_of_other_strides_and_past_32_bits():
    """A pool inside of a larger buffer, whose last pages lie past 2^31 elements."""
    lengths = [100]
    whole, new, cache = _cached(lengths, 1, 64, 2, 1, 64, torch.bfloat16)
    stride = (1 << 31) // 3 + 8
    stride -= stride % 8
    big = {}
    for name in ("key", "value"):
        t = cache[name]
        buffer = torch.empty(stride * (t.shape[0] - 1) + 64 * 64, dtype=torch.bfloat16, device="cuda")
        big[name] = buffer.as_strided(t.shape, (stride, 64, 64, 1))
        big[name].copy_(t)
    assert t.shape[0] >= 4 and stride * 3 > 1 << 31
    cache.update(big)
    cache["pages"] = torch.tensor([[3, 2]], dtype=torch.int32, device="cuda")
    for name, i in (("key", 1), ("value", 2)):
        cache[name][3, :, 0] = whole[i][0, :64, 0]
        cache[name][2, :36, 0] = whole[i][0, 64:100, 0]
    _check_cached(whole, new, cache, lengths, 1, 64, {})


def test_a_recorded_step_over_a_growing_cache():
    lengths = [17, 40]
    whole, new, cache = _cached(lengths, 1, 16, 4, 2, 64, torch.bfloat16, wide=6)
    static = [t.clone() for t in new]
    graph = torch.cuda.CUDAGraph()
    warm = torch.cuda.Stream()
    warm.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(warm):
        keras.ops.dot_product_attention(*static, cache=cache)
    torch.cuda.current_stream().wait_stream(warm)
    with torch.cuda.graph(graph):
        out = keras.ops.dot_product_attention(*static, cache=cache)
    more = _inputs(2, 20, 20, 4, 2, 64, torch.bfloat16, seed=4)
    history = [[t[b, :n] for b, n in enumerate(lengths)] for t in whole]
    for step in range(20):
        for to, t in zip(static, more):
            to.copy_(t[:, step:step + 1])
        graph.replay()
        history = [[torch.cat([h[b], t[b, step:step + 1]]) for b in range(2)] for h, t in zip(history, more)]
        for b in range(2):
            n = lengths[b] + step
            found = definition.attention(history[0][b][None, n:], history[1][b][None], history[2][b][None], torch.ones(1, 1, n + 1, dtype=torch.bool))
            definition.check("out", out[b:b + 1], found)
        cache["lengths"] += 1
    del graph


def test_shared_pages_of_a_common_prompt():
    lengths = [64, 64]
    whole, new, cache = _cached(lengths, 1, 16, 4, 2, 64, torch.bfloat16, wide=5)
    cache["pages"][1, :4] = cache["pages"][0, :4]
    part = [torch.cat([t[:1], torch.cat([t[:1, :64], t[1:, 64:]], 1)]) for t in whole]
    _check_cached(part, new, cache, lengths, 1, 16, {})


def test_cached_results_repeat_and_versions_count():
    lengths = [1000, 333]
    _, new, cache = _cached(lengths, 1, 16, 8, 2, 128, torch.bfloat16)
    version = cache["key"]._version
    first = keras.ops.dot_product_attention(*new, cache=cache)
    assert cache["key"]._version > version
    for _ in range(3):
        assert torch.equal(first, keras.ops.dot_product_attention(*new, cache=cache))


@pytest.mark.parametrize("policy,rtol", [("float32", 1e-4), ("bfloat16", 0.06)])
def test_a_model_generates_through_its_caches(policy, rtol):
    # bfloat16: two blocks of about eight roundings of 2^-8 each, on values of size one
    keras.config.set_dtype_policy(policy)
    _generation("cuda", getattr(torch, policy), rtol)


def test_a_prompt_a_recorded_step_and_training_share_one_model():
    """The run of a user: a few training steps, a prompt into the cache, and single tokens from a recorded step."""
    keras.config.set_dtype_policy("bfloat16")
    model = _Decoder(40, 32, attn_logits_soft_cap=4.0, distance_slopes=SLOPES)
    tokens = torch.randint(0, 40, (2, 12), generator=torch.Generator().manual_seed(0)).cuda()
    model.compile(optimizer=keras.optimizers.SGD(0.01), loss=keras.losses.SparseCategoricalCrossentropy(from_logits=True))
    for _ in range(5):
        model.train_on_batch(tokens, tokens)
    with torch.no_grad():
        whole = model(tokens)
        lengths = torch.zeros(2, dtype=torch.int32, device="cuda")
        pages = torch.arange(8, dtype=torch.int32, device="cuda").reshape(2, 4)
        caches = [{"key": torch.zeros(8, 4, 2, 8, dtype=torch.bfloat16, device="cuda"), "value": torch.zeros(8, 4, 2, 8, dtype=torch.bfloat16, device="cuda"),
                   "pages": pages, "lengths": lengths} for _ in range(2)]
        model(tokens[:, :6], caches=caches)
        lengths += 6
        token = tokens[:, 6:7].clone()
        model(token, caches=caches)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits = model(token, caches=caches)
        for t in range(6, 12):
            token.copy_(tokens[:, t:t + 1])
            graph.replay()
            # bfloat16: two blocks of about eight roundings of 2^-8 each, on values of size one
            torch.testing.assert_close(logits[:, 0].float(), whole[:, t].float(), rtol=0.06, atol=0.06)
            lengths += 1
    del graph


def test_refusals_of_the_entries():
    """What the Python side never sends, the C entries answer with an error."""
    lib = kops._lib()
    q, k, v, _ = _inputs(1, 4, 4, 2, 2, 64, torch.float32)
    rules = attention_rules.Rules(1.0, None, None, False, None, None, None)
    assert attention_rules.attention(q, k[..., :32], v[..., :32], rules, None) is None
    big = torch.empty(1, 4, 2, 300, device="cuda")
    assert attention_rules.attention(big, big, big, rules, None) is None
    assert attention_cache.attention(big, big, big, big, big, torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda"), 1.0, None,
                                     None, None) is None
    V, I = attention_rules._V, attention_rules._I
    fn = attention_rules.launcher("kb200_attention_rules_fwd", [V] * 5 + [I, V] + [I] * 7 + attention_rules._RULES)
    out = torch.empty_like(q)
    at = (q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr())
    tail = attention_rules._tail(rules, (None, None))
    assert fn(*at, None, 128, attention_rules.strides(q, k, v), 0, 1, 2, 2, 4, 4, 300, *tail) == -2 and lib is not None
    fn = attention_rules.launcher("kb200_attention_rules_fwd_sm100", [V] * 6 + [I, V] + [I] * 7 + [V] + attention_rules._RULES)
    assert fn(*at, None, None, 128, attention_rules.strides(q, k, v), 0, 1, 2, 2, 4, 4, 64, None, *tail) == -2  # float32
    assert fn(*at, None, None, 128, attention_rules.strides(q, k, v), 1, 1, 2, 2, 4, 4, 60, None, *tail) == -2
    assert fn(at[0] + 2, *at[1:], None, None, 128, attention_rules.strides(q, k, v), 1, 1, 2, 2, 4, 4, 64, None, *tail) == -2
