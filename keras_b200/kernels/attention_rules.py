"""Front-end of the attention kernels whose scores and masks are given as rules (``csrc/attention_rules*.cu``).

``attention`` takes query/key/value in the ``[batch, time, heads, head_dim]`` layout of the attention layers and a ``Rules``: a cap on the
scores, a bias by distance, causal, prefix, window and segment masks.  Both directions run on this package's kernels; a gradient that is
itself differentiated, or one of a batch of them, takes the plain form.
"""

import collections
import ctypes

import torch

from keras_b200.kernels import ops as kops
from keras_b200.kernels.attention import _err_flag

# cap: number or None; slopes: float32 [heads] or None; causal: bool; window: int or None; prefix: int32 [batch] or None;
# segments: (int32 [batch, rows], int32 [batch, keys]) or None, contiguous
Rules = collections.namedtuple("Rules", "scale cap slopes causal window prefix segments")

_CODES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_HEAD = 256
MAX_LENGTH = 1 << 20  # rows or keys whose tiles the tensor-core kernels keep flags of
_V, _I, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_float
_RULES = [_F, _F, _V, _I, _I, _V, _V, _V, _V, _V, _V]  # scale, cap, slopes, causal, window, prefix, segments of rows and keys, their ranges, stream
_FNS = {}


def launcher(name, arguments):
    """A C entry with its argument types, so that a launch passes plain numbers."""
    fn = _FNS.get(name)
    if fn is None:
        fn = getattr(kops._lib(), name)
        fn.argtypes, fn.restype = arguments, ctypes.c_int
        _FNS[name] = fn
    return fn


def strides(*tensors):
    """Strides of time, heads and batch of each, as the C entries take them; a dimension of one element may carry any."""
    flat = []
    for t in tensors:
        (b, n, h, _), (sb, sn, sh, _) = t.shape, t.stride()
        flat += (0 if n == 1 else sn, 0 if h == 1 else sh, 0 if b == 1 else sb)
    return (ctypes.c_longlong * len(flat))(*flat)


def unit(t):
    """The tensor with unit stride over its last dimension."""
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


class Plan:
    """What a call's types, sizes and strides settle: worked out once for each and kept, as a step calls the same layers again and again."""

    __slots__ = ("fits", "unit", "tensor", "tiled", "grad_strides", "code", "sizes", "out", "lse", "delta", "pitch", "strides", "_work")

    def __init__(self, q, k, v):
        same = (q.dtype in _CODES and k.dtype == q.dtype and v.dtype == q.dtype and k.shape == v.shape and k.shape[0] == q.shape[0] and k.shape[-1] == q.shape[-1]
                and 0 not in q.shape and 0 not in k.shape and q.shape[2] % k.shape[2] == 0 and q.shape[-1] <= MAX_HEAD)
        B, T, H, D = q.shape
        S, K = k.shape[1:3]
        self.fits = same and ((T + 31) // 32) * H * B < 1 << 31 and ((S + 31) // 32) * H * B < 1 << 31
        if not self.fits:
            return
        self.unit = D == 1 or q.stride(3) == k.stride(3) == v.stride(3) == 1
        self.code, self._work = _CODES[q.dtype], None
        # whether the tensor-core kernels take heads of this size and type; layouts they do not read are copied for them
        self.tensor = q.dtype != torch.float32 and D <= 128 and D % 8 == 0 and T <= MAX_LENGTH and S <= MAX_LENGTH
        # strides that tile copies can read: multiples of 16 bytes, none of them zero
        self.tiled = all(n == 1 or (s > 0 and s % 8 == 0) for t in (q, k, v) for n, s in zip(t.shape[:3], t.stride()))
        self.sizes = (B, H, K, T, S, D)
        self.out, self.pitch = (B, T, H, D), (T + 127) // 128 * 128
        self.lse = (B, H, self.pitch)
        self.delta = B * H * self.pitch + (B * (H + K) if self.tensor and q.dtype == torch.float16 else 0)  # float16 keeps norms behind the sums
        self.strides = strides(q, k, v)
        o = (0 if T == 1 else H * D, 0 if H == 1 else D, 0 if B == 1 else T * H * D)
        self.grad_strides = (ctypes.c_longlong * 12)(*self.strides, *o)  # with a contiguous gradient of the result


    def work(self):
        """Floats of workspace of the gradients of key and value."""
        if self._work is None:
            fn = launcher("kb200_attention_rules_bwd_work" if self.tensor else "kb200_attention_rules_bwd_work_plain", [_I] * 6)
            fn.restype = ctypes.c_longlong
            self._work = fn(*self.sizes)
        return self._work


_PLANS = {}


def plan_of(q, k, v):
    key = (q.dtype, k.dtype, v.dtype, q.shape, k.shape, v.shape, q.stride(), k.stride(), v.stride())
    plan = _PLANS.get(key)
    if plan is None:
        if len(_PLANS) >= 1024:  # sizes that change with every call
            _PLANS.clear()
        plan = _PLANS[key] = Plan(q, k, v)
    return plan


_SMALL, _LARGE = 5 << 18, 1 << 30  # pairs of rows and keys, over all heads


def cap_pays(q, k, v, causal):
    """Whether a call whose only rule is a cap is faster on these kernels than in the library's operations over whole score matrices.  On the tensor cores always
    (2 to 20 times).  The FMA kernels are bound by their arithmetic, with nothing but a causal mask to leave out, where the library multiplies
    at twice to fifty times their rate and pays for some ten passes over the matrix.  Measured, as multiples of the library's speed:

    * beyond 2^30 pairs the library's matrices, of 20 bytes a pair at their peak and 8 that the gradients keep, take memory that a model has other use for:
      the kernels, whatever the time
    * up to 1.3 million pairs, where the library's launches last longer than either: 1.0 to 5 (1 x 64 x 8 x 256 float32 forward 43 us against 84)
    * fewer than 128 tiles of 64 rows, which leave SMs without a block: from 0.3 (1 x 1024 x 4 x 64 float32 forward 0.6)
    * heads of up to 64: forward 1.0 to 1.6, causal 1.4 to 3.5; trained 0.6 to 0.85, causal 1.1 to 1.9
    * up to 128: forward 0.4 to 0.95, causal 1.1 to 2.2; trained 0.3 to 0.85, causal 1.0 to 1.3 in float32 and 0.6 to 0.7 in 16 bits
    * beyond: forward 0.2 to 0.9, causal 1.1 to 1.45 in float32 (0.85 to 0.95 with 128 tiles) and 0.6 to 0.8 in 16 bits; trained 0.1 to 0.7
    """
    (B, T, H, D), S, narrow = q.shape, k.shape[1], q.dtype != torch.float32
    if (narrow and D <= 128 and D % 8 == 0) or not _SMALL < B * H * T * S <= _LARGE:
        return True
    tiles = B * H * ((T + 63) // 64)
    if tiles < 128:
        return False
    training = (q.requires_grad or k.requires_grad or v.requires_grad) and torch.is_grad_enabled()
    halved = causal and min(T, S) >= 256  # of one or two tiles a causal mask leaves out nothing
    if D <= 64:
        return halved or not training or max(T, S) <= 128
    return halved and ((D <= 128 and not (narrow and training)) or (tiles >= 148 and not narrow and not training))


def _ptr(t):
    return None if t is None else t.data_ptr()


_RANGES_ARGS = [_V, _V, _I, _I, _V]


def _ranges(seg):
    B, T = seg.shape
    out = torch.empty((B, (T + 127) // 128, 4), dtype=torch.int32, device=seg.device)
    code = launcher("kb200_segment_ranges", _RANGES_ARGS)(seg.data_ptr(), out.data_ptr(), B, T, kops._stream())
    kops._check(code, "segment_ranges")
    return out


def _tail(rules, ranges):
    """The arguments that say the rules, the stream included."""
    if rules.segments is None:
        seg_q = seg_k = range_q = range_k = None
    else:
        seg_q, seg_k, range_q, range_k = (t.data_ptr() for t in (*rules.segments, *ranges))
    return (rules.scale, rules.cap or 0.0, _ptr(rules.slopes), 1 if rules.causal else 0, min(rules.window or 0, 1 << 30), _ptr(rules.prefix), seg_q, seg_k, range_q, range_k,
            kops._stream())


def segment_ranges(rules):
    if rules.segments is None:
        return None, None
    rows, keys = rules.segments
    first = _ranges(rows)
    return first, first if keys is rows else _ranges(keys)


def _tiles(t):
    """A tensor that tile copies can read: base and strides multiples of 16 bytes, none of them zero."""
    if t.data_ptr() % 16 == 0 and all(n == 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape[:3], t.stride())):
        return t
    return kops.aligned(t)


_FWD_SM100 = [_V] * 6 + [_I, _V] + [_I] * 7 + [_V] + _RULES
_FWD = [_V] * 5 + [_I, _V] + [_I] * 7 + _RULES
_GRADS = [_V] * 9 + [_I] + [_V] * 3 + [_I] * 7 + [_V, _V, ctypes.c_longlong] + _RULES


def forward(q, k, v, rules, ranges, training, plan=None):
    """``(out [B, Tq, H, D], lse [B, H, pitch] float32, lo)``; the sums of a row are kept as log2, ``lo`` is what rounding the result lost, both for the
    gradients alone."""
    plan = plan or plan_of(q, k, v)
    out = q.new_empty(plan.out)
    lse = q.new_empty(plan.lse, dtype=torch.float32) if training else None
    if plan.tensor:
        a, b, c = q.data_ptr(), k.data_ptr(), v.data_ptr()
        layout = plan.strides
        if not plan.tiled or (a | b | c) % 16:
            q, k, v = _tiles(q), _tiles(k), _tiles(v)
            a, b, c = q.data_ptr(), k.data_ptr(), v.data_ptr()
            layout = strides(q, k, v)
        lo = q.new_empty(plan.out) if training else None
        code = launcher("kb200_attention_rules_fwd_sm100", _FWD_SM100)(
            a, b, c, out.data_ptr(), _ptr(lo), _ptr(lse), plan.pitch, layout, plan.code, *plan.sizes, _err_flag(q.device).data_ptr(), *_tail(rules, ranges))
        kops._check(code, "attention_rules_fwd_sm100")
        return out, lse, lo
    code = launcher("kb200_attention_rules_fwd", _FWD)(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(lse), plan.pitch, plan.strides, plan.code, *plan.sizes, *_tail(rules, ranges))
    kops._check(code, "attention_rules_fwd")
    return out, lse, None


def _plain_rows(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _as_saved(t, dtype, device, count):
    return t is None or (t.dtype is dtype and t.numel() == count and t.get_device() == device)


def _came_back(q, k, v, out, lo, lse, grad_out, rules, ranges):
    """The plan of the saved tensors as they are now, once hooks have had them: their addresses say nothing of types and sizes."""
    plan, device, d, n = plan_of(q, k, v), q.get_device(), q.dtype, q.numel()
    ok = plan.fits and k.get_device() == device and v.get_device() == device and _as_saved(out, d, device, n) and _as_saved(lo, d, device, n) and _as_saved(grad_out, d, device, n)
    if ok:
        B, H, _, T, S, _ = plan.sizes
        ok = _as_saved(lse, torch.float32, device, B * H * plan.pitch) and _as_saved(rules.slopes, torch.float32, device, H) and _as_saved(rules.prefix, torch.int32, device, B)
        if rules.segments is not None:
            counts = (B * T, B * S, B * ((T + 127) // 128) * 4, B * ((S + 127) // 128) * 4)
            ok = ok and all(_as_saved(t, torch.int32, device, c) for t, c in zip((*rules.segments, *ranges), counts))
    if not ok:
        raise RuntimeError("attention by rules: a tensor that was saved for the gradients came back with another type, size or device")
    return plan


def backward(q, k, v, out, lo, lse, grad_out, rules, ranges, want_q, want_kv):
    # what was saved may have come back in another layout, and the C entries take strides of q, k, v and the gradient alone
    q, k, v, out, lo, lse = unit(q), unit(k), unit(v), _plain_rows(out), _plain_rows(lo), _plain_rows(lse)
    plan = _came_back(q, k, v, out, lo, lse, grad_out, rules, ranges)
    rules = rules._replace(slopes=_plain_rows(rules.slopes), prefix=_plain_rows(rules.prefix))
    if rules.segments is not None:
        rules, ranges = rules._replace(segments=tuple(map(_plain_rows, rules.segments))), tuple(map(_plain_rows, ranges))
    tensor = plan.tensor
    a, b, c, d = q.data_ptr(), k.data_ptr(), v.data_ptr(), grad_out.data_ptr()
    layout = plan.grad_strides
    if not grad_out.is_contiguous() or (tensor and (not plan.tiled or (a | b | c | d) % 16)):
        grad_out = unit(grad_out)
        if tensor:
            q, k, v, grad_out = _tiles(q), _tiles(k), _tiles(v), _tiles(grad_out)
        a, b, c, d = q.data_ptr(), k.data_ptr(), v.data_ptr(), grad_out.data_ptr()
        layout = strides(q, k, v, grad_out)
    delta = lse.new_empty(plan.delta)
    dq = q.new_empty(plan.out) if want_q else None
    dk = dv = work = None
    floats = 0
    if want_kv:
        B, _, K, _, S, D = plan.sizes
        dk, dv = q.new_empty((B, S, K, D)), q.new_empty((B, S, K, D))
        floats = plan.work()
        if floats:  # from the caching allocator, for this call and stream alone: a recorded graph has its own
            work = q.new_empty(floats, dtype=torch.float32)
    # the sums of out * grad_out, then the gradients
    name = "kb200_attention_rules_grads_sm100" if tensor else "kb200_attention_rules_grads"
    code = launcher(name, _GRADS)(
        a, b, c, out.data_ptr(), _ptr(lo), d, layout, lse.data_ptr(), delta.data_ptr(), plan.pitch,
        _ptr(dq), _ptr(dk), _ptr(dv), plan.code, *plan.sizes, _err_flag(q.device).data_ptr(), _ptr(work), floats, *_tail(rules, ranges))
    kops._check(code, name[6:])
    kops.add_launches(1)  # two launchers in one call
    return dq, dk, dv


def _of_a_batch(t):
    """Whether it is many tensors in one (``is_grads_batched``, ``torch.func``), which has no address."""
    return torch._C._functorch.is_legacy_batchedtensor(t) or torch._C._functorch.is_functorch_wrapped_tensor(t)


class RuleAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, prefix, rows, keys, rules, plain, plan):
        ranges = segment_ranges(rules)
        out, lse, lo = forward(q, k, v, rules, ranges, True, plan)
        # the rules' tensors are saved too: one that is written to before the backward pass is an error, as for any operand
        ctx.save_for_backward(q, k, v, out, lo, lse, *ranges, slopes, prefix, rows, keys)
        ctx.rules, ctx.plain = Rules(rules.scale, rules.cap, None, rules.causal, rules.window, None, None), plain
        return out

    @staticmethod
    def backward(ctx, grad_out):
        q, k, v, out, lo, lse, range_q, range_k, slopes, prefix, rows, keys = ctx.saved_tensors
        r = ctx.rules
        rules = Rules(r.scale, r.cap, slopes, r.causal, r.window, prefix, None if rows is None else (rows, keys))
        need = ctx.needs_input_grad
        again = torch.is_grad_enabled()  # the gradient is differentiated in its turn
        if again or _of_a_batch(grad_out):
            wanted = [t for t, n in zip((q, k, v), need) if n]
            with torch.enable_grad():
                given = iter(torch.autograd.grad(ctx.plain(q, k, v, rules), wanted, grad_out, create_graph=again))
            grads = [next(given) if n else None for n in need[:3]]
        else:
            dq, dk, dv = backward(q, k, v, out, lo, lse, grad_out, rules, (range_q, range_k), need[0], need[1] or need[2])
            grads = [dq, dk if need[1] else None, dv if need[2] else None]
        return (*grads, None, None, None, None, None, None, None)


def _savable(rules):
    """The rules with ordinary tensors: one that was made in inference mode cannot be saved for the gradients."""
    slopes, prefix = (t.clone() if t is not None and t.is_inference() else t for t in (rules.slopes, rules.prefix))
    segments = rules.segments
    if segments is not None and (segments[0].is_inference() or segments[1].is_inference()):
        rows = segments[0].clone()
        segments = rows, rows if segments[1] is segments[0] else segments[1].clone()
    return rules if slopes is rules.slopes and prefix is rules.prefix and segments is rules.segments else rules._replace(slopes=slopes, prefix=prefix, segments=segments)


def attention(q, k, v, rules, plain):
    """Attention on this package's kernels, or ``None`` when the call does not fit them.  ``plain(q, k, v, rules)``: the form that second
    derivatives go through."""
    if not q.device == k.device == v.device or torch.is_autocast_enabled("cuda"):
        return None
    plan = plan_of(q, k, v)
    if not plan.fits:
        return None
    if not plan.unit:
        q, k, v = unit(q), unit(k), unit(v)
        plan = plan_of(q, k, v)
    if (q.requires_grad or k.requires_grad or v.requires_grad) and torch.is_grad_enabled():
        rules = _savable(rules)
        rows, keys = rules.segments or (None, None)
        return RuleAttention.apply(q, k, v, rules.slopes, rules.prefix, rows, keys, rules, plain, plan)
    return forward(q, k, v, rules, segment_ranges(rules), False, plan)[0]
