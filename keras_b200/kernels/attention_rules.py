"""Front-end of the attention kernels whose scores and masks are given as rules (``csrc/attention_rules*.cu``).

``attention`` takes query/key/value in the ``[batch, time, heads, head_dim]`` layout of the attention layers and a ``Rules``: a cap on the
scores, a bias by distance, causal, prefix, window and segment masks.  Both directions run on this package's kernels; a gradient that is
itself differentiated takes the plain form.
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
    flat = [0 if t.shape[i] == 1 else t.stride(i) for t in tensors for i in (1, 2, 0)]
    return (ctypes.c_longlong * len(flat))(*flat)


def unit(t):
    """The tensor with unit stride over its last dimension."""
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _ranges(seg):
    out = torch.empty((seg.shape[0], (seg.shape[1] + 127) // 128, 4), dtype=torch.int32, device=seg.device)
    code = launcher("kb200_segment_ranges", [_V, _V, _I, _I, _V])(seg.data_ptr(), out.data_ptr(), seg.shape[0], seg.shape[1], kops._stream())
    kops._check(code, "segment_ranges")
    return out


def _tail(rules, ranges):
    """The arguments that say the rules, the stream included."""
    seg = rules.segments or (None, None)
    return (rules.scale, rules.cap or 0.0, _ptr(rules.slopes), 1 if rules.causal else 0, min(rules.window or 0, 1 << 30), _ptr(rules.prefix), _ptr(seg[0]), _ptr(seg[1]),
            _ptr(ranges[0]), _ptr(ranges[1]), kops._stream())


def segment_ranges(rules):
    if rules.segments is None:
        return None, None
    rows, keys = rules.segments
    first = _ranges(rows)
    return first, first if keys is rows else _ranges(keys)


def tensor_cores(q, k, v):
    """Whether the tensor-core kernels take heads of this size and type; layouts they do not read are copied for them."""
    return q.dtype != torch.float32 and q.shape[-1] <= 128 and q.shape[-1] % 8 == 0 and q.shape[1] <= MAX_LENGTH and k.shape[1] <= MAX_LENGTH


def _tiles(t):
    """A tensor that tile copies can read: base and strides multiples of 16 bytes, none of them zero."""
    if t.data_ptr() % 16 == 0 and all(n == 1 or (s > 0 and s % 8 == 0) for n, s in zip(t.shape[:3], t.stride())):
        return t
    return kops.aligned(t)


def _pitch(T):
    return (T + 127) // 128 * 128


def forward(q, k, v, rules, ranges, training):
    """``(out [B, Tq, H, D], lse [B, H, pitch] float32, lo)``; the sums of a row are kept as log2, ``lo`` is what rounding the result lost, both for the
    gradients alone."""
    B, Tq, H, D = q.shape
    out = torch.empty((B, Tq, H, D), dtype=q.dtype, device=q.device)
    pitch = _pitch(Tq)
    lse = torch.empty((B, H, pitch), dtype=torch.float32, device=q.device) if training else None
    sizes = (_CODES[q.dtype], B, H, k.shape[2], Tq, k.shape[1], D)
    if tensor_cores(q, k, v):
        q, k, v = _tiles(q), _tiles(k), _tiles(v)
        lo = torch.empty_like(out) if training else None
        code = launcher("kb200_attention_rules_fwd_sm100", [_V] * 6 + [_I, _V] + [_I] * 7 + [_V] + _RULES)(
            q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(lo), _ptr(lse), pitch, strides(q, k, v), *sizes, _err_flag(q.device).data_ptr(),
            *_tail(rules, ranges))
        kops._check(code, "attention_rules_fwd_sm100")
        return out, lse, lo
    code = launcher("kb200_attention_rules_fwd", [_V] * 5 + [_I, _V] + [_I] * 7 + _RULES)(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), _ptr(lse), pitch, strides(q, k, v), *sizes, *_tail(rules, ranges))
    kops._check(code, "attention_rules_fwd")
    return out, lse, None


def backward(q, k, v, out, lo, lse, grad_out, rules, ranges, want_q, want_kv):
    B, Tq, H, D = q.shape
    Tk, Hkv, pitch = k.shape[1], k.shape[2], lse.shape[2]
    tensor = tensor_cores(q, k, v)
    grad_out = unit(grad_out)
    if tensor:
        q, k, v, grad_out = _tiles(q), _tiles(k), _tiles(v), _tiles(grad_out)
    delta = torch.empty_like(lse)
    code = launcher("kb200_attention_rules_delta", [_V] * 5 + [_I] * 6 + [_V])(
        out.data_ptr(), _ptr(lo), grad_out.data_ptr(), strides(grad_out), delta.data_ptr(), pitch, _CODES[q.dtype], B, H, Tq, D, kops._stream())
    kops._check(code, "attention_rules_delta")
    dq = torch.empty((B, Tq, H, D), dtype=q.dtype, device=q.device) if want_q else None
    dk, dv = (torch.empty((B, Tk, Hkv, D), dtype=q.dtype, device=q.device) if want_kv else None for _ in range(2))
    name = "kb200_attention_rules_bwd_sm100" if tensor else "kb200_attention_rules_bwd"
    code = launcher(name, [_V] * 7 + [_I] + [_V] * 3 + [_I] * 7 + ([_V] if tensor else []) + _RULES)(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), grad_out.data_ptr(), strides(q, k, v, grad_out), lse.data_ptr(), delta.data_ptr(), pitch, _ptr(dq), _ptr(dk), _ptr(dv),
        _CODES[q.dtype], B, H, Hkv, Tq, Tk, D, *((_err_flag(q.device).data_ptr(),) if tensor else ()), *_tail(rules, ranges))
    kops._check(code, name[6:])
    return dq, dk, dv


class RuleAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, prefix, rows, keys, rules, plain):
        ranges = segment_ranges(rules)
        out, lse, lo = forward(q, k, v, rules, ranges, training=True)
        # the rules' tensors are saved too: one that is written to before the backward pass is an error, as for any operand
        ctx.save_for_backward(q, k, v, out, lo, lse, *ranges, slopes, prefix, rows, keys)
        ctx.rules, ctx.plain = rules._replace(slopes=None, prefix=None, segments=None), plain
        return out

    @staticmethod
    def backward(ctx, grad_out):
        q, k, v, out, lo, lse, range_q, range_k, slopes, prefix, rows, keys = ctx.saved_tensors
        rules = ctx.rules._replace(slopes=slopes, prefix=prefix, segments=None if rows is None else (rows, keys))
        need = ctx.needs_input_grad
        if torch.is_grad_enabled():  # the gradient is differentiated in its turn
            wanted = [t for t, n in zip((q, k, v), need) if n]
            given = iter(torch.autograd.grad(ctx.plain(q, k, v, rules), wanted, grad_out, create_graph=True))
            grads = [next(given) if n else None for n in need[:3]]
        else:
            dq, dk, dv = backward(q, k, v, out, lo, lse, grad_out, rules, (range_q, range_k), need[0], need[1] or need[2])
            grads = [dq, dk if need[1] else None, dv if need[2] else None]
        return (*grads, None, None, None, None, None, None)


def attention(q, k, v, rules, plain):
    """Attention on this package's kernels, or ``None`` when the call does not fit them.  ``plain(q, k, v, rules)``: the form that second
    derivatives go through."""
    if (q.dtype not in _CODES or k.dtype != q.dtype or v.dtype != q.dtype or k.shape != v.shape or k.shape[0] != q.shape[0] or k.shape[-1] != q.shape[-1]
            or not q.device == k.device == v.device or 0 in q.shape or 0 in k.shape or q.shape[2] % k.shape[2] or q.shape[-1] > MAX_HEAD):
        return None
    if torch.is_autocast_enabled("cuda"):
        return None
    if ((q.shape[1] + 31) // 32) * q.shape[2] * q.shape[0] >= 1 << 31 or ((k.shape[1] + 31) // 32) * q.shape[2] * q.shape[0] >= 1 << 31:
        return None
    q, k, v = unit(q), unit(k), unit(v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        rows, keys = rules.segments or (None, None)
        return RuleAttention.apply(q, k, v, rules.slopes, rules.prefix, rows, keys, rules, plain)
    return forward(q, k, v, rules, segment_ranges(rules), training=False)[0]
