"""Front-end of the kernels for attention over a paged key/value cache (``csrc/attention_cache.cu``)."""

import ctypes

import torch

from keras_b200.kernels import attention_rules as rules_mod
from keras_b200.kernels import ops as kops

_V, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float


class Plan:
    """What a call's types, sizes and strides settle: worked out once for each and kept, as a step calls the same layers again and again."""

    __slots__ = ("fits", "unit", "code", "sizes", "out", "strides", "floats")

    def __init__(self, q, k, v, pool_k, pool_v, wide, window):
        B, T, H, D = q.shape
        K = k.shape[2]
        self.fits = (q.dtype in rules_mod._CODES and 0 not in q.shape and 0 not in pool_k.shape and wide != 0 and D <= rules_mod.MAX_HEAD and pool_k.stride(-1) == 1
                     and pool_k.stride() == pool_v.stride() and k.shape == v.shape and B * K * -(-T * (H // K) // 16) < 1 << 27)
        if not self.fits:
            return
        self.unit = D == 1 or q.stride(3) == k.stride(3) == v.stride(3) == 1
        self.code = rules_mod._CODES[q.dtype]
        self.out = (B, T, H, D)
        self.sizes = (B, H, K, T, D, *pool_k.shape[:2], wide)
        flat = [*rules_mod.strides(q, k, v), *pool_k.stride()[:3]]
        self.strides = (ctypes.c_longlong * len(flat))(*flat)
        fn = rules_mod.launcher("kb200_attention_cache_work", [_I] * 8)
        fn.restype = _L
        self.floats = fn(B, H, K, T, D, pool_k.shape[1], wide, window)


_PLANS = {}
_ARGS = [_V] * 10 + [_L] + [_I] * 9 + [_F, _F, _V, _I, _V]


def _plan_of(q, k, v, pool_k, pool_v, wide, window):
    key = (q.dtype, q.shape, k.shape, v.shape, q.stride(), k.stride(), v.stride(), pool_k.shape, pool_k.stride(), pool_v.stride(), wide, window, q.get_device())
    plan = _PLANS.get(key)
    if plan is None:
        if len(_PLANS) >= 1024:  # sizes that change with every call
            _PLANS.clear()
        plan = _PLANS[key] = Plan(q, k, v, pool_k, pool_v, wide, window)
    return plan


def attention(q, k, v, pool_k, pool_v, pages, lengths, scale, cap, slopes, window):
    """The attention of new tokens over their cache, which gets their keys and values; ``None`` when the call does not fit the kernel."""
    wide, window = pages.shape[1], min(window or 0, 1 << 30)
    plan = _plan_of(q, k, v, pool_k, pool_v, wide, window)
    if not plan.fits:
        return None
    if not plan.unit:
        q, k, v = (rules_mod.unit(t) for t in (q, k, v))
        plan = _plan_of(q, k, v, pool_k, pool_v, wide, window)
    out = q.new_empty(plan.out)
    pages, lengths = pages.contiguous(), lengths.contiguous()
    # from the caching allocator, for this call and stream alone: a recorded graph has its own
    work = q.new_empty(plan.floats, dtype=torch.float32) if plan.floats else None
    code = rules_mod.launcher("kb200_attention_cache", _ARGS)(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), pool_k.data_ptr(), pool_v.data_ptr(), out.data_ptr(), pages.data_ptr(), lengths.data_ptr(), plan.strides,
        None if work is None else work.data_ptr(), plan.floats, plan.code, *plan.sizes, scale, cap or 0.0, None if slopes is None else slopes.data_ptr(),
        window, kops._stream())
    kops._check(code, "attention_cache")
    for pool in (pool_k, pool_v):
        if not pool.is_inference():
            torch.autograd.graph.increment_version(pool)
    return out
