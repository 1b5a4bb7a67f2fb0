"""Front-end of the kernels for attention over a paged key/value cache (``csrc/attention_cache.cu``)."""

import ctypes
import functools

import torch

from keras_b200.kernels import attention_rules as rules_mod
from keras_b200.kernels import ops as kops

_V, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float


@functools.lru_cache(maxsize=256)
def _work(device, *sizes):
    """Floats of workspace at these sizes on the current device."""
    fn = kops._lib().kb200_attention_cache_work
    fn.argtypes, fn.restype = [_I] * 7, ctypes.c_longlong
    return fn(*sizes)


def attention(q, k, v, pool_k, pool_v, pages, lengths, scale, cap, slopes, window):
    """The attention of new tokens over their cache, which gets their keys and values; ``None`` when the call does not fit the kernel."""
    codes = rules_mod._CODES
    if (q.dtype not in codes or 0 in q.shape or 0 in pool_k.shape or pages.shape[1] == 0 or q.shape[-1] > rules_mod.MAX_HEAD or pool_k.stride(-1) != 1
            or pool_k.stride() != pool_v.stride() or k.shape != v.shape):
        return None
    B, T, H, D = q.shape
    Hkv = k.shape[2]
    if B * Hkv * -(-T * (H // Hkv) // 16) >= 1 << 27:
        return None
    q, k, v = (rules_mod.unit(t) for t in (q, k, v))
    out = torch.empty((B, T, H, D), dtype=q.dtype, device=q.device)
    pool = [pool_k.stride(i) for i in (0, 1, 2)]
    flat = list(rules_mod.strides(q, k, v)) + pool
    pages, lengths = pages.contiguous(), lengths.contiguous()
    fn = rules_mod.launcher("kb200_attention_cache", [_V] * 10 + [_L] + [_I] * 9 + [_F, _F, _V, _I, _V])
    floats = _work(q.device.index, B, H, Hkv, T, D, pool_k.shape[1], pages.shape[1])
    # from the caching allocator, for this call and stream alone: a recorded graph has its own
    work = torch.empty(floats, dtype=torch.float32, device=q.device) if floats else None
    code = fn(q.data_ptr(), k.data_ptr(), v.data_ptr(), pool_k.data_ptr(), pool_v.data_ptr(), out.data_ptr(), pages.data_ptr(), lengths.data_ptr(),
              (ctypes.c_longlong * len(flat))(*flat), None if work is None else work.data_ptr(), floats, codes[q.dtype], B, H, Hkv, T, D, pool_k.shape[0], pool_k.shape[1], pages.shape[1], scale, cap or 0.0,
              None if slopes is None else slopes.data_ptr(), min(window or 0, 1 << 30), kops._stream())
    kops._check(code, "attention_cache")
    for pool in (pool_k, pool_v):
        if not pool.is_inference():
            torch.autograd.graph.increment_version(pool)
    return out
