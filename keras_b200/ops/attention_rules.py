"""Attention whose scores and masks follow rules, and attention over a paged cache: checks of the arguments, the plain forms, and the way to
the kernels.  ``ops.dot_product_attention`` is the entry.
"""

import math
import numbers
from collections.abc import Mapping

import torch

from keras_b200.core.tensor import convert_to_tensor
from keras_b200.kernels import attention_rules as kernel_rules
from keras_b200.kernels import dispatch

Rules = kernel_rules.Rules
_INT32 = torch.iinfo(torch.int32)
_WIDE = (torch.int64, torch.uint32)


def _refuse(text):
    raise ValueError(f"`dot_product_attention`: {text}")


def _number(value, name):
    if isinstance(value, (bool, torch.Tensor)) or not isinstance(value, numbers.Real) or not math.isfinite(value):
        _refuse(f"`{name}` has to be a finite number. Received: {name}={value}")
    return float(value)


def soft_cap(value):
    value = _number(value, "attn_logits_soft_cap")
    if value <= 0:
        _refuse(f"`attn_logits_soft_cap` has to be positive. Received: attn_logits_soft_cap={value}")
    return value


def window(value):
    if isinstance(value, bool) or not isinstance(value, numbers.Integral) or value <= 0:
        _refuse(f"`sliding_window` has to be `None` or a positive integer. Received: sliding_window={value}")
    return int(value)


def slopes(value, heads, device):
    value = value if isinstance(value, torch.Tensor) else convert_to_tensor(value, dtype="float32").to(device)
    if tuple(value.shape) != (heads,):
        _refuse(f"`distance_slopes` has to hold one number a query head, shape ({heads},). Received: shape {tuple(value.shape)}")
    if value.device != device:
        _refuse(f"`distance_slopes` has to be on the device of the query. Received: {value.device} and {device}")
    if value.requires_grad:
        _refuse("`distance_slopes` are constants: a tensor that requires a gradient gets none.")
    return value.to(torch.float32).contiguous()


def _integers(value, name, shape, device):
    """An integer tensor of that shape on that device."""
    value = convert_to_tensor(value) if not isinstance(value, torch.Tensor) else value
    if value.dtype.is_floating_point or value.dtype.is_complex or value.dtype in (torch.bool, torch.uint64):
        _refuse(f"`{name}` has to be of an integer type. Received: {value.dtype}")
    if tuple(value.shape) != shape:
        _refuse(f"`{name}` has to have the shape {shape}. Received: {tuple(value.shape)}")
    if value.device != device:
        value = value.to(device) if value.device.type == "cpu" else _refuse(f"`{name}` has to be on the device of the query. Received: {value.device} and {device}")
    return value


def _whole(value, name, shape, device):
    """The same as int32; what does not fit is held at the type's ends."""
    value = _integers(value, name, shape, device)
    if value.dtype in _WIDE:
        value = value.to(torch.int64).clamp(_INT32.min, _INT32.max)
    return value.to(torch.int32).contiguous()


def _ids(*tensors):
    """Segment ids as int32.  Wider ones may differ in bits that int32 has no place for (a document's hash): they become their places in the order of a
    sequence's ids, which are equal where the ids are."""
    if not any(t.dtype in _WIDE for t in tensors):
        return tuple(t.to(torch.int32).contiguous() for t in tensors)
    tensors = [t.to(torch.int64).contiguous() for t in tensors]
    order = torch.cat(tensors, dim=1).sort(dim=1).values if len(tensors) > 1 else tensors[0].sort(dim=1).values
    return tuple(torch.searchsorted(order, t, out_int32=True).masked_fill_(t < 0, -1) for t in tensors)


def segments(value, B, T, S, device):
    if isinstance(value, tuple):
        if len(value) != 2:
            _refuse("`segment_ids` has to be one tensor, or a tuple of those of the rows and of the keys.")
        return _ids(_integers(value[0], "segment_ids", (B, T), device), _integers(value[1], "segment_ids", (B, S), device))
    if T != S:
        _refuse("`segment_ids` has to be a tuple of those of the rows and of the keys where their lengths differ.")
    value, = _ids(_integers(value, "segment_ids", (B, T), device))
    return value, value


def _heads(q, k, v):
    if q.shape[0] != k.shape[0] or k.shape[:3] != v.shape[:3] or q.shape[3] != k.shape[3]:
        _refuse(f"query, key and value do not belong together. Received: query.shape={tuple(q.shape)}, key.shape={tuple(k.shape)}, value.shape={tuple(v.shape)}")
    if k.shape[2] == 0 or q.shape[2] % k.shape[2]:
        _refuse(f"the query's heads have to be a multiple of the key's. Received: {q.shape[2]} and {k.shape[2]}")


def make(q, k, v, scale, is_causal, cap, distance_slopes, sliding_window, segment_ids, prefix_lengths):
    """The checked rules of a call."""
    _heads(q, k, v)
    B, T, H, _ = q.shape
    S = k.shape[1]
    if prefix_lengths is not None and not is_causal:
        _refuse("`prefix_lengths` says how many keys are seen in spite of a causal mask: it needs `is_causal=True`.")
    return Rules(
        scale=float(scale), cap=None if cap is None else soft_cap(cap), slopes=None if distance_slopes is None else slopes(distance_slopes, H, q.device),
        causal=bool(is_causal), window=None if sliding_window is None else window(sliding_window),
        prefix=None if prefix_lengths is None else _whole(prefix_lengths, "prefix_lengths", (B,), q.device),
        segments=None if segment_ids is None else segments(segment_ids, B, T, S, q.device))


def _visible(rules, B, T, S, device):
    """Which keys a row sees, as a bool tensor that broadcasts against ``[B, H, T, S]``, or ``None`` for all."""
    i = torch.arange(T, device=device)[:, None]
    j = torch.arange(S, device=device)[None, :]
    seen = None
    if rules.causal:
        seen = j <= i
        if rules.prefix is not None:
            seen = seen | (j < rules.prefix[:, None, None, None])
    if rules.window is not None:
        near = (i - j).abs() < rules.window
        seen = near if seen is None else seen & near
    if rules.segments is not None:
        rows, keys = rules.segments
        same = ((rows[:, :, None] == keys[:, None, :]) & (rows >= 0)[:, :, None])[:, None]
        seen = same if seen is None else seen & same
    return seen


def _weighted(x, seen, values):
    """softmax(x) over the visible keys times the values; rows that see nothing are zero, with zero gradients."""
    if seen is None:
        return torch.matmul(torch.softmax(x, dim=-1), values)
    x = x.masked_fill(~seen, torch.finfo(x.dtype).min)
    return torch.matmul(torch.softmax(x, dim=-1).masked_fill(~seen, 0.0), values)


def plain(q, k, v, rules, bias=None, mask=None):
    """The rules in elementary operations, float32 or wider; for the CPU, for second derivatives, and together with a bias or a mask."""
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    B, T, H, _ = q.shape
    S, K = k.shape[1], k.shape[2]
    qh, kh, vh = (t.to(wide).transpose(1, 2) for t in (q, k, v))
    if K != H:
        kh, vh = (t.repeat_interleave(int(H // K), dim=1) for t in (kh, vh))  # a trace's sizes are tensors of the host
    x = torch.matmul(qh, kh.transpose(-1, -2)) * rules.scale
    if rules.cap is not None:
        x = rules.cap * torch.tanh(x / rules.cap)
    if rules.slopes is not None:
        distance = (torch.arange(T, device=q.device)[:, None] - torch.arange(S, device=q.device)[None, :]).abs()
        x = x - rules.slopes.to(x.dtype)[:, None, None] * distance.to(x.dtype)
    if bias is not None:
        x = x + bias.to(x.dtype)
    seen = _visible(rules, B, T, S, q.device)
    if mask is not None:
        mask = mask.to(torch.bool)
        seen = mask if seen is None else seen & mask
    return _weighted(x, seen, vh).to(q.dtype).transpose(1, 2)


def attend(q, k, v, rules, bias, mask, kernels):
    if kernels and bias is None and mask is None:
        out = dispatch.rule_attention(q, k, v, rules, plain)
        if out is not None:
            return out
    return plain(q, k, v, rules, bias, mask)


def capped(q, k, v, scale, is_causal, cap):
    """A call whose only rule is the cap, on the kernels, or ``None``: what they do not take, or not as fast, stays with the library's operations."""
    if not dispatch.enabled(q) or not kernel_rules.cap_pays(q, k, v, is_causal):  # in this order: an export's sizes decide nothing
        return None
    if isinstance(cap, (bool, torch.Tensor)) or not isinstance(cap, numbers.Real) or not 0 < cap < math.inf or isinstance(scale, torch.Tensor):
        return None
    return kernel_rules.attention(q, k, v, Rules(float(scale), float(cap), None, bool(is_causal), None, None, None), plain)


# ------------------------------------------------------------------------------------------------ the paged cache
_CACHE = {"key", "value", "pages", "lengths"}


def _cache_parts(cache, q, k, v):
    if not isinstance(cache, Mapping) or cache.keys() != _CACHE:
        _refuse("`cache` has to be a dict of `key`, `value`, `pages` and `lengths`.")
    pool_k, pool_v, pages, lengths = (cache[n] for n in ("key", "value", "pages", "lengths"))
    for name, t in cache.items():
        if not isinstance(t, torch.Tensor):
            _refuse(f"`cache['{name}']` has to be a tensor, which the call can write to. Received: {type(t).__name__}")
        if t.device != q.device:
            _refuse(f"the cache has to be on the device of the query. Received: {t.device} and {q.device}")
    if pool_k.ndim != 4 or pool_k.shape != pool_v.shape or tuple(pool_k.shape[2:]) != (k.shape[2], k.shape[3]) or pool_k.shape[1] == 0:
        _refuse("`cache['key']` and `cache['value']` have to be pools of one shape, [pages, positions, key heads, head size]. "
                f"Received: {tuple(pool_k.shape)} and {tuple(pool_v.shape)} for keys of {tuple(k.shape)}")
    if pool_k.dtype != q.dtype or pool_v.dtype != q.dtype:
        _refuse(f"the cache has to be of the type of query, key and value. Received: {pool_k.dtype}, {pool_v.dtype} and {q.dtype}")
    if pool_k.requires_grad or pool_v.requires_grad:
        _refuse("a cache takes no part in gradients.")
    if pages.dtype != torch.int32 or pages.ndim != 2 or pages.shape[0] != q.shape[0]:
        _refuse(f"`cache['pages']` has to be int32 of [batch, pages a sequence]. Received: {pages.dtype} {tuple(pages.shape)}")
    if lengths.dtype != torch.int32 or tuple(lengths.shape) != (q.shape[0],):
        _refuse(f"`cache['lengths']` has to be int32 of [batch]. Received: {lengths.dtype} {tuple(lengths.shape)}")
    return pool_k, pool_v, pages, lengths


def _plain_cached(q, k, v, pool_k, pool_v, pages, lengths, rules):
    wide = torch.float64 if q.dtype == torch.float64 else torch.float32
    B, T, H, D = q.shape
    K, page, wide_pages = k.shape[2], pool_k.shape[1], pages.shape[1]
    S = wide_pages * page
    n = lengths.long()
    at = n[:, None] + torch.arange(T, device=q.device)
    key = torch.arange(S, device=q.device)
    back = at[:, :, None] - key  # [B, T, S]: how far a position lies back
    seen = (back >= 0) & (n >= 0)[:, None, None]
    if rules.window is not None:
        seen = seen & (back < rules.window)
    there = (pages >= 0) & (pages < pool_k.shape[0])
    missing = seen & ~there.repeat_interleave(page, dim=1)[:, None, :]
    bad = (missing.any(dim=-1) | (at >= S)) & (n >= 0)[:, None]  # rows that see a position without a page
    if q.device.type == "cpu" and bool(bad.any()):
        _refuse("the cache has no page for a position that the call reads or writes.")
    slot = (at // page).clamp(0, max(wide_pages - 1, 0))
    keep = (n >= 0)[:, None] & (at < S)
    if wide_pages:
        keep = keep & torch.gather(there, 1, slot)
        to = torch.gather(pages.long(), 1, slot)[keep]
        pool_k[to, (at % page)[keep]] = k[keep]
        pool_v[to, (at % page)[keep]] = v[keep]
    taken = torch.where(there, pages, torch.zeros_like(pages)).long()
    ks, vs = (pool[taken].reshape(B, S, K, D) for pool in (pool_k, pool_v))
    used = seen.any(dim=1)[:, :, None, None] & there.repeat_interleave(page, dim=1)[:, :, None, None]
    ks, vs = (torch.where(used, t, torch.zeros_like(t)).to(wide).transpose(1, 2).repeat_interleave(int(H // K), dim=1) for t in (ks, vs))
    x = torch.matmul(q.to(wide).transpose(1, 2), ks.transpose(-1, -2)) * rules.scale
    if rules.cap is not None:
        x = rules.cap * torch.tanh(x / rules.cap)
    if rules.slopes is not None:
        x = x - rules.slopes.to(x.dtype)[:, None, None] * back[:, None].to(x.dtype)
    out = _weighted(x, seen[:, None], vs).transpose(1, 2)
    return torch.where(bad[:, :, None, None], torch.full_like(out, math.nan), out).to(q.dtype)


def attend_cached(q, k, v, cache, scale, cap, distance_slopes, sliding_window, kernels):
    _heads(q, k, v)
    if k.shape != v.shape or q.shape[1] != k.shape[1]:
        _refuse("with a cache, query, key and value are those of the same new tokens, and keys and values of one size. "
                f"Received: query.shape={tuple(q.shape)}, key.shape={tuple(k.shape)}, value.shape={tuple(v.shape)}")
    if not q.device == k.device == v.device:  # the kernels read all three by their address on the query's device
        _refuse(f"query, key and value have to be on one device. Received: {q.device}, {k.device} and {v.device}")
    pool_k, pool_v, pages, lengths = _cache_parts(cache, q, k, v)
    rules = Rules(float(scale), None if cap is None else soft_cap(cap), None if distance_slopes is None else slopes(distance_slopes, q.shape[2], q.device), True,
                  None if sliding_window is None else window(sliding_window), None, None)
    with torch.no_grad():
        if kernels:
            out = dispatch.cached_attention(q, k, v, pool_k, pool_v, pages, lengths, rules)
            if out is not None:
                return out
        return _plain_cached(q, k, v, pool_k, pool_v, pages, lengths, rules)
