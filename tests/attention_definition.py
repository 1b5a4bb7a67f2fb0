"""Attention by rules in 64 bits, from its definition, pair by pair, and how far an implementation may be from it.

The bounds follow the roundings of an implementation in float32 that stores its results in the type ``t`` (u = eps / 2 of ``t``), and that may round
probabilities and score gradients to ``t`` before the products with them:

* a score is off by at most d = (2 (D + 8) sum |q k| scale + 8 |x| + 8) 2^-24, and 4e-7 cap where there is one (sums of float32 that may truncate, the
  exponential's and the tanh's own error); a probability is then off by 2 d of itself
* out_i:  u |out| + (u + 2 d) sum_j P |v|                        dV_j:  u |dV| + (u + 2 d) sum_i P |dO|
* dS_ij:  (u + 4 d) |dS| + P through (u + 2 d) (sum |dO||out| + sum_j P |dO||v|) + 2 D 2^-24 P sum |dO||v|
* dQ_i, dK_j:  u |dQ| + scale sum |dS's error| |k| and so on

A rounding to float16 is off by a = 2^-25 at least: below 2^-14 its steps are 2^-24 whatever the value, half of which is a.  So each result, each probability
and each score gradient is off by a more, whatever its size.  (The same of bfloat16 and float32, 2^-134 and 2^-150, is nothing.)
"""

import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
F32 = 2.0 ** -24
A = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -25, torch.float32: 0.0}


def visible(T, S, B, causal=False, window=None, prefix=None, segments=None):
    """``[B, T, S]``."""
    out = torch.ones(B, T, S, dtype=torch.bool)
    i, j = torch.arange(T).view(1, T, 1), torch.arange(S).view(1, 1, S)
    if causal:
        out &= (j <= i) | ((j < prefix.cpu().view(B, 1, 1)) if prefix is not None else False)
    if window is not None:
        out &= (i - j).abs() < window
    if segments is not None:
        rows, keys = (t.cpu() for t in segments)
        out &= (rows.unsqueeze(2) == keys.unsqueeze(1)) & (rows.unsqueeze(2) >= 0)
    return out


def attention(q, k, v, seen, cap=None, slopes=None, scale=None, grad_out=None):
    """``{name: (value, bound)}`` for ``out`` and, with ``grad_out``, ``dq``, ``dk`` and ``dv``, in 64 bits on the CPU."""
    dtype = q.dtype
    u = U[dtype]
    a = A[dtype]
    up = 0.0 if dtype == torch.float32 else u
    q, k, v = (t.detach().double().cpu().transpose(1, 2) for t in (q, k, v))
    B, H, T, D = q.shape
    K, S = k.shape[1], k.shape[2]
    group = H // K
    scale = D ** -0.5 if scale is None else scale
    kr, vr = (t.repeat_interleave(group, 1) for t in (k, v))
    x = q @ kr.transpose(2, 3) * scale
    size = q.abs() @ kr.abs().transpose(2, 3) * abs(scale)
    through = torch.ones_like(x)
    if cap is not None:
        t = torch.tanh(x / cap)
        through, x = 1 - t * t, cap * t
    if slopes is not None:
        x = x - torch.as_tensor(slopes).double().cpu().view(1, H, 1, 1) * (torch.arange(T).view(T, 1) - torch.arange(S).view(1, S)).abs().double()
    seen = seen.unsqueeze(1)
    d = torch.where(seen, (2 * (D + 8) * size + 8 * x.abs() + 8) * F32 + (4e-7 * cap if cap else 0.0), torch.zeros(())).amax(-1, keepdim=True)
    top = torch.where(seen, x, torch.full_like(x, -math.inf)).amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(x - torch.where(top.isinf(), torch.zeros_like(top), top)), torch.zeros_like(x))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    out = p @ vr
    found = {"out": (out.transpose(1, 2), (u * out.abs() + (up + 2 * d) * (p @ vr.abs()) + a * (1 + seen.double() @ vr.abs())).transpose(1, 2) + 1e-30)}
    if grad_out is None:
        return found
    go = grad_out.detach().double().cpu().transpose(1, 2)
    dp = go @ vr.transpose(2, 3)
    delta = (go * out).sum(-1, keepdim=True)
    raw = p * (dp - delta)
    ds = raw * through
    dp_size = go.abs() @ vr.abs().transpose(2, 3)
    own = (u + 2 * d) * ((go.abs() * out.abs()).sum(-1, keepdim=True) + (p * dp_size).sum(-1, keepdim=True)) + 2 * D * F32 * dp_size
    # the derivative of the cap is off by twice the tanh's error, of itself by no more than its own distance from one
    e = a * seen + (up + 4 * d) * ds.abs() + p * through * own + (8 * d / cap * raw.abs() if cap else 0.0)

    def heads(t):
        return t.reshape(B, K, group, S, D).sum(2).transpose(1, 2)

    dq, dk, dv = ds @ kr * scale, heads(ds.transpose(2, 3) @ q) * scale, heads(p.transpose(2, 3) @ go)
    found["dq"] = (dq.transpose(1, 2), (u * dq.abs() + abs(scale) * (e @ kr.abs())).transpose(1, 2) + a + 1e-30)
    found["dk"] = (dk, u * dk.abs() + abs(scale) * heads(e.transpose(2, 3) @ q.abs()) + a + 1e-30)
    found["dv"] = (dv, u * dv.abs() + heads((a * seen + (up + 2 * d) * p).transpose(2, 3) @ go.abs()) + a + 1e-30)
    return found


def check(name, got, found):
    value, bound = found[name]
    got = got.detach().double().cpu()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    off = (got - value).abs()
    worst = (off / bound).max().item() if off.numel() else 0.0
    assert torch.isfinite(got).all() and worst <= 1.0, f"{name}: {worst:.3g} times what roundings explain (off by {off.max().item():.3g})"
    return worst


def pool_of(keys, values, page, spare=2, seed=0, wide=None):
    """Pools and a page table that hold ``[B, S, K, D]``, the pages in no order and with rubbish (NaN) wherever nothing was written."""
    B, S, K, D = keys.shape
    need = max(1, -(-S // page)) if wide is None else wide
    g = torch.Generator().manual_seed(seed)
    table = torch.randperm(B * need + spare, generator=g)[: B * need].reshape(B, need).to(torch.int32)
    pools = []
    for t in (keys, values):
        pool = torch.full((B * need + spare, page, K, D), float("nan"), dtype=t.dtype)
        for b in range(B):
            for n in range(need):
                part = t[b, n * page:(n + 1) * page].cpu()
                pool[table[b, n], : part.shape[0]] = part
        pools.append(pool)
    return pools[0], pools[1], table
