"""Attention of decoders: scores with a cap, a bias by distance and masks given as rules, its gradients, and its serving from a paged cache.

Three kinds of pass:

* ``score``   the attention of whole sequences without gradients (scoring, prompts)
* ``train``   the same with the gradients of query, key and value
* ``decode``  the attention of one or a few new tokens a sequence over a paged key/value cache, to which it adds their keys and values

Scores are ``s = scale * q.k``, with a cap ``cap * tanh(s / cap)``, less ``slope * |i - j|`` of the head where there are slopes.  A row sees
the keys that every rule of the case allows:

* ``causal``     keys up to its own position
* ``prefix``     those, and the first keys of the sequence, as many as its prefix is long
* ``window``     (with causal) keys nearer than the window's width
* ``documents``  (with causal) keys of its own document; the end of a sequence is padding, which sees nothing, is seen by nobody and gives zeros
"""

import math
import random

import torch

own = False

_TYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}


# ------------------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one short prompt with capped scores: the latency of a call
        _dense("score_prompt", "score", "bfloat16", 1, 77, 12, 12, 64, cap=30.0),
        # packed documents at the batch, length and heads of the GPT-2 benchmark configuration
        _dense("score_documents", "score", "float16", 16, 1024, 12, 12, 64, rule="documents", mean=300),
        # the 8B decoder configuration at its own context length, with capped scores
        _dense("score_8b", "score", "bfloat16", 2, 4096, 32, 8, 128, cap=50.0),
        # the default float32 policy on a small model with distance slopes, a length that is no multiple of a tile
        _dense("train_small", "train", "float32", 4, 333, 8, 8, 64, slopes=True),
        # the GPT-2 benchmark configuration on packed documents, with capped scores
        _dense("train_documents", "train", "bfloat16", 16, 1024, 12, 12, 64, rule="documents", mean=300, cap=30.0),
        # the 1.3B decoder configuration with distance slopes
        _dense("train_slopes", "train", "bfloat16", 8, 2048, 16, 16, 128, slopes=True),
        # instructions that are read both ways before the answer; few key heads, a head size between the usual ones
        _dense("train_prefix", "train", "float16", 6, 777, 8, 2, 80, rule="prefix", mean=200, cap=50.0),
        # long sequences within a window, shared key heads
        _dense("train_window", "train", "bfloat16", 1, 8192, 32, 8, 128, rule="window", width=1024, cap=50.0),
        # one user's next token: the latency of a step
        _paged("decode_one", "bfloat16", 1, 1, 12, 12, 64, 900, 900, 16),
        # many users at lengths of their own, the heads of the 8B configuration
        _paged("decode_batch", "bfloat16", 64, 1, 32, 8, 128, 200, 4000, 64, cap=50.0),
        # two long contexts: the work is in the length
        _paged("decode_long", "float16", 2, 1, 32, 8, 128, 60000, 65000, 128, slopes=True),
        # a handful of proposed tokens verified at once, within a window
        _paged("decode_verify", "bfloat16", 16, 5, 16, 16, 128, 500, 3001, 32, width=1024),
    ]


def _dense(name, kind, dtype, batch, length, heads, kv_heads, dim, rule="causal", mean=0, width=0, cap=0.0, slopes=False):
    """``mean``: the mean length of documents or prefixes; ``width``: of the window; 0 stands for none."""
    return {"name": name, "kind": kind, "dtype": dtype, "batch": batch, "length": length, "heads": heads, "kv_heads": kv_heads, "dim": dim, "rule": rule,
            "mean": mean, "width": width, "cap": cap, "slopes": slopes}


def _paged(name, dtype, batch, new, heads, kv_heads, dim, shortest, longest, page, width=0, cap=0.0, slopes=False):
    """``new``: tokens a sequence that the call adds; the lengths before it lie between ``shortest`` and ``longest``."""
    return {"name": name, "kind": "decode", "dtype": dtype, "batch": batch, "new": new, "heads": heads, "kv_heads": kv_heads, "dim": dim, "shortest": shortest,
            "longest": longest, "page": page, "width": width, "cap": cap, "slopes": slopes}


def _between(rng, low, high):
    """A whole number, even over the logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    case = _drawn(rng)
    del case["name"]
    return case


def _drawn(rng):
    kind = rng.choice(["score", "train", "decode"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    kv_heads = rng.choice([1, 2, 4, 8, 12])
    heads = kv_heads * rng.choice([1, 1, 2, 4, 7] if kv_heads < 8 else [1, 2, 4])
    dim = rng.choice([64, 64, 128, 128, 32, 48, 80, 96])
    cap = rng.choice([0.0, 20.0, 30.0, 50.0])
    slopes = rng.random() < 0.3
    if kind == "decode":
        longest = _between(rng, 1, 30000)
        shortest = rng.randint(0, longest)
        new = rng.choice([1, 1, 1, 2, 3, 8])
        most = max(1, int(6e7 / (kv_heads * dim * (longest + new))))
        batch = min(_between(rng, 1, 128), most)
        return _paged(None, dtype, batch, new, heads, kv_heads, dim, shortest, longest, rng.choice([16, 16, 32, 64, 128, 256, 24]),
                      width=rng.choice([0, 0, _between(rng, 1, 4096)]), cap=cap, slopes=slopes)
    # a gradient that is nothing but zeros says nothing: no training on single tokens, nor on rows that all see one key
    length = _between(rng, 1 if kind == "score" else 8, 4096)
    pairs = (1e9 if kind == "score" else 4e8) * (1 if dtype != "float32" else 0.25)
    while heads * length * length > pairs:
        length //= 2
    batch = min(_between(rng, 1, 32), max(1, int(pairs / (heads * length * length))))
    rule = rng.choice(["causal", "prefix", "window", "documents"])
    if rule == "causal" and not cap:
        slopes = True
    return _dense(None, kind, dtype, batch, length, heads, kv_heads, dim, rule=rule, mean=_between(rng, 4, max(4, length)) if rule in ("prefix", "documents") else 0,
                  width=_between(rng, 2, max(2, length)) if rule == "window" else 0, cap=cap, slopes=slopes)


# ------------------------------------------------------------------------------------------------ what the sizes of a case leave open
def _layout(case):
    """Whole numbers that go with a case whatever the seed: a document of every token (-1: padding), or the lengths of the prefixes."""
    rng = random.Random(case["length"] * 131 + case["batch"] * 17 + case["mean"])
    B, T, mean = case["batch"], case["length"], case["mean"]
    if case["rule"] == "documents":
        rows = []
        for b in range(B):
            row, n = [], 0
            real = T - (rng.randint(0, T // 8) if b % 2 else 0)
            while len(row) < real:
                row += [n] * max(1, min(real - len(row), round(rng.expovariate(1 / mean))))
                n += 1
            rows.append(row + [-1] * (T - len(row)))
        return rows
    if case["rule"] == "prefix":
        return [rng.randint(0, min(T, 2 * mean)) for _ in range(B)]
    return None


def _lengths(case):
    rng = random.Random(case["longest"] * 131 + case["batch"])
    lengths = [rng.randint(case["shortest"], case["longest"]) for _ in range(case["batch"])]
    lengths[0] = case["longest"]
    return lengths


def _pairs(case):
    """How many (row, key) pairs of one head are visible, over the batch."""
    if case["kind"] == "decode":
        w = case["width"] or 1 << 60
        return sum(min(n + t + 1, w) for n in _lengths(case) for t in range(case["new"]))
    B, T = case["batch"], case["length"]
    causal = T * (T + 1) // 2
    if case["rule"] == "causal":
        return B * causal
    if case["rule"] == "window":
        w = min(case["width"], T)
        return B * (w * (w + 1) // 2 + (T - w) * w)
    if case["rule"] == "prefix":
        return sum(causal + p * (p - 1) // 2 for p in _layout(case))
    total = 0
    for row in _layout(case):
        sizes = {}
        for d in row:
            sizes[d] = sizes.get(d, 0) + 1
        total += sum(n * (n + 1) // 2 for d, n in sizes.items() if d >= 0)
    return total


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    H, K, D = case["heads"], case["kv_heads"], case["dim"]
    pairs = _pairs(case)
    if case["kind"] == "decode":
        w = case["width"] or 1 << 60
        T = case["new"]
        read = sum(min(n, w + T - 1) for n in _lengths(case)) * K * D * 2
        new = case["batch"] * T * (2 * H * D + 4 * K * D)  # query and output; new keys and values read and written
        return {"bytes": size * (read + new), "flops": 4 * D * H * pairs}
    rows = case["batch"] * case["length"] * D
    if case["kind"] == "score":
        return {"bytes": size * rows * (2 * H + 2 * K), "flops": 4 * D * H * pairs}
    return {"bytes": size * rows * (4 * H + 4 * K), "flops": 14 * D * H * pairs}


# ------------------------------------------------------------------------------------------------ inputs
def _slopes(heads):
    """A geometric row of slopes, as models with a bias by distance take them."""
    return [2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype, H, K, D = _TYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    state = {"kind": case["kind"], "cap": case["cap"] or None, "width": case["width"] or None,
             "slopes": torch.tensor(_slopes(H), device="cuda") if case["slopes"] else None, "segments": None, "prefix": None}
    if case["kind"] == "decode":
        B, T, page = case["batch"], case["new"], case["page"]
        lengths = _lengths(case)
        wide = max(-(-(n + T) // page) for n in lengths)
        total = B * wide + 3  # a few pages belong to nobody
        table = torch.randperm(total, generator=g, device="cuda")[: B * wide].reshape(B, wide).to(torch.int32)
        pools = [normal(total, page, K, D) for _ in range(2)]
        return state | {"q": normal(B, T, H, D, scale=3.0), "k": normal(B, T, K, D), "v": normal(B, T, K, D), "pool_k": pools[0], "pool_v": pools[1], "pages": table,
                        "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda")}
    B, T = case["batch"], case["length"]
    state |= {"q": normal(B, T, H, D, scale=3.0), "k": normal(B, T, K, D), "v": normal(B, T, K, D)}
    if case["rule"] == "documents":
        state["segments"] = torch.tensor(_layout(case), dtype=torch.int32, device="cuda")
    if case["rule"] == "prefix":
        state["prefix"] = torch.tensor(_layout(case), dtype=torch.int32, device="cuda")
    if case["kind"] == "train":
        for name in ("q", "k", "v"):
            state[name].requires_grad_(True)
        state["dout"] = normal(B, T, H, D)
    return state


# ------------------------------------------------------------------------------------------------ a pass
def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain_decode(state) if state["kind"] == "decode" else _plain_dense(state)


def _own(s):
    import keras_b200 as keras

    rules = {"attn_logits_soft_cap": s["cap"], "distance_slopes": s["slopes"], "sliding_window": s["width"]}
    if s["kind"] == "decode":
        cache = {"key": s["pool_k"], "value": s["pool_v"], "pages": s["pages"], "lengths": s["lengths"]}
        with torch.no_grad():
            out = keras.ops.dot_product_attention(s["q"], s["k"], s["v"], cache=cache, **rules)
        return out, s["pool_k"], s["pool_v"]
    rules |= {"is_causal": True, "segment_ids": s["segments"], "prefix_lengths": s["prefix"]}
    if s["kind"] == "score":
        with torch.no_grad():
            return keras.ops.dot_product_attention(s["q"], s["k"], s["v"], **rules)
    out = keras.ops.dot_product_attention(s["q"], s["k"], s["v"], **rules)
    return (out.detach(), *torch.autograd.grad(out, (s["q"], s["k"], s["v"]), s["dout"]))


def _plain_dense(s):
    q, k, v = s["q"], s["k"], s["v"]
    B, T, H, D = q.shape
    K = k.shape[2]
    scale = D ** -0.5
    at = torch.arange(T, device=q.device)
    visible = (at[None, :] <= at[:, None])[None]
    if s["prefix"] is not None:
        visible = visible | (at[None, None, :] < s["prefix"][:, None, None])
    if s["width"] is not None:
        visible = visible & ((at[:, None] - at[None, :]).abs() < s["width"])
    if s["segments"] is not None:
        seg = s["segments"]
        visible = visible & (seg[:, :, None] == seg[:, None, :]) & (seg >= 0)[:, :, None]
    visible = visible[:, None]
    q32, k32, v32 = (t.float().transpose(1, 2) for t in (q, k, v))  # [B, heads, T, D]
    kr, vr = (t.repeat_interleave(H // K, dim=1) for t in (k32, v32))
    x = torch.matmul(q32, kr.transpose(2, 3)).mul_(scale)
    through = None
    if s["cap"] is not None:
        t = x.div_(s["cap"]).tanh_()
        if s["kind"] == "train":
            through = 1 - t * t
        x = t * s["cap"]
    if s["slopes"] is not None:
        x = x - s["slopes"][:, None, None] * (at[:, None] - at[None, :]).abs().float()
    x = x.masked_fill_(~visible, -math.inf)
    top = x.amax(dim=-1, keepdim=True)
    p = x.sub_(torch.where(torch.isfinite(top), top, torch.zeros_like(top))).exp_()
    total = p.sum(dim=-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    out = torch.matmul(p, vr)
    if s["kind"] == "score":
        return out.transpose(1, 2).to(q.dtype).contiguous()
    do = s["dout"].float().transpose(1, 2)
    dv = torch.matmul(p.transpose(2, 3), do)
    dp = torch.matmul(do, vr.transpose(2, 3))
    ds = dp.sub_((do * out).sum(dim=-1, keepdim=True)).mul_(p)
    if through is not None:
        ds = ds.mul_(through)
    dq = torch.matmul(ds, kr) * scale
    dk = torch.matmul(ds.transpose(2, 3), q32) * scale
    dk, dv = (t.reshape(B, K, H // K, T, D).sum(dim=2) for t in (dk, dv))
    return tuple(t.transpose(1, 2).to(q.dtype).contiguous() for t in (out, dq, dk, dv))


def _plain_decode(s):
    q, pages = s["q"], s["pages"].long()
    B, T, H, D = q.shape
    K, page = s["k"].shape[2], s["pool_k"].shape[1]
    lengths = s["lengths"].long()
    at = lengths[:, None] + torch.arange(T, device=q.device)  # positions of the new tokens
    slot = torch.gather(pages, 1, at // page)
    s["pool_k"][slot, at % page] = s["k"]
    s["pool_v"][slot, at % page] = s["v"]
    k, v = (pool[pages].reshape(B, -1, K, D) for pool in (s["pool_k"], s["pool_v"]))
    S = k.shape[1]
    key = torch.arange(S, device=q.device)
    far = at[:, :, None] - key  # how far a key lies back
    visible = far >= 0
    if s["width"] is not None:
        visible = visible & (far < s["width"])
    q32 = q.float().reshape(B, T, K, H // K, D).permute(0, 2, 1, 3, 4).reshape(B, K, T * (H // K), D)
    x = torch.matmul(q32, k.float().permute(0, 2, 3, 1)).mul_(D ** -0.5).reshape(B, K, T, H // K, S)
    if s["cap"] is not None:
        x = x.div_(s["cap"]).tanh_().mul_(s["cap"])
    if s["slopes"] is not None:
        x = x - s["slopes"].reshape(K, 1, H // K, 1) * far[:, None, :, None, :].float()
    x = x.masked_fill_(~visible[:, None, :, None, :], -math.inf)
    p = torch.exp(x - x.amax(dim=-1, keepdim=True))
    p = p / p.sum(dim=-1, keepdim=True)
    out = torch.matmul(p.reshape(B, K, -1, S), v.float().transpose(1, 2))
    out = out.reshape(B, K, T, H // K, D).permute(0, 2, 1, 3, 4).reshape(B, T, H, D)
    return out.to(q.dtype), s["pool_k"], s["pool_v"]


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _exact_decode(s) if case["kind"] == "decode" else _exact_dense(s, case["kind"] == "train")


def _head(q, k, v, visible, cap, slope, distance):
    """One head of one sequence in 64 bits."""
    x = (q @ k.T) / math.sqrt(q.shape[1])
    if cap is not None:
        x = cap * torch.tanh(x / cap)
    if slope is not None:
        x = x - slope * distance
    weights = torch.softmax(torch.where(visible, x, torch.full_like(x, -1e300)), dim=1) * visible
    return weights @ v


def _exact_dense(s, train):
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    B, T, H, D = q.shape
    group = H // k.shape[2]
    row = torch.arange(T, device=q.device).unsqueeze(1)
    key = torch.arange(T, device=q.device).unsqueeze(0)
    distance = (row - key).abs().double()
    outs = [torch.zeros_like(t) for t in ((q, q, k, v) if train else (q,))]
    for b in range(B):
        visible = key <= row
        if s["prefix"] is not None:
            visible = visible | (key < int(s["prefix"][b]))
        if s["width"] is not None:
            visible = visible & (distance < s["width"])
        if s["segments"] is not None:
            d = s["segments"][b]
            visible = visible & (d.unsqueeze(1) == d.unsqueeze(0)) & (d.unsqueeze(1) >= 0)
        for h in range(H):
            leaves = [t[b, :, i].clone().requires_grad_(train) for t, i in ((q, h), (k, h // group), (v, h // group))]
            slope = None if s["slopes"] is None else s["slopes"][h].double()
            with torch.set_grad_enabled(train):
                out = _head(*leaves, visible, s["cap"], slope, distance)
            outs[0][b, :, h] = out.detach()
            if train:
                for to, i, grad in zip(outs[1:], (h, h // group, h // group), torch.autograd.grad(out, leaves, s["dout"][b, :, h].double())):
                    to[b, :, i] += grad
    return tuple(outs) if train else outs[0]


def _exact_decode(s):
    q = s["q"].double()
    B, T, H, D = q.shape
    K, page = s["k"].shape[2], s["pool_k"].shape[1]
    out = torch.zeros_like(q)
    for b in range(B):
        n = int(s["lengths"][b])
        used = s["pages"][b, : -(-n // page)].long()
        k, v = (torch.cat([pool[used].reshape(-1, K, D)[:n], new[b]]).double() for pool, new in ((s["pool_k"], s["k"]), (s["pool_v"], s["v"])))
        back = n + torch.arange(T, device=q.device).unsqueeze(1) - torch.arange(n + T, device=q.device).unsqueeze(0)
        visible = back >= 0
        if s["width"] is not None:
            visible = visible & (back < s["width"])
        for h in range(H):
            slope = None if s["slopes"] is None else s["slopes"][h].double()
            out[b, :, h] = _head(q[b, :, h], k[:, h * K // H], v[:, h * K // H], visible, s["cap"], slope, back.double())
    return out, None, None
