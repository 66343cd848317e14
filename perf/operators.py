"""The generation operators' cases: the gated delta rule, attention over the 8-bit paged cache (with
the append that writes it) and the rules on logits.  `run` computes a case in plain torch operations,
or with the framework's kernels where `own` is true."""
import math
import random

import torch

own = False

BLOCK = 64  # tokens of one cache block
FLT_MIN = torch.finfo(torch.float32).tiny
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # one token of one sequence through a layer of 16 key and 32 value heads: latency
        dict(name="delta_token", op="delta", items=1, lo=1, hi=1, k_heads=16, v_heads=32, dtype="bf16", state="own"),
        # one token of each of 128 running sequences: every state is read and written
        dict(name="delta_tokens", op="delta", items=128, lo=1, hi=1, k_heads=16, v_heads=32, dtype="f16", state="own"),
        # a request's shared prefix of 512 tokens, from nothing
        dict(name="delta_prefix", op="delta", items=1, lo=512, hi=512, k_heads=16, v_heads=32, dtype="bf16", state="none"),
        # 64 packed prompts of 16 to 1024 tokens
        dict(name="delta_ragged", op="delta", items=64, lo=16, hi=1024, k_heads=16, v_heads=32, dtype="f16", state="none"),
        # one long document, continued from a kept state
        dict(name="delta_long", op="delta", items=1, lo=8229, hi=8229, k_heads=16, v_heads=32, dtype="bf16", state="shared"),
        # one token of one sequence after a 512-token prefix and some answer tokens: latency
        dict(name="cache_token", op="cache", items=1, rows=1, lo=543, hi=543, q_heads=32, kv_heads=8, dtype="bf16"),
        # one token of each of 64 running sequences of uneven lengths
        dict(name="cache_tokens", op="cache", items=64, rows=1, lo=1, hi=8191, q_heads=32, kv_heads=8, dtype="f16"),
        # one token of each of 4 sequences with long histories
        dict(name="cache_long", op="cache", items=4, rows=1, lo=60001, hi=65535, q_heads=32, kv_heads=8, dtype="bf16"),
        # a chunk of a long prompt: 1000 new rows over 7000 cached tokens
        dict(name="cache_chunk", op="cache", items=1, rows=1000, lo=7000, hi=7000, q_heads=16, kv_heads=8, dtype="f16"),
        # four prompts written into the cache and read back as values (a cache handed to another program)
        dict(name="cache_write", op="write", items=4, rows=1024, lo=0, hi=300, q_heads=32, kv_heads=8, dtype="bf16"),
        # the next token of the four questions of a request
        dict(name="rules_questions", op="rules", items=4, vocab=151936, lo=512, hi=576, biases=8, dtype="f32"),
        # the next token of 256 running sequences
        dict(name="rules_tokens", op="rules", items=256, vocab=151936, lo=16, hi=2048, biases=64, dtype="bf16"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("delta", "delta", "cache", "cache", "write", "rules"))
    dtype = rng.choice(("bf16", "f16"))
    if op == "delta":
        kh = rng.choice((1, 2, 4, 8, 16))
        vh = kh * rng.choice((1, 2, 3)) if kh < 16 else rng.choice((16, 32))
        hi = _log(rng, 1, 8229)
        lo = hi if rng.random() < 0.5 else max(1, hi // rng.choice((2, 8, 64)))
        # rows of all items together, and their states, stay under the largest listed case's
        items = _log(rng, 1, max(1, min(128, 32000 // hi)))
        return dict(op=op, items=items, lo=lo, hi=hi, k_heads=kh, v_heads=vh, dtype=dtype,
                    state=rng.choice(("own", "none", "shared")))
    if op in ("cache", "write"):
        kv = rng.choice((1, 2, 4, 8))
        qh = kv * rng.choice((1, 2, 4, 5, 8)) if kv < 8 else rng.choice((8, 16, 32))
        rows = 1 if op == "cache" and rng.random() < 0.5 else _log(rng, 2, 1000)
        hi = _log(rng, 1, 65535 if rows == 1 else 8000)
        lo = hi if rng.random() < 0.5 else max(0, hi // rng.choice((2, 8, 64)))
        # cached tokens of all items together: at most the listed cases', less with many rows
        items = _log(rng, 1, max(1, min(64, (260000 if rows == 1 else 8000 * 1000 // rows) // (hi + rows))))
        if op == "write":
            items = min(items, max(1, 4096 // rows))
            lo, hi = min(lo, 1000), min(hi, 1000)
        return dict(op=op, items=items, rows=rows, lo=lo, hi=hi, q_heads=qh, kv_heads=kv, dtype=dtype)
    hi = _log(rng, 1, 4096)
    return dict(op=op, items=_log(rng, 1, 256), vocab=rng.choice((1000, 32000, 128100, 151936, _log(rng, 33, 151936))),
                lo=max(0, hi // rng.choice((1, 2, 16))), hi=hi, biases=rng.choice((0, 1, 7, 64, 300)),
                dtype=rng.choice(("f32", "bf16", "f16")))


# ------------------------------------------------------------------ inputs
def _lengths(case):
    """The items' lengths: part of the case (the same for every seed), the ends of the range among them."""
    r = random.Random(case["items"] * 1000003 + case["hi"])
    n = [r.randint(case["lo"], case["hi"]) for _ in range(case["items"])]
    n[0] = case["hi"]
    if len(n) > 1:
        n[-1] = case["lo"]
    return n


def _starts(lengths):
    at = [0]
    for n in lengths:
        at.append(at[-1] + n)
    return at


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dev = "cuda"

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device=dev).to(dtype)

    def uniform(lo, hi, *shape):
        return torch.rand(shape, generator=gen, device=dev) * (hi - lo) + lo

    dt = TYPES[case["dtype"]]
    op, B = case["op"], case["items"]
    if op == "delta":
        n = _lengths(case)
        at = _starts(n)
        R, Hk, Hv = at[-1], case["k_heads"], case["v_heads"]
        # the projections' outputs after their short convolution: q, k and v side by side in one row
        qkv = normal(R, (2 * Hk + Hv) * 128, dtype=dt)
        q, k, v = (x.view(R, -1, 128) for x in qkv.split((Hk * 128, Hk * 128, Hv * 128), dim=1))
        # decay: a rate per head times a softplus per token; writing strength in (0, 1)
        rate = torch.exp(uniform(math.log(1e-3), math.log(2.0), Hv))
        g = -rate * torch.nn.functional.softplus(normal(R, Hv))
        beta = torch.sigmoid(normal(R, Hv))
        state = None
        if case["state"] != "none":
            state = normal(B if case["state"] == "own" else 1, Hv, 128, 128) * 0.1
        even = min(n) == max(n)
        return dict(op=op, B=B, q=q, k=k, v=v, g=g, beta=beta, state=state, even=even, max_len=max(n),
                    cu=torch.tensor(at, dtype=torch.int32, device=dev), n=torch.tensor(n, device=dev))
    if op in ("cache", "write"):
        n, T, Hq, Hk = _lengths(case), case["rows"], case["q_heads"], case["kv_heads"]
        touched = (BLOCK - 1 + T - 1) // BLOCK + 1  # blocks that T new tokens can reach
        need = [x // BLOCK + touched for x in n]
        pages, width = sum(need), max(need)
        ids = torch.randperm(pages, generator=gen, device=dev).to(torch.int32)
        table = torch.zeros((B, width), dtype=torch.int32)
        where = _starts(need)
        at = torch.tensor(where[:-1])[:, None] + torch.arange(width)[None]
        inside = torch.arange(width)[None] < torch.tensor(need)[:, None]
        table = torch.where(inside.to(dev), ids[at.clamp(max=pages - 1).to(dev)], table.to(dev)).contiguous()

        def codes(*shape):
            return (torch.randn(shape, generator=gen, device=dev, dtype=torch.float16) * 34).clamp_(-127, 127).to(torch.int8)

        s = dict(op=op, B=B, T=T, lengths=torch.tensor(n, dtype=torch.int32, device=dev), touched=touched, max_keys=max(n) + T,
                 k_codes=codes(pages, Hk, BLOCK, 128), v_codes=codes(pages, Hk, 128, BLOCK),
                 k_scales=uniform(0.02, 0.04, pages, Hk), v_scales=uniform(0.02, 0.04, pages, Hk),
                 k_tail=normal(B, Hk, BLOCK, 128, dtype=dt), v_tail=normal(B, Hk, 128, BLOCK, dtype=dt), table=table)
        qkv = normal(B * T, (Hq + 2 * Hk) * 128, dtype=dt)
        s["q"], s["k"], s["v"] = (x.view(B * T, -1, 128) for x in qkv.split((Hq * 128, Hk * 128, Hk * 128), dim=1))
        return s
    V, n = case["vocab"], _lengths(case)
    # logits a few units wide; histories that repeat common tokens; a mask that leaves about a third
    H = max(1, case["hi"])
    skew = uniform(0.0, 1.0, B, H) ** 3
    history = (skew * V).to(torch.int32).clamp(max=V - 1)
    mask = torch.randint(-2**31, 2**31 - 1, (B, (V + 31) // 32), generator=gen, device=dev, dtype=torch.int64).to(torch.int32)
    mask |= torch.randint(-2**31, 2**31 - 1, mask.shape, generator=gen, device=dev, dtype=torch.int64).to(torch.int32) & 0x0F0F0F0F
    bias_ids = bias_values = None
    if case["biases"]:
        k = min(case["biases"], V)
        step = V // k
        bias_ids = (torch.arange(k, device=dev) * step + torch.randint(0, step, (B, k), generator=gen, device=dev)).to(torch.int32)
        bias_values = normal(B, k) * 2
    return dict(op=op, B=B, V=V, logits=normal(B, V).mul_(3).to(dt), history=history,
                history_lengths=torch.tensor(n, dtype=torch.int32, device=dev), repetition=uniform(1.0, 1.3, B),
                presence=uniform(0.0, 0.5, B), frequency=uniform(0.0, 0.2, B), bias_ids=bias_ids, bias_values=bias_values,
                mask=mask)


# ------------------------------------------------------------------ one pass
def run(s):
    if own:
        return _own(s)
    return {"delta": _delta, "cache": _cache, "write": _write, "rules": _rules}[s["op"]](s)


def _own(s):
    import decisive_b200 as db
    if s["op"] == "delta":
        cu = None if s["even"] else s["cu"]
        return db.gated_delta(s["q"], s["k"], s["v"], s["g"], s["beta"], items=s["B"], cu_seqlens=cu, max_len=s["max_len"],
                              state=s["state"])
    if s["op"] == "rules":
        return db.logit_rules(s["logits"], s["history"], s["history_lengths"], repetition=s["repetition"],
                              presence=s["presence"], frequency=s["frequency"], bias_ids=s["bias_ids"],
                              bias_values=s["bias_values"], mask=s["mask"])
    cache = db.KvCache8(s["k_codes"], s["k_scales"], s["v_codes"], s["v_scales"], s["k_tail"], s["v_tail"], s["table"])
    db.kv8_append(cache, s["k"], s["v"], s["lengths"])
    if s["op"] == "write":
        return db.kv8_read(cache, s["lengths"] + s["T"], s["max_keys"])
    out = db.kv8_attention(cache, s["q"], s["lengths"], max_keys=s["max_keys"])
    return out, s["k_tail"], s["v_tail"], s["k_scales"], s["v_scales"]


def _delta(s):
    """q, k: unit length (1e-6 added under the root), q also over sqrt(128).  Up to 16 tokens: token by
    token; more: chunks of 64 with a forward substitution over all chunks at once."""
    B, T, cu, n = s["B"], s["max_len"], s["cu"].long(), s["n"]
    Hk, Hv = s["k"].shape[1], s["v"].shape[1]
    t = torch.arange(T, device=cu.device)
    valid = t < n[:, None]
    rows = (cu[:-1, None] + t).clamp(max=s["q"].shape[0] - 1)

    def padded(x):  # [R, H, ...] -> [B, H, T, ...] with zeros past an item's end
        y = x[rows].float()
        return torch.where(valid.view(B, T, *([1] * (y.dim() - 2))), y, 0.0).transpose(1, 2)

    q, k, v, g, beta = (padded(s[x]) for x in ("q", "k", "v", "g", "beta"))
    q = q * torch.rsqrt((q * q).sum(-1, keepdim=True) + 1e-6) * 128 ** -0.5
    k = k * torch.rsqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    head = torch.arange(Hv, device=q.device) * Hk // Hv
    q, k = q[:, head], k[:, head]
    S = torch.zeros((B, Hv, 128, 128), device=q.device) if s["state"] is None else s["state"].expand(B, -1, -1, -1).clone()
    out = torch.empty_like(v)
    if T <= 16:
        for i in range(T):
            S = S * torch.exp(g[:, :, i])[..., None, None]
            u = beta[:, :, i, None] * (v[:, :, i] - (S @ k[:, :, i, :, None])[..., 0])
            S = S + u[..., :, None] * k[:, :, i, None, :]
            out[:, :, i] = (S @ q[:, :, i, :, None])[..., 0]
    else:
        C, N = 64, (T + 63) // 64

        def chunks(x):
            return torch.nn.functional.pad(x, (0, 0) * (x.dim() - 3) + (0, N * C - T)).view(B, Hv, N, C, *x.shape[3:])

        q, k, v, g, beta = (chunks(x) for x in (q, k, v, g, beta))
        G = g.cumsum(-1)
        lower = torch.ones((C, C), dtype=torch.bool, device=q.device).tril()
        D = torch.where(lower, torch.exp((G[..., :, None] - G[..., None, :]).clamp(max=0.0)), 0.0)
        A = beta[..., None] * D.tril(-1) * (k @ k.transpose(-1, -2))
        inv = torch.eye(C, device=q.device).expand_as(A).clone()
        for i in range(1, C):
            inv[..., i, :i] = -(A[..., i, None, :i] @ inv[..., :i, :i])[..., 0, :]
        W = inv * beta[..., None, :]
        P = D * (q @ k.transpose(-1, -2))
        e = torch.exp(G)[..., None]
        last = torch.exp(G[..., -1:] - G)[..., None]
        out = torch.empty((B, Hv, N, C, 128), device=q.device)
        for c in range(N):
            U = W[:, :, c] @ (v[:, :, c] - e[:, :, c] * (k[:, :, c] @ S.transpose(-1, -2)))
            out[:, :, c] = e[:, :, c] * (q[:, :, c] @ S.transpose(-1, -2)) + P[:, :, c] @ U
            S = S * e[:, :, c, -1, :, None] + (last[:, :, c] * U).transpose(-1, -2) @ k[:, :, c]
        out = out.view(B, Hv, N * C, 128)
    # the items' rows one after another again
    item = torch.searchsorted(cu, torch.arange(s["q"].shape[0], device=cu.device), right=True) - 1
    out = out[item, :, torch.arange(s["q"].shape[0], device=cu.device) - cu[item]]
    return out.to(s["v"].dtype), S


def _append(s):
    """The new tokens into the open blocks; the blocks they fill are quantised, in place."""
    B, T, n, table, W = s["B"], s["T"], s["lengths"].long(), s["table"].long(), s["touched"]
    first = n // BLOCK
    p = first[:, None] * BLOCK + torch.arange(W * BLOCK, device=n.device)  # positions of the blocks reached
    new = ((p >= n[:, None]) & (p < n[:, None] + T))[..., None, None]
    rows = (torch.arange(B, device=n.device)[:, None] * T + p - n[:, None]).clamp(0, B * T - 1)
    old = (p < n[:, None])[..., None, None]
    page = table.gather(1, first[:, None] + torch.arange(W, device=n.device))
    full = ((first[:, None] + torch.arange(1, W + 1, device=n.device)) * BLOCK <= n[:, None] + T)
    for x, tail, codes, scales, flip in ((s["k"], s["k_tail"], s["k_codes"], s["k_scales"], False),
                                         (s["v"], s["v_tail"], s["v_codes"], s["v_scales"], True)):
        kept = (tail.transpose(2, 3) if flip else tail).transpose(1, 2)  # [B, 64, Hk, 128]
        kept = torch.cat((kept, kept.new_zeros((B, (W - 1) * BLOCK, *kept.shape[2:]))), 1)
        y = torch.where(new, x[rows], torch.where(old, kept, torch.zeros_like(kept)))
        z = y.float().view(B, W, BLOCK, -1, 128).transpose(2, 3)  # [B, W, Hk, 64, 128]
        scale = (z.abs().amax((3, 4)) / 127).clamp(min=FLT_MIN)
        code = torch.round(z / scale[..., None, None]).clamp(-127, 127).to(torch.int8)
        code = code.transpose(3, 4) if flip else code
        codes[page] = torch.where(full[..., None, None, None], code, codes[page])
        scales[page] = torch.where(full[..., None], scale, scales[page])
        # what stays open: the block that holds the next position
        open_ = ((n + T) // BLOCK - first)[:, None] * BLOCK + torch.arange(BLOCK, device=n.device)
        keep = open_ + first[:, None] * BLOCK < (n + T)[:, None]
        rest = y[torch.arange(B, device=n.device)[:, None], open_.clamp(max=W * BLOCK - 1)].transpose(1, 2)
        keep = keep[:, None, :, None]
        if flip:
            rest, keep = rest.transpose(2, 3), keep.transpose(2, 3)
        tail.copy_(torch.where(keep, rest, tail))


def _values(s, n, blocks):
    """The cached keys and values of the first `blocks` blocks, f32 [B, Hk, tokens, 128]; n: tokens cached."""
    page = s["table"].long()[:, :blocks]
    L = page.shape[1] * BLOCK
    t = torch.arange(L, device=n.device)
    whole = (t < (n // BLOCK * BLOCK)[:, None])[:, None, :, None]
    inside = (t < n[:, None])[:, None, :, None]
    got = []
    for codes, scales, tail, flip in ((s["k_codes"], s["k_scales"], s["k_tail"], False),
                                      (s["v_codes"], s["v_scales"], s["v_tail"], True)):
        x = codes[page].float() * scales[page][..., None, None]  # [B, blocks, Hk, ., .]
        x = (x.transpose(3, 4) if flip else x).transpose(1, 2).flatten(2, 3)
        y = (tail.transpose(2, 3) if flip else tail).float().repeat(1, 1, page.shape[1], 1)
        got.append(torch.where(whole, x, torch.where(inside, y, 0.0)))
    return got


def _cache(s):
    _append(s)
    B, T, n = s["B"], s["T"], s["lengths"].long()
    q = s["q"].float()
    Hq, Hk = q.shape[1], s["k"].shape[1]
    k, v = _values(s, n + T, (s["max_keys"] + BLOCK - 1) // BLOCK)
    q = q.view(B, T, Hk, Hq // Hk, 128).permute(0, 2, 3, 1, 4).reshape(B, Hk, -1, 128) * 128 ** -0.5
    score = (q @ k.transpose(-1, -2)).view(B, Hk, Hq // Hk, T, -1)
    last = n[:, None] + torch.arange(T, device=n.device)
    seen = torch.arange(k.shape[2], device=n.device) <= last[..., None]
    score = torch.where(seen[:, None, None], score, -math.inf)
    e = torch.exp(score - score.amax(-1, keepdim=True))
    out = (e.flatten(2, 3) @ v).view(B, Hk, Hq // Hk, T, 128) / e.sum(-1, keepdim=True)
    out = out.permute(0, 3, 1, 2, 4).reshape(B * T, Hq, 128).to(s["q"].dtype)
    return out, s["k_tail"], s["v_tail"], s["k_scales"], s["v_scales"]


def _write(s):
    _append(s)
    k, v = _values(s, s["lengths"].long() + s["T"], (s["max_keys"] + BLOCK - 1) // BLOCK)
    return k[:, :, :s["max_keys"]].transpose(1, 2).contiguous(), v[:, :, :s["max_keys"]].transpose(1, 2).contiguous()


def _rules(s):
    B, V = s["B"], s["V"]
    x = s["logits"].float()
    dev = x.device
    count = torch.zeros((B, V), device=dev)
    inside = torch.arange(s["history"].shape[1], device=dev) < s["history_lengths"][:, None]
    count.scatter_add_(1, s["history"].long(), inside.float())
    rho = s["repetition"][:, None]
    there = count > 0
    x = torch.where(there, torch.where(x > 0, x / rho, x * rho), x)
    x = torch.where(there, x - (s["presence"][:, None] + s["frequency"][:, None] * count), x)
    if s["bias_ids"] is not None:
        x = x.scatter_add(1, s["bias_ids"].long(), s["bias_values"])
    bit = (s["mask"][:, :, None] >> torch.arange(32, device=dev, dtype=torch.int32)) & 1
    x = torch.where(bit.view(B, -1)[:, :V] != 0, x, -math.inf)
    top = x.amax(1, keepdim=True)
    none = top == -math.inf
    ids = torch.arange(V, device=dev, dtype=torch.int32)
    best = torch.where((x == top) & ~none, ids, V).amin(1)
    best = torch.where(none[:, 0], -1, best).to(torch.int32)
    lse = torch.where(none, -math.inf, top + torch.log(torch.exp(x - torch.where(none, 0.0, top)).sum(1, keepdim=True)))[:, 0]
    return x, best, lse


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    B = case["items"]
    n = _lengths(case)
    if case["op"] == "delta":
        R, Hk, Hv = sum(n), case["k_heads"], case["v_heads"]
        states = B + {"own": B, "shared": 1, "none": 0}[case["state"]]
        return {"bytes": R * (2 * Hk + 2 * Hv) * 128 * size + R * Hv * 8 + states * Hv * 128 * 128 * 4,
                "flops": R * Hv * 7 * 128 * 128}
    if case["op"] in ("cache", "write"):
        T, Hq, Hk = case["rows"], case["q_heads"], case["kv_heads"]
        new = 2 * B * T * Hk * 128
        filled = sum((x + T) // BLOCK - x // BLOCK for x in n)
        tail = 2 * sum(min((x + T) % BLOCK, T) + (x % BLOCK if (x + T) // BLOCK > x // BLOCK else 0) for x in n) * Hk * 128 * size
        append = new * size + tail + filled * Hk * 2 * (BLOCK * 128 + 4)
        keys = sum(x + T for x in n)
        codes = 2 * Hk * sum((x + T) // BLOCK * (BLOCK * 128 + 4) + (x + T) % BLOCK * 128 * size for x in n)
        if case["op"] == "write":
            return {"bytes": append + codes + 2 * B * (max(n) + T) * Hk * 128 * 4, "flops": keys * Hk * 128 * 4}
        pairs = sum(x * T + T * (T + 1) // 2 for x in n)
        return {"bytes": append + codes + 2 * B * T * Hq * 128 * size, "flops": 4 * 128 * Hq * pairs}
    V = case["vocab"]
    return {"bytes": B * (V * (size + 4) + (V + 31) // 32 * 4 + case["biases"] * 8) + 4 * sum(n), "flops": 6 * B * V}


# ------------------------------------------------------------------ 64 bits, from the definitions
def exact(case, seed):
    s = prepare(case, seed)
    return {"delta": _exact_delta, "cache": _exact_cache, "write": _exact_write, "rules": _exact_rules}[s["op"]](s)


def _exact_delta(s):
    """The recurrence token by token, the items that are still running together."""
    dev = s["q"].device
    n = s["n"].tolist()
    begin = s["cu"].tolist()
    Hk, Hv = s["k"].shape[1], s["v"].shape[1]
    r = torch.tensor([h * Hk // Hv for h in range(Hv)], device=dev)
    S = torch.zeros((s["B"], Hv, 128, 128), dtype=torch.float64, device=dev)
    if s["state"] is not None:
        S += s["state"].double()
    out = torch.zeros(s["v"].shape, dtype=torch.float64, device=dev)
    order = sorted(range(s["B"]), key=lambda b: -n[b])
    S = S[order]
    base = torch.tensor([begin[b] for b in order], device=dev)
    lens = [n[b] for b in order]
    live = len(order)
    q64, k64 = s["q"].double(), s["k"].double()
    q64 = q64 / torch.sqrt((q64 ** 2).sum(-1, keepdim=True) + 1e-6) / math.sqrt(128)
    k64 = k64 / torch.sqrt((k64 ** 2).sum(-1, keepdim=True) + 1e-6)
    v64, decay, b64 = s["v"].double(), torch.exp(s["g"].double()), s["beta"].double()
    for t in range(max(n)):
        while lens[live - 1] <= t:
            live -= 1
        at = base[:live] + t
        k, q, v = k64[at][:, r], q64[at][:, r], v64[at]
        H = S[:live]
        H *= decay[at][..., None, None]
        u = b64[at][..., None] * (v - torch.einsum("bhvk,bhk->bhv", H, k))
        H += torch.einsum("bhv,bhk->bhvk", u, k)
        out[at] = torch.einsum("bhvk,bhk->bhv", H, q)
    back = torch.empty_like(S)
    back[order] = S
    return out, back


def _exact_tokens(s, b):
    """Item b's tokens after the append, [tokens, Hk, 128] keys and values in 64 bits."""
    n, T = int(s["lengths"][b]), s["T"]
    pages = s["table"][b].tolist()
    both = []
    for x, codes, scales, tail, flip in ((s["k"], s["k_codes"], s["k_scales"], s["k_tail"], False),
                                         (s["v"], s["v_codes"], s["v_scales"], s["v_tail"], True)):
        kept, done = [], n // BLOCK
        if done:
            at = torch.tensor(pages[:done], device=x.device)
            c = codes[at].double() * scales[at].double()[..., None, None]
            c = c.permute(0, 3, 1, 2) if flip else c.permute(0, 2, 1, 3)
            kept.append(c.reshape(done * BLOCK, -1, 128))
        open_ = tail[b].permute(2, 0, 1) if flip else tail[b].permute(1, 0, 2)
        fresh = torch.cat((open_[:n % BLOCK], x[b * T:(b + 1) * T])).double()
        count = fresh.shape[0] // BLOCK
        whole = fresh[:count * BLOCK].view(count, BLOCK, x.shape[1], 128)
        step = (whole.abs().amax((1, 3), keepdim=True) / 127).clamp(min=FLT_MIN)
        kept += [(torch.round(whole / step) * step).view(count * BLOCK, x.shape[1], 128), fresh[count * BLOCK:]]
        both.append(torch.cat(kept))
    return both


def _exact_cache(s):
    T, outs = s["T"], []
    Hq, Hk = s["q"].shape[1], s["k"].shape[1]
    for b in range(s["B"]):
        k, v = _exact_tokens(s, b)
        n = k.shape[0] - T
        rows = []
        for h in range(Hq):
            m = h // (Hq // Hk)
            a = (s["q"][b * T:(b + 1) * T, h].double() @ k[:, m].T) / math.sqrt(128)
            if T > 1:
                a = a.masked_fill(torch.arange(n + T, device=a.device)[None] > n + torch.arange(T, device=a.device)[:, None], -math.inf)
            rows.append(torch.softmax(a, -1) @ v[:, m])
        outs.append(torch.stack(rows, 1))
    return torch.cat(outs), None, None, None, None


def _exact_write(s):
    got = []
    for which in (0, 1):
        x = torch.zeros((s["B"], s["max_keys"], s["k"].shape[1], 128), dtype=torch.float64, device=s["k"].device)
        for b in range(s["B"]):
            y = _exact_tokens(s, b)[which]
            x[b, :y.shape[0]] = y
        got.append(x)
    return tuple(got)


def _exact_rules(s):
    outs, ids, sums = [], [], []
    V, dev = s["V"], s["logits"].device
    for b in range(s["B"]):
        x = s["logits"][b].double()
        c = torch.bincount(s["history"][b, :int(s["history_lengths"][b])].long(), minlength=V).double()
        rho, pres, freq = (s[w][b].double() for w in ("repetition", "presence", "frequency"))
        y = torch.where(x > 0, x / rho, x * rho) - pres - freq * c
        x = torch.where(c > 0, y, x)
        if s["bias_ids"] is not None:
            x[s["bias_ids"][b].long()] += s["bias_values"][b].double()
        word = s["mask"][b].long() & 0xFFFFFFFF
        v = torch.arange(V, device=dev)
        x[(word[v // 32] >> (v % 32)) % 2 == 0] = -math.inf
        outs.append(x)
        sums.append(torch.logsumexp(x, 0))
    return torch.stack(outs), None, torch.stack(sums)
