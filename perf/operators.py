"""What is measured of the paged K/V cache and of the windowed attention operators.

A streaming model keeps K and V of its past tokens in a paged cache (``cache_write``), attends from
each new chunk, or from one new token per sequence, over it (``paged_attention``), reads stretches of
it back (``cache_read``), and attends over contiguous tensors with a token-exact window and sinks
(``window_attention``).  Where ``own`` is false, ``run`` computes them in elementary torch operations
in 32 bits.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "solattn-amd_b200"))

own = False

E4M3_MAX = 448.0


def listed():
    return [
        # One stream, one new token over a short history: the smallest call, latency alone.
        {"name": "decode one bf16", "op": "paged", "type": "bf16", "batch": 1, "new": 1, "keys": 1000, "heads": 16,
         "kv_heads": 2, "dim": 128, "page": 64, "window": 0, "sinks": 0, "ahead": 0},
        # A serving batch, one new token each, ragged histories, grouped heads.
        {"name": "decode batch bf16", "op": "paged", "type": "bf16", "batch": 64, "new": 1, "keys": 8192, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "window": 0, "sinks": 0, "ahead": 0},
        # The same with an 8-bit cache, smaller heads, odd lengths and small pages.
        {"name": "decode batch e4m3", "op": "paged", "type": "e4m3", "batch": 96, "new": 1, "keys": 12345, "heads": 24,
         "kv_heads": 24, "dim": 64, "page": 16, "window": 0, "sinks": 0, "ahead": 0},
        # A new chunk of a streamed video over a long history, every head its own K/V, the chunk's tokens see each other.
        {"name": "chunk long bf16", "op": "paged", "type": "bf16", "batch": 1, "new": 2048, "keys": 32768, "heads": 24,
         "kv_heads": 24, "dim": 128, "page": 64, "window": 0, "sinks": 0, "ahead": -1},
        # Ragged causal chunks of several streams over an 8-bit cache, with a window and sinks.
        {"name": "chunk ragged e4m3", "op": "paged", "type": "e4m3", "batch": 6, "new": 777, "keys": 9001, "heads": 16,
         "kv_heads": 4, "dim": 128, "page": 32, "window": 4096, "sinks": 100, "ahead": 0},
        # A video transformer's layer with local attention in both directions.
        {"name": "window video", "op": "window", "batch": 1, "new": 16384, "keys": 16384, "heads": 12, "kv_heads": 12,
         "dim": 128, "window": 2048, "sinks": 256, "ahead": 2047},
        # A causal prompt, odd length, grouped heads, narrow window and a few sinks.
        {"name": "window causal odd", "op": "window", "batch": 2, "new": 8191, "keys": 8191, "heads": 16, "kv_heads": 4,
         "dim": 64, "window": 1000, "sinks": 13, "ahead": 0},
        # One new token over contiguous K/V.
        {"name": "window single", "op": "window", "batch": 8, "new": 1, "keys": 5000, "heads": 16, "kv_heads": 4, "dim": 128,
         "window": 4096, "sinks": 64, "ahead": 0},
        # The cache rows of one decoding step.
        {"name": "write step e4m3", "op": "write", "type": "e4m3", "batch": 64, "new": 1, "keys": 4096, "heads": 8,
         "kv_heads": 8, "dim": 128, "page": 64},
        # The rows of a long prompt.
        {"name": "write prompt e4m3", "op": "write", "type": "e4m3", "batch": 2, "new": 16384, "keys": 16384, "heads": 24,
         "kv_heads": 24, "dim": 128, "page": 64},
        # A whole history read back for routed attention.
        {"name": "read long e4m3", "op": "read", "type": "e4m3", "batch": 1, "new": 1, "keys": 32768, "heads": 24,
         "kv_heads": 24, "dim": 128, "page": 64},
        # Short ragged histories read back.
        {"name": "read ragged bf16", "op": "read", "type": "bf16", "batch": 5, "new": 1, "keys": 1000, "heads": 8,
         "kv_heads": 8, "dim": 64, "page": 16},
    ]


def _log(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["paged", "paged", "window", "window", "write", "read"])
    kv_heads = rng.choice([1, 2, 4, 8, 16, 24])
    group = rng.choice([1, 1, 2, 3, 4, 8])
    group = min(group, max(1, 32 // kv_heads))
    c = {"op": op, "kv_heads": kv_heads, "heads": kv_heads * group, "dim": rng.choice([64, 128])}
    if op != "window":
        c["type"] = rng.choice(["bf16", "e4m3"])
        c["page"] = rng.choice([16, 32, 64, 128])
    if op in ("paged", "window"):
        c["window"] = rng.choice([0, _log(rng, 1, 8192)])
        c["sinks"] = rng.choice([0, _log(rng, 1, 512)])
        c["ahead"] = rng.choice([0, 0, -1, _log(rng, 1, 4096)])
        if rng.random() < 0.5:  # one or a few new tokens for each sequence
            c["new"] = rng.choice([1, 1, 2, 3, 5])
            c["batch"] = _log(rng, 1, 64)
            c["keys"] = max(c["new"], _log(rng, 16, 16384))
        else:
            c["batch"] = rng.choice([1, 1, 2, 3])
            c["new"] = _log(rng, 17, 6000)
            c["keys"] = c["new"] if op == "window" and rng.random() < 0.6 else c["new"] + _log(rng, 1, 10000)
        most = 1 << 30  # scores, and key rows below: no dearer than the largest listed case
        while c["batch"] * c["heads"] * c["new"] * c["keys"] > most or c["batch"] * c["keys"] * c["kv_heads"] * c["dim"] > most // 2:
            if c["batch"] > 1:
                c["batch"] //= 2
            else:
                c["new"], c["keys"] = max(1, c["new"] * 3 // 4), max(1, c["keys"] * 3 // 4)
                c["keys"] = max(c["new"], c["keys"])
    else:
        c["batch"] = _log(rng, 1, 16)
        c["new"] = _log(rng, 1, 4000) if op == "write" else 1
        c["keys"] = c["new"] + _log(rng, 1, 4000)
    return c


def _lengths(case):
    """New tokens and keys of each sequence: the first has the case's own, the others fewer (a fixed ragged pattern)."""
    b = np.arange(case["batch"])
    if case["op"] == "window":
        return np.full(len(b), case["new"]), np.full(len(b), case["keys"])
    cut = (b * 0.6180339887498949) % 1.0
    new = np.maximum(1, case["new"] - (0.9 * cut * case["new"]).astype(np.int64))
    keys = np.maximum(new, case["keys"] - (0.8 * ((b * 0.7548776662466927) % 1.0) * case["keys"]).astype(np.int64))
    return new, keys


def _visible(case):
    """Visible (query, key) pairs, and keys that some query sees, summed over the sequences."""
    pairs = rows = 0
    window = case["window"] or 1 << 40
    ahead = case["ahead"] if case["ahead"] >= 0 else 1 << 40
    for n, L in zip(*_lengths(case)):
        p = np.arange(L - n, L)
        high = np.minimum(L - 1, p + ahead) + 1
        low = np.minimum(np.maximum(0, p - window + 1), high)
        sink = np.minimum(np.minimum(case["sinks"], high), low)
        pairs += int((high - low + sink).sum())
        rows += int(high.max() - low.min() + sink.max())
    return pairs, rows


def work(case):
    new, keys = _lengths(case)
    D, Hq, Hkv = case["dim"], case["heads"], case["kv_heads"]
    size = 2 * D if case.get("type", "bf16") == "bf16" else D + 1
    if case["op"] in ("paged", "window"):
        pairs, rows = _visible(case)
        return {"bytes": int(new.sum()) * Hq * D * 4 + rows * Hkv * 2 * size, "flops": 4 * D * Hq * pairs}
    if case["op"] == "write":
        return {"bytes": int(new.sum()) * Hkv * 2 * (2 * D + size), "flops": 0}
    return {"bytes": int(keys.sum()) * Hkv * 2 * size + case["batch"] * case["keys"] * Hkv * 4 * D, "flops": 0}


def _random(case, seed):
    """The case's numbers, from the seed alone."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new, keys = _lengths(case)
    D, Hq, Hkv = case["dim"], case["heads"], case["kv_heads"]

    def rand(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.bfloat16)

    # Keys have a few channels of larger size, as trained models' have.
    gain = torch.ones(D, device="cuda", dtype=torch.bfloat16)
    gain[:: D // 4] = 3
    if case["op"] == "window":
        B = case["batch"]
        q = rand(B, case["new"], Hq, D)
        k, v = rand(B, case["keys"], Hkv, D) * gain, rand(B, case["keys"], Hkv, D)
        return {"q": q, "k": k, "v": v}
    ps = case["page"]
    width = -(-int(keys.max()) // ps)
    used = [-(-int(n) // ps) for n in keys]
    pages = sum(used) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").cpu().numpy()
    table = np.full((len(keys), width), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(used):
        table[b, :n] = order[at:at + n]
        at += n
    starts = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    d = {"table": torch.from_numpy(table), "lengths": torch.from_numpy(keys.astype(np.int32)), "starts": torch.from_numpy(starts)}
    N = int(new.sum())
    pool_k, pool_v = rand(pages, Hkv, ps, D) * gain, rand(pages, Hkv, ps, D)
    d["pool"] = (pool_k, pool_v)
    if case["op"] == "paged":
        d["q"] = rand(N, Hq, D)
    if case["op"] == "write":
        d["k"], d["v"] = rand(N, Hkv, D) * gain, rand(N, Hkv, D)
    return d


def _quantise(x):
    """E4M3 codes and exponents of rows: the least power of two under which the row's largest value is at most 448."""
    x = x.float()
    top = x.abs().amax(dim=-1)
    f, e = torch.frexp(top)
    e = torch.where(top > 0, e - 9 + (f > 0.875).to(e.dtype), torch.full_like(e, -127)).clamp(-127, 127)
    code = (x * ((127 - e.int()) << 23).view(torch.float32)[..., None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
    return code, (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def prepare(case, seed):
    d = _random(case, seed)
    state = {"case": case}
    if case["op"] == "window":
        state.update(q=d["q"], k=d["k"], v=d["v"])
        return state
    pool_k, pool_v = d["pool"]
    if case["type"] == "e4m3":
        (k, ks), (v, vs) = _quantise(pool_k), _quantise(pool_v)
    else:
        k, v, ks, vs = pool_k, pool_v, None, None
    if own:
        from sol_attn_b200 import PagedKVCache, PagedPlan
        state["cache"] = PagedKVCache(k, v, ks, vs)
        state["plan"] = PagedPlan.create(d["table"], d["lengths"], d["starts"], page_size=case["page"]).to("cuda")
    state.update(k_pages=k, v_pages=v, k_scale=ks, v_scale=vs, table=d["table"].cuda(), lengths=d["lengths"].cuda(),
                 starts=d["starts"].cuda(), new=int(max(np.diff(d["starts"].numpy()))))
    for name in ("q", "k", "v"):
        if name in d:
            state[name] = d[name]
    return state


def _attend(q, k, v, p, L, case):
    """Plain attention in 32 bits: q [B, n, Hq, D] at positions p [B, n] over k and v [B, T, Hkv, D], of which L [B] are keys."""
    B, n, Hq, D = q.shape
    T, Hkv = k.shape[1], k.shape[2]
    j = torch.arange(T, device=q.device)
    mask = (j < L[:, None])[:, None, :].expand(B, n, T)
    if case["ahead"] >= 0:
        mask = mask & (j <= p[:, :, None] + case["ahead"])
    if case["window"]:
        mask = mask & ((j > p[:, :, None] - case["window"]) | (j < case["sinks"]))
    mask = mask[:, None, None]
    q = q.float().reshape(B, n, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4) * D ** -0.5
    k, v = k.float().permute(0, 2, 1, 3)[:, :, None], v.float().permute(0, 2, 1, 3)[:, :, None]
    s = torch.matmul(q, k.transpose(-1, -2))
    s = torch.where(mask, s, -math.inf)
    top = s.amax(dim=-1, keepdim=True)
    s = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = s.sum(dim=-1, keepdim=True)
    o = torch.matmul(s, v) / torch.where(total > 0, total, 1.0)
    return o.permute(0, 3, 1, 2, 4).reshape(B, n, Hq, D).to(torch.bfloat16)


def _gather(s, tokens):
    """The plain K and V [B, tokens, Hkv, D] of the cache's sequences in 32 bits, zero behind their ends."""
    ps = s["k_pages"].shape[2]
    pos = torch.arange(tokens, device="cuda")
    page = s["table"].long()[:, pos // ps].clamp(min=0)
    off = (pos % ps).expand_as(page)
    there = (pos < s["lengths"][:, None])[:, :, None, None]
    if s["k_scale"] is None:
        k, v = s["k_pages"][page, :, off].float(), s["v_pages"][page, :, off].float()
    else:
        k, v = ((x.view(torch.uint8)[page, :, off].view(x.dtype).float()
                 * y.view(torch.uint8)[page, :, off].view(y.dtype).float()[..., None])
                for x, y in ((s["k_pages"], s["k_scale"]), (s["v_pages"], s["v_scale"])))
    return torch.where(there, k, 0.0), torch.where(there, v, 0.0)


def run(s):
    case = s["case"]
    if own:
        import sol_attn_b200
    rule = {"window": case.get("window") or None, "lookahead": None if case.get("ahead", 0) < 0 else case.get("ahead", 0),
            "sink_tokens": case.get("sinks", 0)}
    if case["op"] == "window":
        if own:
            return sol_attn_b200.window_attention(s["q"], s["k"], s["v"], **rule)
        B, n, T = s["q"].shape[0], s["q"].shape[1], s["k"].shape[1]
        p = torch.arange(T - n, T, device="cuda").expand(B, n)
        return _attend(s["q"], s["k"], s["v"], p, torch.full((B,), T, device="cuda"), case)
    if case["op"] == "paged":
        if own:
            return sol_attn_b200.paged_attention(s["q"], s["cache"], s["plan"], **rule)
        k, v = _gather(s, case["keys"])
        starts, L = s["starts"].long(), s["lengths"].long()
        count = starts[1:] - starts[:-1]
        i = torch.arange(s["new"], device="cuda")
        rows = (starts[:-1, None] + i).clamp(max=s["q"].shape[0] - 1)
        p = (L - count)[:, None] + i
        o = _attend(s["q"][rows], k, v, p, L, case)
        return o[i < count[:, None]]
    if case["op"] == "write":
        if own:
            sol_attn_b200.cache_write(s["cache"], s["plan"], s["k"], s["v"])
        else:
            starts, L = s["starts"].long(), s["lengths"].long()
            t = torch.arange(s["k"].shape[0], device="cuda")
            b = torch.searchsorted(starts, t, right=True) - 1
            pos = L[b] - starts[b + 1] + t
            ps = s["k_pages"].shape[2]
            page, off = s["table"].long()[b, pos // ps], pos % ps
            if case["type"] == "e4m3":
                (k, ks), (v, vs) = _quantise(s["k"]), _quantise(s["v"])
                s["k_pages"].view(torch.uint8)[page, :, off] = k.view(torch.uint8)
                s["v_pages"].view(torch.uint8)[page, :, off] = v.view(torch.uint8)
                s["k_scale"].view(torch.uint8)[page, :, off] = ks.view(torch.uint8)
                s["v_scale"].view(torch.uint8)[page, :, off] = vs.view(torch.uint8)
            else:
                s["k_pages"][page, :, off], s["v_pages"][page, :, off] = s["k"], s["v"]
        return [x for x in (s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]) if x is not None]
    if own:
        return sol_attn_b200.cache_read(s["cache"], s["plan"], case["keys"])
    k, v = _gather(s, case["keys"])
    return k.to(torch.bfloat16), v.to(torch.bfloat16)


def _two64(e):
    """2^e for whole e, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _codes64(x):
    """E4M3 rounding in 64 bits, written from the format: 3 mantissa bits, least exponent -6, ties to even."""
    x = x.double()
    top = x.abs().amax(dim=-1, keepdim=True)
    e = torch.ceil(torch.log2(torch.clamp(top, min=1e-300) / 448.0))
    e = torch.where(top > 448.0 * _two64(e), e + 1, torch.where(top <= 448.0 * _two64(e - 1), e - 1, e)).clamp(-127, 127)
    y = x * _two64(-e)
    step = _two64(torch.floor(torch.log2(torch.clamp(y.abs(), min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step, _two64(e)


def exact(case, seed):
    d = _random(case, seed)
    D, Hq, Hkv = case["dim"], case["heads"], case["kv_heads"]
    new, keys = _lengths(case)
    if case["op"] == "write":
        ps, (pool_k, pool_v) = case["page"], d["pool"]
        parts = []
        for pool, x in ((pool_k, d["k"]), (pool_v, d["v"])):
            whole = pool.clone()
            at = 0
            for b, (n, L) in enumerate(zip(new, keys)):
                pos = torch.arange(L - n, L)
                page = d["table"][b, pos // ps].long().cuda()
                whole[page, :, (pos % ps).cuda()] = x[at:at + n]
                at += n
            parts.append(_codes64(whole) if case["type"] == "e4m3" else (whole.double(), None))
        out = [parts[0][0], parts[1][0]]
        if case["type"] == "e4m3":
            out += [parts[0][1][..., 0], parts[1][1][..., 0]]
        return out
    if case["op"] == "window":
        sequences = [(d["q"][b], d["k"][b], d["v"][b]) for b in range(case["batch"])]
    else:
        pools = []
        for pool in d["pool"]:
            if case["type"] == "e4m3":
                code, scale = _codes64(pool)
                pools.append((code * scale).to(torch.bfloat16))  # exact: 4 significant bits
            else:
                pools.append(pool)
        sequences, at = [], 0
        for b, (n, L) in enumerate(zip(new, keys)):
            page = d["table"][b, : -(-int(L) // case["page"])].long().cuda()
            k, v = (x[page].transpose(1, 2).reshape(-1, Hkv, D)[:L] for x in pools)
            sequences.append((d["q"][at:at + n] if case["op"] == "paged" else None, k, v))
            at += n
    if case["op"] == "read":
        outs = [torch.zeros(case["batch"], case["keys"], Hkv, D, dtype=torch.float64, device="cuda") for _ in range(2)]
        for b, (_, k, v) in enumerate(sequences):
            outs[0][b, : len(k)], outs[1][b, : len(v)] = k.double(), v.double()
        return outs
    found = []
    for q, k, v in sequences:
        n, L = q.shape[0], k.shape[0]
        out = torch.zeros(n, Hq, D, dtype=torch.float64, device="cuda")
        j = torch.arange(L, device="cuda")
        for h in range(Hq):
            kk, vv = k[:, h // (Hq // Hkv)].double(), v[:, h // (Hq // Hkv)].double()
            for a in range(0, n, 2048):
                p = torch.arange(L - n + a, L - n + min(n, a + 2048), device="cuda")[:, None]
                hidden = torch.zeros(len(p), L, dtype=torch.bool, device="cuda")
                if case["ahead"] >= 0:
                    hidden = hidden | (j > p + case["ahead"])
                if case["window"]:
                    hidden = hidden | ((j <= p - case["window"]) & (j >= case["sinks"]))
                t = (q[a:a + 2048, h].double() @ kk.T) / math.sqrt(D)
                t = torch.softmax(t.masked_fill(hidden, -math.inf), dim=-1)
                out[a:a + 2048, h] = torch.nan_to_num(t) @ vv
        found.append(out)
    return torch.stack(found) if case["op"] == "window" else torch.cat(found)
