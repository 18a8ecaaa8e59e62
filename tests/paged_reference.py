"""Plain 64-bit forms of the windowed and paged operators, and the error their kernels may make."""

from __future__ import annotations

import math

import torch

E4M3 = torch.float8_e4m3fn
E8M0 = torch.float8_e8m0fnu


def visible(n, L, window, lookahead, sinks):
    """[n, L] truth values: what query i (position L - n + i) sees."""
    p = torch.arange(L - n, L)[:, None]
    j = torch.arange(L)[None]
    m = torch.ones((n, L), dtype=torch.bool)
    if lookahead is not None:
        m &= j <= p + lookahead
    if window is not None:
        m &= (j > p - window) | (j < sinks)
    return m


def attend(q, k, v, *, window=None, lookahead=0, sink_tokens=0, scale=None):
    """One sequence: q [n, Hq, D], k and v [L, Hkv, D] -> (out, tolerance), 64 bits, on the CPU.

    Keys that a query does not see are cut out, so that they have no influence whatever they hold.

    The kernels round twice: P to BF16 (each p off by at most 2^-8 relative, half a step of BF16,
    so o by at most 2^-8 * sum p |v| / sum p), and o to BF16 (2^-8 |o|).  S, the exponentials and
    the sums are in FP32: a score is a sum of D products, off by at most D * 2^-24 * sum |q k| scale
    (times log2 e and back), and a relative error of p of twice that (numerator and denominator)
    enters o, besides 2^-21 for the exponential and its argument's rounding per unit of score.
    """
    n, Hq, D = q.shape
    L, Hkv = k.shape[0], k.shape[1]
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros((n, Hq, D), dtype=torch.float64)
    tol = torch.zeros_like(out)
    m = visible(n, L, window, lookahead, sink_tokens)
    for h in range(Hq):
        kv = h // (Hq // Hkv)
        for i in range(n):
            idx = m[i].nonzero()[:, 0]
            if len(idx) == 0:
                continue
            kk, vv = k[idx, kv], v[idx, kv]
            s = (kk @ q[i, h]) * scale
            w = torch.softmax(s, 0)
            out[i, h] = w @ vv
            size = float((kk.abs() @ q[i, h].abs()).max()) * scale if len(idx) else 0.0
            err = 2 * (D * 2.0 ** -24 * size + 2.0 ** -21 * (1 + size))
            tol[i, h] = 2.0 ** -8 * out[i, h].abs() + (2.0 ** -8 * 1.01 + err) * (w @ vv.abs()) + 1e-30
    return out, tol


def assert_within(actual, expected, tolerance):
    actual = actual.double().cpu()
    assert torch.equal(torch.isnan(actual), torch.isnan(expected))
    fine = torch.isfinite(expected)
    assert torch.equal(actual[~fine & ~torch.isnan(expected)], expected[~fine & ~torch.isnan(expected)])
    excess = ((actual - expected).abs() - tolerance)[fine]
    assert excess.numel() == 0 or float(excess.max()) <= 0, float(excess.max())


def quantise(x):
    """E4M3 codes and E8M0 scales of rows [..., D] (finite values), from the definition."""
    x = x.double().cpu()
    top = x.abs().amax(-1)
    e = torch.full(top.shape, -127, dtype=torch.int64)
    for cand in range(127, -128, -1):  # the least e with top <= 448 * 2^e
        e = torch.where(top <= 448.0 * 2.0 ** cand, torch.full_like(e, cand), e)
    y = torch.ldexp(x, -e[..., None].double())
    codes = y.float().to(E4M3)  # (exact in FP32, one rounding)
    return codes, (e + 127).to(torch.uint8).view(E8M0)


def values(codes, scales):
    return codes.cpu().float().double() * scales.cpu().float().double()[..., None]


class Sequences:
    """A paged cache with random K/V for sequences of the given (new, keys), pages in random order."""

    def __init__(self, counts, *, heads, dim, page, kind, seed=0, extra=2, device="cuda", width=None,
                 v_gain=None):
        from sol_attn_b200 import PagedKVCache, PagedPlan
        gen = torch.Generator().manual_seed(seed)
        self.counts, self.page = counts, page
        self.k = [torch.randn((L, heads, dim), generator=gen, dtype=torch.bfloat16) * 2 for _, L in counts]
        self.v = [torch.randn((L, heads, dim), generator=gen, dtype=torch.bfloat16) for _, L in counts]
        if v_gain is not None:  # (L, heads) -> factors of V's rows
            self.v = [x * v_gain(*x.shape[:2])[..., None].to(x.dtype) for x in self.v]
        used = [-(-L // page) for _, L in counts]
        pages = sum(used) + extra
        order = torch.randperm(pages, generator=gen)
        width = max(1, max(used)) if width is None else width
        table = torch.full((len(counts), width), -1, dtype=torch.int32)
        # Unused places of the pool hold NaN: nothing may read them into a result.
        k = torch.full((pages, heads, page, dim), math.nan, dtype=torch.bfloat16)
        v = k.clone()
        if kind == "e4m3":
            k, v = (torch.full(k.shape, 0x7F, dtype=torch.uint8).view(E4M3) for _ in range(2))
            ks, vs = (torch.full(k.shape[:3], 255, dtype=torch.uint8).view(E8M0) for _ in range(2))
        at = 0
        for b, (_, L) in enumerate(counts):
            table[b, :used[b]] = order[at:at + used[b]].int()
            at += used[b]
            pos = torch.arange(L)
            pg, off = table[b, pos // page].long(), pos % page
            if kind == "e4m3":
                for pool, sc, rows in ((k, ks, self.k), (v, vs, self.v)):
                    c, s = quantise(rows[b])
                    pool.view(torch.uint8)[pg, :, off] = c.view(torch.uint8)
                    sc.view(torch.uint8)[pg, :, off] = s.view(torch.uint8)
                    rows[b] = values(c, s)
            else:
                k[pg, :, off], v[pg, :, off] = self.k[b], self.v[b]
        starts = torch.tensor([0] + [n for n, _ in counts]).cumsum(0).int()
        lengths = torch.tensor([L for _, L in counts], dtype=torch.int32)
        self.host_plan = PagedPlan(table, lengths, starts)
        scales = (ks, vs) if kind == "e4m3" else ()
        self.host = (k, v) + scales
        self.cache = PagedKVCache(*(x.to(device) for x in self.host))
        self.plan = self.host_plan.to(device)
        self.tokens = int(starts[-1])

    def queries(self, heads, dim, seed=1, rows=None):
        gen = torch.Generator().manual_seed(seed)
        return torch.randn((self.tokens if rows is None else rows, heads, dim), generator=gen, dtype=torch.bfloat16)

    def expected(self, q, **rule):
        outs = [attend(q[a:b], k, v, **rule) for (a, b), k, v in zip(self.spans(), self.k, self.v)]
        return torch.cat([o for o, _ in outs]), torch.cat([t for _, t in outs])

    def spans(self):
        s = self.host_plan.query_starts.tolist()
        return list(zip(s[:-1], s[1:]))
