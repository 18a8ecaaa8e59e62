"""Windowed and paged attention, the paged cache's writing and reading, against plain 64-bit forms."""

import math

import pytest
import torch

from helpers import to_device
from paged_reference import E4M3, E8M0, Sequences, assert_within, attend, quantise, values, visible
from sol_attn_b200 import (PagedKVCache, PagedPlan, cache_read, cache_write, dense_attention,
                           paged_attention, window_attention)
from sol_attn_b200.status import DeviceError, check_device_errors

pytestmark = pytest.mark.gpu

RULES = [dict(), dict(lookahead=None), dict(window=1), dict(window=37, sink_tokens=5),
         dict(window=100, lookahead=60, sink_tokens=70), dict(window=16, lookahead=None, sink_tokens=16),
         dict(window=5, sink_tokens=100000)]


def _plain_gpu(q, k, v, *, window=None, lookahead=0, sink_tokens=0):
    """Plain attention in 64 bits on the GPU (larger cases) with the tolerance of paged_reference.attend,
    whose score errors are bounded by the largest score of the call."""
    G, D = q.shape[2] // k.shape[2], q.shape[3]
    n, L = q.shape[1], k.shape[1]
    m = visible(n, L, window, lookahead, sink_tokens).cuda()
    out, tol = [], []
    for h in range(q.shape[2]):
        kk, vv = k[:, :, h // G].double(), v[:, :, h // G].double()
        s = torch.einsum("bqd,bkd->bqk", q[:, :, h].double(), kk) * D ** -0.5
        size = float(torch.einsum("bqd,bkd->bqk", q[:, :, h].double().abs(), kk.abs()).max()) * D ** -0.5
        w = torch.softmax(s.masked_fill(~m, -math.inf), -1).nan_to_num()
        err = 2 * (D * 2.0 ** -24 * size + 2.0 ** -21 * (1 + size))
        o = w @ vv
        out.append(o)
        tol.append(2.0 ** -8 * o.abs() + (2.0 ** -8 * 1.01 + err) * (w @ vv.abs()) + 1e-30)
    return torch.stack(out, 2).cpu(), torch.stack(tol, 2).cpu()


@pytest.mark.parametrize("rule", [dict(), dict(lookahead=None), dict(window=700, lookahead=300, sink_tokens=130)])
@pytest.mark.parametrize("B,Tq,Tk,Hq,Hkv,D", [
    (2, 3001, 3001, 8, 8, 128), (3, 2000, 4500, 12, 4, 64), (1, 1000, 20000, 16, 8, 128), (1, 5, 30000, 12, 1, 64),
    (40, 2, 3000, 8, 8, 128),
])
def test_window_attention_many_items(B, Tq, Tk, Hq, Hkv, D, rule):
    """Several items per CTA, whole and split ones, clusters and joined splits."""
    q, k, v = (x.cuda() for x in _bthd(B, Tq, Tk, Hq, Hkv, D, seed=7))
    assert_within(window_attention(q, k, v, **rule), *_plain_gpu(q, k, v, **rule))
    check_device_errors()


def _bthd(B, Tq, Tk, Hq, Hkv, D, seed=0):
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn((B, Tq, Hq, D), generator=gen, dtype=torch.bfloat16)
    k = torch.randn((B, Tk, Hkv, D), generator=gen, dtype=torch.bfloat16) * 2
    v = torch.randn((B, Tk, Hkv, D), generator=gen, dtype=torch.bfloat16)
    return q, k, v


def _check_window(q, k, v, **rule):
    out = window_attention(*(to_device(x) for x in (q, k, v)), **rule)
    assert out.shape == q.shape and out.is_contiguous()
    for b in range(q.shape[0]):
        assert_within(out[b], *attend(q[b], k[b], v[b], **rule))
    check_device_errors()


@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("B,Tq,Tk,Hq,Hkv,D", [
    (1, 1, 1, 1, 1, 64), (2, 1, 333, 8, 2, 128), (1, 3, 130, 6, 2, 64), (1, 16, 16, 3, 3, 128),
    (2, 70, 200, 2, 1, 128), (1, 300, 300, 2, 2, 64), (1, 140, 40, 3, 1, 64), (1, 5, 700, 16, 1, 128),
])
def test_window_attention(B, Tq, Tk, Hq, Hkv, D, rule):
    _check_window(*_bthd(B, Tq, Tk, Hq, Hkv, D), **rule)


@pytest.mark.parametrize("Tq", [1, 200])
def test_window_attention_strided_and_misaligned(Tq):
    """Views of a packed buffer, a start off the 16-byte boundary, an odd stride of a dimension of 1."""
    gen = torch.Generator().manual_seed(3)
    buf = torch.randn((2, 260, 3, 4, 64), generator=gen, dtype=torch.bfloat16)
    _check_window(buf[:, 260 - Tq:, 0], buf[:, :, 1, ::2], buf[:, :, 2, ::2], window=50)
    flat = torch.randn(1 + Tq * 2 * 64, generator=gen, dtype=torch.bfloat16).cuda()
    q = flat[1:].view(1, Tq, 2, 64)
    k, v = (torch.randn((1, 260, 2, 64), generator=gen, dtype=torch.bfloat16).cuda() for _ in range(2))
    assert_within(window_attention(q, k, v)[0], *attend(q[0], k[0], v[0]))
    q = torch.as_strided(flat, (1, 1, 2, 64), (7, 3, 64, 1))
    assert_within(window_attention(q, k, v)[0], *attend(q[0], k[0], v[0]))
    check_device_errors()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("Tq", [1, 4, 150])
def test_values_that_a_query_does_not_see_have_no_influence(Tq, bad):
    """Non-finite K and V outside the window, behind the queries (the chunk's own later tokens among
    them) leave every query that does not see them as it was, and reach those that do."""
    q, k, v = _bthd(1, Tq, 400, 4, 2, 128)
    for j in (0, 130, 399, 399 - Tq // 2):
        k[0, j, 0] = bad
        v[0, j, 1, 17] = bad
    rule = dict(window=120, sink_tokens=0)
    out = window_attention(q.cuda(), k.cuda(), v.cuda(), **rule)[0].cpu()
    want, tol = attend(q[0], k[0], v[0], **rule)
    # An infinite score is an infinity minus itself in any softmax: compare what the definition gives.
    assert_within(out, want, tol)
    assert torch.isfinite(want).any()
    check_device_errors()


PAGED = [
    ([(1, 1)], 1, 1, 64, 16), ([(1, 1000)], 16, 2, 128, 64), ([(1, 77), (1, 5), (1, 300), (1, 64)], 8, 8, 64, 32),
    ([(0, 0), (3, 3), (0, 40), (1, 129), (2, 700)], 6, 2, 128, 16), ([(17, 30), (140, 600), (0, 9), (65, 65)], 4, 4, 64, 128),
    ([(200, 231), (1, 500), (33, 400)], 4, 2, 128, 64), ([(90, 90)], 5, 1, 128, 16),
]


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("rule", RULES)
@pytest.mark.parametrize("counts,Hq,Hkv,D,page", PAGED)
def test_paged_attention(counts, Hq, Hkv, D, page, rule, kind):
    s = Sequences(counts, heads=Hkv, dim=D, page=page, kind=kind)
    q = s.queries(Hq, D)
    out = paged_attention(q.cuda(), s.cache, s.plan, **rule)
    assert_within(out, *s.expected(q, **rule))
    check_device_errors()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("new", [1, 300])
def test_paged_long_split(kind, new):
    """Lengths that are split over many CTAs, next to short ones; twice, to the same bits."""
    s = Sequences([(new, 9000), (1, 40), (1, 4097)], heads=1, dim=128, page=64, kind=kind)
    q = s.queries(2, 128)
    out = paged_attention(q.cuda(), s.cache, s.plan, sink_tokens=3)
    rows = torch.tensor([0, new - 1, new // 2, new, new + 1]).unique()
    want, tol = s.expected(q, sink_tokens=3) if new == 1 else (None, None)
    if new == 1:
        assert_within(out, want, tol)
    else:
        for i in rows.tolist():
            b = 0 if i < new else i - new + 1
            L = s.counts[b][1] - (new - 1 - i if b == 0 else 0)
            assert_within(out[i:i + 1], *attend(q[i:i + 1], s.k[b][:L], s.v[b][:L]))
    assert torch.equal(out, paged_attention(q.cuda(), s.cache, s.plan, sink_tokens=3))
    check_device_errors()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("new", [1, 130])
def test_rows_behind_the_last_sequence(kind, new):
    s = Sequences([(new, 200), (1, 3)], heads=2, dim=64, page=16, kind=kind)
    q = s.queries(4, 64, rows=s.tokens + 37)
    want, tol = s.expected(q[:s.tokens])
    out = paged_attention(q.cuda(), s.cache, s.plan)
    assert_within(out[:s.tokens], want, tol)
    assert not out[s.tokens:].any()
    mine = torch.full_like(out, 7.0)
    assert paged_attention(q.cuda(), s.cache, s.plan, out=mine) is mine
    assert torch.equal(mine[:s.tokens], out[:s.tokens])
    assert bool((mine[s.tokens:] == 7.0).all())
    check_device_errors()


@pytest.mark.parametrize("new", [1, 2, 200])
def test_e4m3_nan_codes_and_scales(new):
    """A NaN code or scale reaches the queries that see it, and no others."""
    s = Sequences([(new, 300)], heads=1, dim=64, page=16, kind="e4m3")
    q = s.queries(2, 64)
    table = s.host_plan.page_table[0]
    rule = dict(window=150)

    def place(j):
        return int(table[j // 16]), j % 16

    for j, what in ((20, "k"), (299, "v"), (299 - new // 2, "vs"), (160, "v")):
        pg, off = place(j)
        if what == "vs":
            s.cache.v_scale.view(torch.uint8)[pg, 0, off] = 255
            s.v[0][j] = math.nan
        else:
            pool = s.cache.k if what == "k" else s.cache.v
            pool.view(torch.uint8)[pg, 0, off, 33] = 0xFF
            (s.k if what == "k" else s.v)[0][j, 0, 33] = math.nan
    out = paged_attention(q.cuda(), s.cache, s.plan, **rule)
    want, tol = s.expected(q, **rule)
    assert_within(out, want, tol)
    check_device_errors()


@pytest.mark.parametrize("new", [1, 3, 150])
@pytest.mark.parametrize("D,page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("spread", [6, 40])
def test_e4m3_scales_far_apart(new, D, page, spread):
    """V rows (and so their scales) that differ by powers of two, rows of zeros among them, large ones
    that only a few queries see, and one so large that it dwarfs the rest."""
    gen = torch.Generator().manual_seed(11)

    def gain(L, heads):
        g = torch.exp2(torch.randint(-spread, 4, (L, heads), generator=gen).float())
        g[::7] = 0
        g[L // 2] = 2.0 ** 30
        return g

    s = Sequences([(new, 500), (1, 33)], heads=2, dim=D, page=page, kind="e4m3", v_gain=gain)
    q = s.queries(4, D)
    for rule in (dict(), dict(window=100, sink_tokens=5)):
        assert_within(paged_attention(q.cuda(), s.cache, s.plan, **rule), *s.expected(q, **rule))
    check_device_errors()


@pytest.mark.parametrize("new", [1, 150])
@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_large_scores(kind, new):
    """Scores of hundreds, at which the running maximum moves in most tiles."""
    s = Sequences([(new, 700)], heads=1, dim=64, page=16, kind=kind)
    q = s.queries(2, 64) * 40
    assert_within(paged_attention(q.cuda(), s.cache, s.plan), *s.expected(q))
    check_device_errors()


def test_pages_that_no_key_needs_are_not_read():
    """Window pages given back (-1, or far outside) are never addressed; a needed one is reported."""
    s = Sequences([(1, 640)], heads=1, dim=64, page=16, kind="bf16")
    q = s.queries(1, 64)
    want, tol = s.expected(q, window=64, sink_tokens=10)
    s.plan.page_table[0, 1:36] = 1 << 30
    out = paged_attention(q.cuda(), s.cache, s.plan, window=64, sink_tokens=10)
    assert_within(out, want, tol)
    check_device_errors()
    s.plan.page_table[0, 39] = s.cache.pages
    paged_attention(q.cuda(), s.cache, s.plan, window=64, sink_tokens=10)
    with pytest.raises(DeviceError, match="status 2"):
        check_device_errors()
    check_device_errors()


@pytest.mark.parametrize("new", [1, 200])
def test_bad_plans_are_reported(new):
    s = Sequences([(new, 300), (1, 20)], heads=2, dim=64, page=32, kind="bf16")
    q = s.queries(2, 64).cuda()
    k = torch.zeros((q.shape[0], 2, 64), dtype=torch.bfloat16, device="cuda")
    for field, index, value in (("key_lengths", 0, 100000), ("key_lengths", 1, -5), ("query_starts", 1, -3),
                                ("query_starts", 1, 100000), ("query_starts", 2, 1 << 30)):
        t = getattr(s.plan, field)
        old = int(t[index])
        t[index] = value
        for call in (lambda: paged_attention(q, s.cache, s.plan), lambda: cache_write(s.cache, s.plan, k, k)):
            call()
            with pytest.raises(DeviceError, match="status 2"):
                check_device_errors()
        t[index] = old
    s.plan.key_lengths[0] = 1 << 20
    cache_read(s.cache, s.plan, 64)
    with pytest.raises(DeviceError, match="status 2"):
        check_device_errors()
    check_device_errors()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("D,page,heads", [(64, 16, 3), (128, 64, 8), (128, 128, 1)])
def test_cache_write_and_read(kind, D, page, heads):
    """Codes and scales bit for bit, nothing else touched; reading gives the values back."""
    counts = [(5, 9), (0, 33), (70, 200), (1, 1)]
    s = Sequences(counts, heads=heads, dim=D, page=page, kind=kind)
    gen = torch.Generator().manual_seed(9)
    rows = s.tokens + 3  # three behind the last sequence
    buf = torch.randn((rows, 2, 2 * heads, D), generator=gen, dtype=torch.bfloat16)
    buf *= torch.exp2(torch.randint(-140, 100, (rows, 2, 2 * heads, 1), generator=gen).float())
    buf[1, :, :, :] = 0
    buf[2, 0, 0, 3] = 448.0
    k, v = buf[:, 0, ::2], buf[:, 1, ::2]
    cache_write(s.cache, s.plan, to_device(buf)[:, 0, ::2], to_device(buf)[:, 1, ::2])
    host = [x.clone() for x in s.host]
    for (a, b), (n, L), row in zip(s.spans(), counts, s.host_plan.page_table):
        pos = torch.arange(L - n, L)
        pg, off = row[pos // page].long(), pos % page
        for z, x in enumerate((k, v)):
            if kind == "e4m3":
                c, e = quantise(x[a:b])
                host[z].view(torch.uint8)[pg, :, off] = c.view(torch.uint8)
                host[2 + z].view(torch.uint8)[pg, :, off] = e.view(torch.uint8)
            else:
                host[z][pg, :, off] = x[a:b]
    got = [s.cache.k, s.cache.v] + ([s.cache.k_scale, s.cache.v_scale] if kind == "e4m3" else [])
    for x, y in zip(got, host):
        assert torch.equal(x.cpu().view(torch.uint8), y.view(torch.uint8))
    for tokens in (1, 64, 201, 300):
        rk, rv = cache_read(s.cache, s.plan, tokens)
        assert rk.shape == rv.shape == (len(counts), tokens, heads, D)
        for b, (n, L) in enumerate(counts):
            pos = torch.arange(min(L, tokens))
            pg, off = s.host_plan.page_table[b][pos // page].long(), pos % page
            for z, r in enumerate((rk, rv)):
                x = host[z][pg, :, off] if kind == "bf16" else values(
                    host[z].view(torch.uint8)[pg, :, off].view(E4M3),
                    host[2 + z].view(torch.uint8)[pg, :, off].view(E8M0)).to(torch.bfloat16)
                assert torch.equal(r[b, :len(pos)].cpu(), x)
                assert not r[b, len(pos):].any()
    check_device_errors()


def test_cache_write_non_finite():
    """The scale comes from the finite values; infinities saturate, NaN stays NaN."""
    cache = PagedKVCache.create(1, 1, 64, page_size=16, dtype=E4M3)
    plan = PagedPlan.create(torch.tensor([[0]], dtype=torch.int32), torch.tensor([2], dtype=torch.int32),
                            torch.tensor([0, 2], dtype=torch.int32), page_size=16).to("cuda")
    x = torch.ones((2, 1, 64), dtype=torch.bfloat16)
    x[0, 0, :3] = torch.tensor([math.inf, -math.inf, math.nan])
    x[1] = math.inf
    cache_write(cache, plan, x.cuda(), x.cuda())
    codes, scale = cache.k[0, 0].float().cpu(), cache.k_scale[0, 0].float().cpu()
    assert float(scale[0]) == 2.0 ** -8  # 1 <= 448 * 2^-8 and not 448 * 2^-9
    assert codes[0, 0] == 448 and codes[0, 1] == -448 and torch.isnan(codes[0, 2])
    assert bool((codes[0, 3:] == 256).all())
    assert bool((codes[1] == 448).all()) and float(scale[1]) == 2.0 ** -127
    check_device_errors()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
def test_a_stream_of_chunks_and_tokens(kind):
    """Chunks written, attended to and read back, then single tokens: the paged path gives what the
    same attention over the tensors read back gives, and the dense operator agrees."""
    D, H, page = 128, 4, 32
    dtype = torch.bfloat16 if kind == "bf16" else E4M3
    gen = torch.Generator().manual_seed(5)
    cache = PagedKVCache.create(40, H, D, page_size=page, dtype=dtype)
    table = torch.randperm(40, generator=gen).int().reshape(2, 20)
    have = [0, 0]
    for new in ([130, 64], [1, 1], [0, 200], [1, 1], [257, 3]):
        starts = torch.tensor([0, new[0], sum(new)], dtype=torch.int32)
        have = [a + b for a, b in zip(have, new)]
        plan = PagedPlan.create(table, torch.tensor(have, dtype=torch.int32), starts, page_size=page,
                                pages=cache.pages).to("cuda")
        q, k, v = (torch.randn((sum(new), H, D), generator=gen, dtype=torch.bfloat16).cuda() for _ in range(3))
        cache_write(cache, plan, k, v)
        for rule in (dict(), dict(window=100, sink_tokens=20), dict(lookahead=None)):
            out = paged_attention(q, cache, plan, **rule)
            rk, rv = cache_read(cache, plan, max(have))
            for b in range(2):
                a, e = starts[b:b + 2].tolist()
                if a == e:
                    continue
                kb, vb = rk[b:b + 1, :have[b]], rv[b:b + 1, :have[b]]
                flat = window_attention(q[None, a:e], kb, vb, **rule)[0]
                # Both round P and the result (see attend): twice its tolerance, with |v| in the mean.
                _, tol = attend(q[a:e].cpu(), kb[0].cpu(), vb[0].cpu(), **rule)
                assert_within(out[a:e], flat.double().cpu(), 2 * tol)
                if rule.get("lookahead", 0) is None:
                    dense = dense_attention(q[None, a:e].contiguous(), kb.contiguous(), vb.contiguous())[0]
                    assert_within(dense, flat.double().cpu(), 2 * tol)
    check_device_errors()


@pytest.mark.parametrize("new", [1, 150])
def test_streams_and_graphs(new):
    """A call on a side stream, and a step captured once and replayed with other contents: lengths,
    pages and queries changed in place; two graphs with splits live at the same time."""
    s = Sequences([(new, 4000), (1, 1500)], heads=2, dim=64, page=16, kind="e4m3", width=300)
    q = s.queries(4, 64)
    dq = q.cuda()
    first = paged_attention(dq, s.cache, s.plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = paged_attention(dq, s.cache, s.plan)
    side.synchronize()
    assert torch.equal(first, other)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        k = torch.ones((dq.shape[0], 2, 64), dtype=torch.bfloat16, device="cuda")
        with torch.cuda.graph(graph):
            out = paged_attention(dq, s.cache, s.plan)
            rk, _ = cache_read(s.cache, s.plan, 8)
            win = window_attention(dq[None, :1], rk[:1], rk[:1])
        graphs.append((graph, out, win, k))
    for graph, out, win, _ in graphs:
        graph.replay()
        assert torch.equal(first, out)
    s.plan.key_lengths.sub_(100)
    dq.mul_(0.5)
    again = paged_attention(dq, s.cache, s.plan)
    for graph, out, win, _ in graphs:
        graph.replay()
        assert torch.equal(again, out)
    assert not torch.equal(again, first)
    check_device_errors()
    del graphs


def test_copies_and_overlaps():
    """A deep copy of cache and plan is a cache and a plan of its own; out may not lie over Q."""
    import copy
    s = Sequences([(2, 40), (1, 9)], heads=2, dim=64, page=16, kind="e4m3")
    q = s.queries(2, 64).cuda()
    first = paged_attention(q, s.cache, s.plan)
    cache, plan = copy.deepcopy(s.cache), copy.deepcopy(s.plan)
    s.cache.k.view(torch.uint8).zero_()
    s.plan.key_lengths.zero_()
    assert torch.equal(paged_attention(q, cache, plan), first)
    assert not paged_attention(q, s.cache, s.plan).any()  # no keys
    both = torch.zeros((2 * q.shape[0],) + q.shape[1:], dtype=torch.bfloat16, device="cuda")
    both[:q.shape[0]] = q
    with pytest.raises(ValueError, match="share"):
        paged_attention(both[:3], cache, plan, out=both[1:4])
    assert torch.equal(paged_attention(both[:3], cache, plan, out=both[3:]), first)
    check_device_errors()


@pytest.mark.parametrize("new", [1, 160])
def test_offsets_past_32_bits(new):
    """Pages whose byte offsets pass 2^32."""
    pages, H, ps, D = 40000, 8, 64, 128
    k, v = (torch.empty((pages, H, ps, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cache = PagedKVCache(k, v)
    gen = torch.Generator().manual_seed(2)
    L = 200
    table = torch.tensor([[39999, 39001, 3, 38888]], dtype=torch.int32)
    plan = PagedPlan.create(table, torch.tensor([L], dtype=torch.int32), torch.tensor([0, L], dtype=torch.int32),
                            pages=pages).to("cuda")
    x, y = (torch.randn((L, H, D), generator=gen, dtype=torch.bfloat16) for _ in range(2))
    cache_write(cache, plan, x.cuda(), y.cuda())
    q = torch.randn((new, H, D), generator=gen, dtype=torch.bfloat16)
    step = PagedPlan(plan.page_table, plan.key_lengths, torch.tensor([0, new], dtype=torch.int32, device="cuda"))
    assert_within(paged_attention(q.cuda(), cache, step), *attend(q, x, y))
    rk, rv = cache_read(cache, plan, L)
    assert torch.equal(rk[0].cpu(), x) and torch.equal(rv[0].cpu(), y)
    check_device_errors()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("behind", [0, 400])
@pytest.mark.parametrize("hint", [0, 1, 3, 200, 1000])
@pytest.mark.parametrize("counts", [[(1, 300)], [(3, 200), (1, 50)], [(200, 400), (1, 30), (0, 9)]])
def test_paged_attention_hints_and_padding(kind, behind, hint, counts):
    """most_new chooses kernels only, right or wrong, with many rows behind the last sequence too."""
    s = Sequences(counts, heads=2, dim=64, page=16, kind=kind)
    q = s.queries(4, 64, rows=s.tokens + behind)
    plan = PagedPlan(s.plan.page_table, s.plan.key_lengths, s.plan.query_starts, hint)
    expected, tolerance = s.expected(q)
    out = paged_attention(to_device(q), s.cache, plan)
    assert_within(out[:s.tokens], expected, tolerance)
    assert not out[s.tokens:].any()
    kept = torch.full_like(out, 7.0)
    paged_attention(to_device(q), s.cache, plan, out=kept)
    assert torch.equal(kept[:s.tokens], out[:s.tokens]) and bool((kept[s.tokens:] == 7.0).all())
    check_device_errors()


@pytest.mark.parametrize("kind", ["bf16", "e4m3"])
@pytest.mark.parametrize("heads", [95, 128, 300])
def test_many_query_heads_of_one_kv_head(kind, heads):
    """One new token is many rows where the heads share K and V."""
    s = Sequences([(1, 300), (2, 70), (0, 5), (1, 1)], heads=1, dim=64, page=16, kind=kind)
    q = s.queries(heads, 64)
    for rule in (dict(), dict(window=33, sink_tokens=3)):
        assert_within(paged_attention(to_device(q), s.cache, s.plan, **rule), *s.expected(q, **rule))
    check_device_errors()
    if kind == "bf16":
        _check_window(*_bthd(2, 1, 300, heads, 1, 64), window=100)
