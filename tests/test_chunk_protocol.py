"""Randomised interleaving check of the many-rows attention kernel's mbarrier protocol (csrc/chunk.cu),
on the CPU.

A CTA works through items (256 rows: two stages of 128); an item has a list of key tiles, of which a
stage needs some.  The roles are generators: the item warp (descriptions into a ring of two, Q), the
loader (K and V rings, or the ring of E4M3 codes), the V checker or the E4M3 converters, the MMA warp,
and four softmax warps per stage, whose epilogue ends an item; a second round of items (the careful
one) starts when every item of the first is finished.  Each yields ("wait", barrier, n), a wait for
completion n of a barrier, or ("do", action).  MMAs complete in the order of issue, copies in any
order.  A barrier keeps its number of completed phases c; a wait for completion n by parity is right
only while c is n or n + 1, which every poll asserts (else the hardware would pass a phase early, or
wait for good).  Asserted besides: an S reads the K tile and the Q of its own item and never goes
over a P whose P V is not done or an S that was not read; a P V reads the V and P of its own tile;
slots are filled again only after their readers; O is rescaled, read and zeroed only while no P V
into it is under way.
"""
import random

import pytest


class Bar:
    def __init__(self, name, count):
        self.name, self.count, self.pending, self.c = name, count, count, 0

    def arrive(self):
        self.pending -= 1
        assert self.pending >= 0, self.name
        if self.pending == 0:
            self.c += 1
            self.pending = self.count


def run(items, again, ahead, slots, qbufs, codes, seed):
    """items: per item a list of (stage 0 needs, stage 1 needs) for its tiles; again: those done twice."""
    rng = random.Random(seed)
    nbuf = 3 if ahead else 2
    code_slots = 4 if slots == 3 else 2
    order = items + [items[k] for k in again]
    B = {}

    def bar(name, count=1):
        B[name] = Bar(name, count)

    for j in range(2):
        bar(f"IF{j}")
        bar(f"IE{j}", 11)  # MMA, loader, V checker or converters, 8 softmax warps
        bar(f"QF{j}")
        bar(f"QR{j}")
        bar(f"QE{j}")
        bar(f"OF{j}", 4)
    for j in range(4):
        bar(f"SF{j}")
        bar(f"PF{j}", 4)
        bar(f"PV{j}")
        bar(f"CF{j}")
        bar(f"CE{j}")
    for j in range(slots):
        for n in ("KF", "KE", "VF", "VO", "VE"):
            bar(f"{n}{j}")

    def turn(st, n):
        return 2 * st + (n & 1 if ahead else 0)

    def phase(n):
        return n >> 1 if ahead else n

    k_in, v_in, code_in = [None] * slots, [None] * slots, [None] * code_slots
    q_in = [None] * qbufs
    buf = [("free",)] * nbuf         # S buffer: ("S" | "P", item, tile, stage, warps that read or wrote)
    pv_busy = [0, 0]                 # P V under way, per stage
    o_item = [None, None]
    done_pv = [[], []]
    copies, mma = [], []             # copies under way; MMA queue, in order
    finished = set()

    def item_warp():
        for k, it in enumerate(order):
            if k == len(items):      # the careful round: every item so far is finished
                for j in range(max(0, k - 2), k):
                    yield ("wait", f"IE{j & 1}", j >> 1)
                assert len(finished) == 2 * k
            if k >= 2:
                yield ("wait", f"IE{k & 1}", (k >> 1) - 1)
            yield ("do", B[f"IF{k & 1}"].arrive)
            qb = k % qbufs
            if k >= qbufs:
                yield ("wait", f"QE{qb}", k // qbufs - 1)

            def load(qb=qb, k=k):
                assert q_in[qb] is None
                q_in[qb] = k
                B[f"QR{qb}" if codes else f"QF{qb}"].arrive()

            yield ("do", load)

    def take(k):
        yield ("wait", f"IF{k & 1}", k >> 1)

    def let_go(k):
        B[f"IE{k & 1}"].arrive()

    def loader():
        g = 0
        for k, it in enumerate(order):
            yield from take(k)
            yield ("do", lambda k=k: let_go(k))
            for i in range(len(it)):
                for z in range(2):
                    if codes:
                        ci = 2 * g + z
                        sl = ci % code_slots
                        if ci >= code_slots:
                            yield ("wait", f"CE{sl}", ci // code_slots - 1)

                        def land(sl=sl, what=(k, i, z)):
                            assert code_in[sl] is None
                            code_in[sl] = what
                            B[f"CF{sl}"].arrive()
                    else:
                        sl = g % slots
                        if g >= slots:
                            yield ("wait", f"{'KV'[z]}E{sl}", g // slots - 1)

                        def land(sl=sl, z=z, what=(k, i)):
                            ring = v_in if z else k_in
                            assert ring[sl] is None
                            ring[sl] = what
                            B[f"{'KV'[z]}F{sl}"].arrive()

                    yield ("do", lambda land=land: copies.append(land))
                g += 1

    def v_checker():
        g = 0
        for k, it in enumerate(order):
            yield from take(k)
            yield ("do", lambda k=k: let_go(k))
            for i in range(len(it)):
                yield ("wait", f"VF{g % slots}", g // slots)
                yield ("do", B[f"VO{g % slots}"].arrive)
                g += 1

    def converter():
        g = 0
        for k, it in enumerate(order):
            yield from take(k)
            yield ("do", lambda k=k: let_go(k))

            def order_q(k=k):
                yield ("wait", f"QR{k % qbufs}", k // qbufs)
                yield ("do", B[f"QF{k % qbufs}"].arrive)

            if not it:
                yield from order_q()
            for i in range(len(it)):
                for z in range(2):
                    ci, sl = 2 * g + z, g % slots
                    cs = ci % code_slots
                    yield ("wait", f"CF{cs}", ci // code_slots)
                    if g >= slots:
                        yield ("wait", f"{'KV'[z]}E{sl}", g // slots - 1)

                    def put(cs=cs, sl=sl, z=z, what=(k, i)):
                        assert code_in[cs] == (*what, z)
                        ring = v_in if z else k_in
                        assert ring[sl] is None
                        ring[sl] = what
                        code_in[cs] = None
                        B[f"CE{cs}"].arrive()
                        B[("VO" if z else "KF") + str(sl)].arrive()

                    yield ("do", put)
                    if z == 0 and i == 0:
                        yield from order_q()
                g += 1

    def mma_warp():
        g, nq, np, nf = 0, [0, 0], [0, 0], [0, 0]
        for k, it in enumerate(order):
            yield from take(k)
            yield ("do", lambda k=k: let_go(k))
            qb, count = k % qbufs, len(it)
            yield ("wait", f"QF{qb}", k // qbufs)

            def issue_s(s, i):
                b, full = (2 * i + s) % nbuf, f"SF{turn(s, nq[s])}"
                nq[s] += 1

                def go(b=b, sl=(g + i) % slots):
                    assert k_in[sl] == (k, i) and q_in[qb] == k
                    assert buf[b][0] in ("free", "used"), buf[b]
                    buf[b] = ("S", k, i, s, 0)
                    B[full].arrive()

                return ("do", lambda: mma.append(go))

            def commit(name, clear=None):
                def go():
                    if clear:
                        clear()
                    B[name].arrive()
                return ("do", lambda: mma.append(go))

            def free_k(i):
                sl = (g + i) % slots
                return commit(f"KE{sl}", lambda: k_in.__setitem__(sl, None))

            release_q = commit(f"QE{qb}", lambda qb=qb: q_in.__setitem__(qb, None))
            if count:
                yield ("wait", f"KF{g % slots}", g // slots)
                for s in range(2):
                    if it[0][s]:
                        yield issue_s(s, 0)
                yield free_k(0)
                if ahead and count > 1:
                    yield ("wait", f"KF{(g + 1) % slots}", (g + 1) // slots)
                    if it[1][0]:
                        yield issue_s(0, 1)
            if count <= 1:
                yield release_q
            started = [False, False]
            for i in range(count):
                gi = g + i
                sl = gi % slots
                more = i + 1 < count
                yield ("wait", f"VO{sl}", gi // slots)
                if not ahead and more:
                    yield ("wait", f"KF{(gi + 1) % slots}", (gi + 1) // slots)
                for s in range(2):
                    if it[i][s]:
                        if not started[s]:
                            started[s] = True
                            yield ("wait", f"OF{s}", nf[s])
                            nf[s] += 1
                        yield ("wait", f"PF{turn(s, np[s])}", phase(np[s]))
                        b, name = (2 * i + s) % nbuf, f"PV{turn(s, np[s])}"
                        np[s] += 1

                        def issue(b=b, s=s, i=i, sl=sl, name=name, k=k):
                            assert buf[b] == ("P", k, i, s, 4), (buf[b], k, i, s)
                            pv_busy[s] += 1

                            def go():
                                assert v_in[sl] == (k, i) and buf[b] == ("P", k, i, s, 4)
                                buf[b] = ("used",)
                                pv_busy[s] -= 1
                                o_item[s] = k
                                done_pv[s].append((k, i))
                                B[name].arrive()

                            mma.append(go)

                        yield ("do", issue)
                    if not ahead:
                        if more and it[i + 1][s]:
                            yield issue_s(s, i + 1)
                    elif s == 0:
                        if more and it[i + 1][1]:
                            yield issue_s(1, i + 1)
                    elif i + 2 < count:
                        yield ("wait", f"KF{(gi + 2) % slots}", (gi + 2) // slots)
                        if it[i + 2][0]:
                            yield issue_s(0, i + 2)
                yield commit(f"VE{sl}", lambda sl=sl: v_in.__setitem__(sl, None))
                if more:
                    yield free_k(i + 1)
                if i + 2 == count:
                    yield release_q
            g += count

    def softmax(st, w):
        ns = 0
        yield ("do", B[f"OF{st}"].arrive)
        for k, it in enumerate(order):
            yield from take(k)
            has = False
            for i in range(len(it)):
                if not it[i][st]:
                    continue
                first, has = not has, True
                mine = turn(st, ns)
                yield ("wait", f"SF{mine}", phase(ns))
                ns += 1
                b = (2 * i + st) % nbuf

                def read(b=b, k=k, i=i):
                    assert buf[b][:4] in (("S", k, i, st), ("P", k, i, st)), (buf[b], k, i, st)
                yield ("do", read)
                if rng.random() < 0.3 and not first:  # O is rescaled
                    yield ("wait", f"PV{turn(st, ns - 2)}", phase(ns - 2))

                    def rescale(k=k):
                        assert pv_busy[st] == 0 and o_item[st] == k
                    yield ("do", rescale)

                def write(b=b, k=k, i=i, mine=mine):
                    n = buf[b][4] + 1
                    buf[b] = ("P" if n == 4 else "S", k, i, st, n)
                    B[f"PF{mine}"].arrive()
                yield ("do", write)
            if has:
                yield ("wait", f"PV{turn(st, ns - 1)}", phase(ns - 1))

                def epilogue(k=k):
                    assert pv_busy[st] == 0 and o_item[st] == k
                    want = [(k, i) for i in range(len(order[k])) if order[k][i][st]]
                    assert [x for x in done_pv[st] if x[0] == k] == want
                    B[f"OF{st}"].arrive()
                yield ("do", epilogue)

            def end(k=k):
                finished.add((k, st)) if w == 0 else None
                let_go(k)
            yield ("do", end)

    roles = [item_warp(), loader(), converter() if codes else v_checker(), mma_warp()]
    roles += [softmax(st, w) for st in range(2) for w in range(4)]
    state = [next(r, None) for r in roles]
    weights = [rng.choice((1, 1, 4, 20)) for _ in roles]
    while any(s is not None for s in state) or copies or mma:
        ready = []
        for j, s in enumerate(state):
            if s is None:
                continue
            if s[0] == "do":
                ready.append(j)
            else:
                b, n = B[s[1]], s[2]
                assert b.c in (n, n + 1), (s, b.c)
                if b.c == n + 1:
                    ready.append(j)
        choices = ready + (["copy"] if copies else []) + (["mma"] if mma else [])
        assert choices, [s for s in state if s]
        pick = rng.choices(choices, [weights[c] if isinstance(c, int) else 3 for c in choices])[0]
        if pick == "copy":
            copies.pop(rng.randrange(len(copies)))()
        elif pick == "mma":
            mma.pop(0)()
        else:
            if state[pick][0] == "do":
                state[pick][1]()
            state[pick] = next(roles[pick], None)
    assert all(len([x for x in done_pv[s] if x[0] == k]) == sum(t[s] for t in it)
               for k, it in enumerate(order) for s in range(2))


def make_items(rng):
    items = []
    for _ in range(rng.randrange(1, 6)):
        count = rng.choice((0, 1, 1, 2, 3, 5, 9))
        kind = rng.randrange(4)
        it = []
        for i in range(count):
            if kind == 0:
                it.append((True, True))
            elif kind == 1:  # an item of 128 rows or fewer
                it.append((True, False))
            else:            # window edges: a stage begins later and ends later
                it.append((i < count - rng.randrange(2) or count == 1, i >= rng.randrange(2) * (count > 1)))
        items.append([t if any(t) else (True, True) for t in it])
    return items


@pytest.mark.parametrize("ahead, slots, qbufs, codes",
                         [(True, 3, 2, False), (False, 2, 1, False), (False, 2, 1, True), (False, 3, 2, True)])
def test_protocol(ahead, slots, qbufs, codes):
    for seed in range(60):
        rng = random.Random(seed)
        items = make_items(rng)
        again = [k for k in range(len(items)) if rng.random() < 0.3]
        run(items, again, ahead, slots, qbufs, codes, seed)
