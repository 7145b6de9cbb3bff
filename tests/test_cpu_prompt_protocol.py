"""The barrier protocol of the packed prompt attention kernel (csrc/prompt_attention.cuh), searched on the
CPU: every order in which one thread block's warps, copies and products can come about, for short
lists of items.

A warp's work is a list of steps (its control flow depends on the items alone).  A wait is the hardware's: by
the parity of a phase, so it passes whenever the last completed phase has the wanted parity, the
wanted phase or not.  In every reachable state
  * a wait that passes has met its own phase,
  * what a product or a softmax warp reads is what it is meant to read (K and V parts, S, P, O in place),
  * somebody can go on, until all are done.
The four warps of a half of a row tile stand for one another."""
import pytest


class Model:
    def __init__(self):
        self.warps, self.counts, self.cells = {}, {}, {}

    def bar(self, name, count):
        self.counts[name] = count

    def steps(self, name):
        return self.warps.setdefault(name, [])


class Wrong(Exception):
    pass


def search(m, limit=3_000_000):
    """Visits every reachable state; raises Wrong."""
    names, bars = list(m.warps), {b: i for i, b in enumerate(m.counts)}
    counts = list(m.counts.values())
    cells = {}
    for steps in m.warps.values():
        for s in steps:
            for c in ([x for x, _ in s[1]] + [x for x, _ in s[2]] if s[0] in ("do", "mma") else [s[2]] if s[0] == "load" else []):
                cells.setdefault(c, len(cells))
    progs = [m.warps[n] for n in names]

    def arrive(bar, b):
        i = bars[b]
        done, n = bar[i]
        n += 1
        bar[i] = (done + 1, 0) if n == counts[i] else (done, n)

    def touch(cell, reads, writes, who):
        for c, tag in reads:
            if cell[cells[c]] != tag:
                raise Wrong(f"{who} finds {cell[cells[c]]} in {c}, not {tag}")
        for c, tag in writes:
            cell[cells[c]] = tag

    # (places of the warps, barriers, copies in flight, products in each warp's queue, cells)
    start = (tuple([0] * len(names)), tuple([(0, 0)] * len(counts)), frozenset(), tuple([()] * len(names)), tuple([None] * len(cells)))
    seen, todo = {start}, [start]
    while todo:
        pcs, bar0, flying, queues, cell0 = todo.pop()
        after = []
        for w, prog in enumerate(progs):
            pc = pcs[w]
            if pc == len(prog):
                continue
            if prog[pc][0] == "wait":       # with what follows it up to the next wait (to wait later is another order)
                _, b, phase = prog[pc]
                done = bar0[bars[b]][0]
                if done % 2 == phase % 2:
                    if done == phase + 2:
                        raise Wrong(f"{names[w]} is overtaken: phase {phase} of {b} has gone by")
                    continue
                if done != phase + 1:
                    raise Wrong(f"{names[w]} takes another phase of {b} for phase {phase} ({done} are complete)")
                pc += 1
            bar, cell, fly, queue = list(bar0), list(cell0), set(flying), [list(q) for q in queues]
            while pc < len(prog) and prog[pc][0] != "wait":
                s = prog[pc]
                if s[0] == "arrive":
                    arrive(bar, s[1])
                elif s[0] == "load":
                    cell[cells[s[2]]] = None
                    fly.add(s[1:])
                elif s[0] == "mma":
                    queue[w].append(tuple(map(tuple, s[1:])))
                else:
                    touch(cell, s[1], s[2], names[w])
                pc += 1
            after.append((pcs[:w] + (pc,) + pcs[w + 1:], tuple(bar), frozenset(fly), tuple(map(tuple, queue)), tuple(cell)))
        for f in flying:
            bar, cell = list(bar0), list(cell0)
            cell[cells[f[1]]] = f[2]
            arrive(bar, f[0])
            after.append((pcs, tuple(bar), flying - {f}, queues, tuple(cell)))
        for w, q in enumerate(queues):
            if q:
                bar, cell = list(bar0), list(cell0)
                touch(cell, q[0][0], q[0][1], names[w] + "'s product")
                for b in q[0][2]:
                    arrive(bar, b)
                after.append((pcs, tuple(bar), flying, queues[:w] + (q[1:],) + queues[w + 1:], tuple(cell)))
        if not after and any(pc < len(p) for pc, p in zip(pcs, progs)):
            raise Wrong("nobody can go on: " + ", ".join(f"{n} at {p[pc]}" for n, pc, p in zip(names, pcs, progs) if pc < len(p)))
        for s in after:
            if s not in seen:
                seen.add(s)
                todo.append(s)
        assert len(seen) < limit, "too many states: a shorter list of items"
    return len(seen)


def kernel(items, slots, first_half_waits_for_both=True, one_ring=False):
    """The kernel's steps for items (key tiles of A, key tiles of B) with `slots` K and `slots` V parts in flight.  one_ring: K
    and V through one ring of 2 * slots in the order of use; first_half_waits_for_both false: the first half of P V
    does not wait for the second half's scaling of O.  (Forms that go wrong, which the search has to find.)"""
    m = Model()
    loader, scores, values, looker = (m.steps(n) for n in ("loader", "scores", "values", "looker"))
    tiles = [w for w in range(2) if any(it[w] for it in items)]
    soft = {(w, h): m.steps(f"softmax {w} {h}") for w in tiles for h in range(2)}
    order = []                              # one ring: (kind, item, tile) in the order of use

    def place(kind, it, i):                 # (full / empty barrier's name, number of its use)
        if one_ring:
            x = order.index((kind, it, i))
            return x % (2 * slots), x // (2 * slots)
        x = sum(max(items[j]) for j in range(it)) + i
        return f"{kind}{x % slots}", x // slots

    for it, n in enumerate(items):
        t = max(n)
        for i in range(t):
            order.append(("K", it, i))
            if i:
                order.append(("V", it, i - 1))
        if t:
            order.append(("V", it, t - 1))
    for it, n in enumerate(items):
        for i in range(max(n)):
            for kind in "KV":
                s, _ = place(kind, it, i)
                m.bar(f"full {s}", 1)
                m.bar(f"empty {s}", 1)
    looks = 8 if one_ring else slots
    for s in range(looks):
        m.bar(f"clean {s}", 1)
    for s in range(4):
        m.bar(f"given {s}", 1)
        m.bar(f"taken {s}", len(soft) + 3)
    m.bar("sread", 2)
    for w in tiles:
        for b, n in (("qfull", 1), ("qempty", 1), ("sfull", 1), ("odone", 1), ("pfull 0", 2 if first_half_waits_for_both else 1), ("pfull 1", 1), ("pair", 2)):
            m.bar(f"{b} {w}", n)

    formed, used, steps, pairs, looked = 0, [0, 0], [0, 0], [0, 0], 0
    for it, n in enumerate(items):
        slot, turn = it % 4, it // 4
        if turn:
            loader.append(("wait", f"taken {slot}", turn - 1))
        loader.append(("arrive", f"given {slot}"))

        def rows(w):
            if n[w]:
                if used[w]:
                    loader.append(("wait", f"qempty {w}", used[w] - 1))
                loader.append(("load", f"qfull {w}", f"Q {w}", it))

        def part(kind, i):
            s, use = place(kind, it, i)
            if use:
                loader.append(("wait", f"empty {s}", use - 1))
            loader.append(("load", f"full {s}", f"part {s}", (kind, it, i)))

        t = max(n)
        rows(0)
        for i in range(t):
            part("K", i)
            if i == 0:
                rows(1)
            else:
                part("V", i - 1)
        if t:
            part("V", t - 1)
        for prog in (scores, values, looker, *soft.values()):
            prog.append(("wait", f"given {slot}", turn))
        for i in range(t):                  # S
            s, use = place("K", it, i)
            scores.append(("wait", f"full {s}", use))
            for w in tiles:
                if i >= n[w]:
                    continue
                if i == 0:
                    scores.append(("wait", f"qfull {w}", used[w]))
                if formed:
                    scores.append(("wait", "sread", formed - 1))
                formed += 1
                scores.append(("mma", [(f"part {s}", ("K", it, i)), (f"Q {w}", it)], [("S", (w, it, i))], [f"sfull {w}"] + ([f"qempty {w}"] if i + 1 == n[w] else [])))
            scores[-1][3].append(f"empty {s}")
        for i in range(t):                  # the looker, P V
            s, use = place("V", it, i)
            looker += [("wait", f"full {s}", use), ("do", [(f"part {s}", ("V", it, i))], [(f"part {s}", ("V", it, i))]), ("arrive", f"clean {(looked + i) % looks}")]
            values.append(("wait", f"clean {(looked + i) % looks}", (looked + i) // looks))
            for w in tiles:
                if i >= n[w]:
                    continue
                for h in range(2):
                    values.append(("wait", f"pfull {h} {w}", steps[w] + i))
                    values.append(("mma", [(f"part {s}", ("V", it, i)), (f"P {w} {h}", (it, i))] + [(f"scaled {w} {x}", (it, i)) for x in range(2)],
                                   [(f"O {w}", (it, i))] if h else [], [f"odone {w}"] if h else []))
            values[-1][3].append(f"empty {s}")
        if one_ring:                        # the looker waited for K parts too, in the order of use
            del looker[-3 * t:]
            for kind, _, i in [x for x in order if x[1] == it]:
                s, use = place(kind, it, i)
                looker.append(("wait", f"full {s}", use))
                if kind == "V":
                    looker += [("do", [(f"part {s}", ("V", it, i))], [(f"part {s}", ("V", it, i))]), ("arrive", f"clean {(looked + i) % looks}")]
        looked += t
        for (w, h), prog in soft.items():
            swap = pairs[w]
            for i in range(n[w]):
                prog += [("wait", f"sfull {w}", steps[w] + i), ("do", [("S", (w, it, i))], []), ("arrive", "sread")]
                prog += [("arrive", f"pair {w}"), ("wait", f"pair {w}", swap)]
                swap += 1
                if i:                       # the base has risen: O of the tile before, times a factor
                    prog.append(("wait", f"odone {w}", steps[w] + i - 1))
                    prog.append(("do", [(f"O {w}", (it, i - 1))], []))
                prog.append(("do", [], [(f"scaled {w} {h}", (it, i))]))
                if h and first_half_waits_for_both:
                    prog.append(("arrive", f"pfull 0 {w}"))
                prog += [("do", [], [(f"P {w} {h}", (it, i))]), ("arrive", f"pfull {h} {w}")]
            if n[w]:
                prog += [("arrive", f"pair {w}"), ("wait", f"pair {w}", swap), ("wait", f"odone {w}", steps[w] + n[w] - 1), ("do", [(f"O {w}", (it, n[w] - 1))], [])]
            prog.append(("arrive", f"taken {slot}"))
        for w in tiles:
            pairs[w] += n[w] + (1 if n[w] else 0)
            steps[w] += n[w]
            used[w] += 1 if n[w] else 0
        for prog in (scores, values, looker):
            prog.append(("arrive", f"taken {slot}"))
    return m


@pytest.mark.parametrize("items,slots", [([(4, 0)], 2), ([(5, 0)], 4), ([(1, 0)] * 4, 2), ([(3, 0), (1, 0)], 2), ([(2, 0), (0, 0), (1, 0)], 2), ([(1, 1)], 2), ([(2, 1)], 2),
                                         ([(1, 2)], 2)])
def test_protocol_has_no_wrong_state(items, slots):
    assert search(kernel(items, slots)) > 1000


@pytest.mark.parametrize("items", [[(3, 0)], [(2, 0), (1, 0)]])
def test_search_finds_one_ring_for_both(items):
    """A warp that looks at V parts alone, in a ring through which K parts go too, is overtaken."""
    with pytest.raises(Wrong, match="overtaken"):
        search(kernel(items, 2, one_ring=True))


@pytest.mark.parametrize("items", [[(2, 0)], [(1, 0)] * 2])
def test_search_finds_products_beside_scaling(items):
    """A product that takes the first half's P adds to an O that the second half's warps are still scaling, or reading."""
    with pytest.raises(Wrong, match="product finds"):
        search(kernel(items, 2, first_half_waits_for_both=False))
