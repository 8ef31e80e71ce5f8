"""The ring of page tiles in the tensor-memory attention kernel (ttq_paged_tc.cu), as a model on the CPU.

Two product warps read one ring of slots that one copying warp fills.  A barrier's parity tells a phase only from its neighbours,
so a warp that skips a fill may take the phase before it for the one that it waits for.  The model runs the kernel's warps, their
barriers, the copies in flight and the tensor core's queue in random order; every product checks that the slot it reads holds the
tile that it means.
"""
import random

import pytest


class Barrier:
    """An mbarrier: `count` arrivals complete a phase; a wait passes while the phase of the other parity is the running one."""

    def __init__(self, count):
        self.count = self.left = count
        self.phase = 0

    def arrive(self):
        self.left -= 1
        assert self.left >= 0
        if self.left == 0:
            self.phase, self.left = self.phase + 1, self.count

    def passes(self, parity):
        return (self.phase & 1) != parity


class Stale(Exception):
    pass


def simulate(items, slots, every_fill, rng):
    """items: (units, pair).  `every_fill`: both product warps see every fill, and let go of the other's at once (the kernel's rule);
    else each waits for its own units only, whose slots it frees twice in an item of one stream."""
    full, empty = [Barrier(1) for _ in range(slots)], [Barrier(2) for _ in range(slots)]
    holds = [-1] * slots
    s_full, p_full = [[Barrier(1) for _ in range(2)] for _ in range(2)], [[Barrier(1) for _ in range(2)] for _ in range(2)]
    q_full, q_empty, done = [Barrier(1) for _ in range(2)], [Barrier(1) for _ in range(2)], [0, 0]
    records, read = 0, [0] * 3   # items published; items that the copying and the product warps have taken
    queues = [[], []]            # products of the streams, in the order of issue
    flight = []                  # copies that have not landed: (what, slot or stream)

    def copier():
        n = 0
        for k, (m, _) in enumerate(items):
            yield lambda: records > k
            read[2] = k + 1
            for _ in range(2 * m):
                if n >= slots:
                    yield lambda: empty[n % slots].passes((n // slots - 1) & 1)
                flight.append((n, n % slots))
                n += 1

    def walker():
        nonlocal records
        used = [0, 0]
        for k, (m, pair) in enumerate(items):
            yield lambda: min(read + done) > k - 4
            records = k + 1
            for st in range(2 if pair or m > 1 else 1):
                if used[st]:
                    yield lambda: q_empty[st].passes((used[st] - 1) & 1)
                used[st] += 1
                flight.append((None, st))

    def softmax(st):
        par = [0, 0]
        for k, (m, pair) in enumerate(items):
            yield lambda: records > k
            for _ in range(0 if pair else st, m, 1 if pair else 2):
                for h in range(2):
                    yield lambda: s_full[st][h].passes(par[h])
                    par[h] ^= 1
                    yield lambda: True
                    p_full[st][h].arrive()
            done[st] = k + 1
            if not pair:  # the streams exchange their results
                yield lambda: min(done) > k

    def products(st):
        n, seen, q_par, p_par = 0, 0, 0, [0, 0]
        for k, (m, pair) in enumerate(items):
            yield lambda: records > k
            read[st] = k + 1
            first, step = (0, 1) if pair else (st, 2)
            if first < m:
                yield lambda: q_full[st].passes(q_par)
                q_par ^= 1
            for i in list(range(first - step, m, step)) + ([None] if every_fill else []):
                if i is None:
                    wanted = [n + 2 * m - 1]  # those behind the stream's last unit
                else:
                    with_v, with_k = i >= first, i + step < m
                    wanted = [n + 2 * i + 1] * with_v + [n + 2 * (i + step)] * with_k
                for last in wanted:
                    for f in range(seen, last + 1) if every_fill else [last]:
                        yield lambda: full[f % slots].passes((f // slots) & 1)
                        if every_fill and not pair and (f - n) // 2 % 2 != st:
                            empty[f % slots].arrive()
                    seen = max(seen, last + 1)
                if i is None:
                    continue
                for h in range(2):
                    if with_v:
                        yield lambda: p_full[st][h].passes(p_par[h])
                        p_par[h] ^= 1
                    frees = 1 if pair or every_fill else 2
                    if with_v:
                        vs = n + 2 * i + 1
                        queues[st].append((vs, [empty[vs % slots]] * (frees if h else 0)))
                    if with_k:
                        ks = n + 2 * (i + step)
                        queues[st].append((ks, [s_full[st][h]] + ([empty[ks % slots]] * frees if h else []) + ([q_empty[st]] if h and i + 2 * step >= m else [])))
            n += 2 * m

    procs = [[g, next(g, None)] for g in (copier(), walker(), softmax(0), softmax(1), products(0), products(1))]
    slow = [rng.choice([0.02, 0.2, 1.0]) for _ in procs]           # some warps lag
    late = {f: rng.random() < 0.2 for f in range(2 * sum(m for m, _ in items))}   # some copies do
    while any(p[1] for p in procs) or flight or queues[0] or queues[1]:
        moves = [("proc", i) for i, p in enumerate(procs) if p[1] and p[1]()]
        moves += [("land", x) for x in flight] + [("run", st) for st in range(2) if queues[st]]
        assert moves, "the warps wait for one another"
        weights = [slow[x] if what == "proc" else (0.01 if what == "land" and late.get(x[0]) else 0.5) for what, x in moves]
        what, x = rng.choices(moves, weights)[0]
        if what == "proc":
            procs[x][1] = next(procs[x][0], None)
        elif what == "land":
            flight.remove(x)
            if x[0] is None:
                q_full[x[1]].arrive()
            else:
                holds[x[1]] = x[0]
                full[x[1]].arrive()
        else:
            fill, then = queues[x].pop(0)
            if holds[fill % slots] != fill:
                raise Stale(f"slot {fill % slots} holds tile {holds[fill % slots]}, not {fill}")
            for bar in then:
                bar.arrive()


def random_items(rng):
    return [(rng.choice([1, 1, 2, 3, 4, 5, 7]), rng.random() < 0.4) for _ in range(rng.randint(1, 8))]


@pytest.mark.parametrize("slots", [4, 8])
def test_every_product_reads_its_own_tile(slots):
    rng = random.Random(slots)
    for _ in range(400):
        simulate(random_items(rng), slots, True, rng)


def test_the_model_shows_a_skipped_fill():
    """Warps that wait for their own units only, on a ring of two units: an item of an odd number of units changes their slots."""
    rng = random.Random(0)
    with pytest.raises(Stale):
        for _ in range(2000):
            simulate([(3, False), (4, False)], 4, False, rng)
