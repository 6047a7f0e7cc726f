"""The prompt kernel's schedule, on the CPU: a model of its warps as processes over the kernel's barriers.

The loads, the queries, the score products, the value products and the rows of the two row tiles wait
for one another through mbarriers, whose waits only tell two phases apart, over rings of shared memory.
The model steps the processes in random order, with the kernel's waits and parities, over random rows,
groups, windows, first tokens and parts, and looks for a wait that nothing ends, a buffer that is
overwritten or read before its time, a key tile that no row tile needs, and a visible key that no step
covers."""
from __future__ import annotations

import random

import pytest

TILE, ROWS = 128, 256


def spans(pos0, rows, group, head0, window, q_sinks, part=None):
    """The item of one unit: ([key tile at or after i, per row tile], first key tile, end), as the kernel
    plans it; None where no row sees a key."""
    position = lambda r: pos0 + (head0 + r) // group  # noqa: E731
    lo, hi = pos0, position(rows - 1)
    if hi < 0:
        return None
    begin = lo + 1 - window if window and lo + 1 > window else 0
    sinks = min(q_sinks, begin)
    if sinks == begin:
        sinks = begin = 0
    n_keys = sinks + hi + 1 - begin
    end = begin + n_keys - sinks
    start = begin // TILE
    first = min(start, -(-sinks // TILE))
    n = first + (end - 1) // TILE - start + 1
    a, z = (0, n) if part is None else (n * part[0] // part[1], n * (part[0] + 1) // part[1])
    key0 = lambda i: (i if i < first else i - first + start) * TILE  # noqa: E731
    out = []
    for t in range(2):
        s = dict(first=0, begin=0, end=0)
        if t * 128 < rows:
            t_lo, t_hi = position(t * 128), position(min(rows, (t + 1) * 128) - 1)
            if t_hi >= 0:
                s = dict(first=first, begin=first, end=min(z, first + t_hi // TILE - start + 1))
                if begin > 0 and sinks <= start * TILE:
                    s["begin"] += max(0, (t_lo + 1 - window) // TILE - start)

        def at(i, s=s):
            i = i if i < s["first"] else max(i, s["begin"])
            return i if i < s["end"] else z

        out.append(at)
        if part is None and t * 128 < rows:
            need, i = set(), at(a)
            while i < z:
                need.add(key0(i))
                i = at(i + 1)
            for r in {t * 128, min(rows, (t + 1) * 128) - 1, min(rows - 1, t * 128 + 64)}:
                p = position(r)
                seen = range(max(0, p - window + 1 if window else 0), p + 1)
                some = list(seen[::7]) + list(seen[-1:]) + (list(range(min(q_sinks, p + 1))) if window else [])
                assert all(j // TILE * TILE in need for j in some)
    for i in range(a, z):
        assert any(at(i) == i for at in out), "a key tile that no row tile needs"
    return out, a, z


class Bar:
    """An mbarrier: phases, and a wait that knows the parity alone."""

    def __init__(self):
        self.phase = 0

    def arrive(self):
        self.phase += 1

    def passed(self, parity):
        return (self.phase - 1) & 1 == parity & 1


def run(items, stages, rng):
    many = lambda n: [Bar() for _ in range(n)]  # noqa: E731
    k_full, k_empty, v_full, v_empty = many(stages), many(stages), many(stages), many(stages)
    s_full, s_read, p_full, o_empty, q_full, q_empty = many(2), many(2), many(2), many(2), many(2), many(2)
    o_done = [many(2), many(2)]
    ring, score = {}, [None, None, "read"]  # what the stages hold; tile, key tile and state of S

    def loads():
        turn = 0
        for _, a, z in items:
            for _ in range(a, z):
                st, parity = turn % stages, ((turn // stages) & 1) ^ 1
                while not k_empty[st].passed(parity):
                    yield
                ring["K", st] = turn
                k_full[st].arrive()
                yield
                while not v_empty[st].passed(parity):
                    yield
                ring["V", st] = turn
                v_full[st].arrive()
                yield
                turn += 1

    def queries():
        turn = 0
        for at, a, z in items:
            for t in range(2):
                if at[t](a) >= z:
                    continue
                while not q_empty[t].passed((turn >> t & 1) ^ 1):
                    yield
                turn ^= 1 << t
                q_full[t].arrive()
                yield

    def scores():
        turn, q_turn, read, last = 0, 0, 3, 0
        for at, a, z in items:
            for i in range(a, z):
                st = turn % stages
                while not k_full[st].passed(turn // stages):
                    yield
                for t in range(2):
                    if at[t](i) != i:
                        continue
                    if i == at[t](a):
                        while not q_full[t].passed(q_turn >> t):
                            yield
                    while not s_read[last].passed(read >> last):
                        yield
                    last = t
                    read ^= 1 << t
                    assert ring["K", st] == turn and score[2] == "read"
                    score[:] = [t, turn, "full"]
                    s_full[t].arrive()
                    if at[t](i + 1) >= z:
                        q_turn ^= 1 << t
                        q_empty[t].arrive()
                    yield
                k_empty[st].arrive()
                turn += 1
                yield

    def values():
        turn, p_turn, active = 0, [0, 0], 0
        for at, a, z in items:
            for i in range(a, z):
                st = turn % stages
                while not v_full[st].passed(turn // stages):
                    yield
                for t in range(2):
                    if at[t](i) != i:
                        continue
                    if i == at[t](a):
                        while not o_empty[t].passed((active >> t & 1) ^ 1):
                            yield
                        active ^= 1 << t
                    while not p_full[t].passed(p_turn[t]):
                        yield
                    assert ring["V", st] == turn
                    o_done[t][p_turn[t] & 1].arrive()
                    p_turn[t] += 1
                    yield
                v_empty[st].arrive()
                turn += 1
                yield

    def rows(t):
        turn = base = 0
        for at, a, z in items:
            i = first = at[t](a)
            while i < z:
                while not s_full[t].passed(turn):
                    yield
                assert score == [t, base + i - a, "full"]
                score[2] = "read"
                s_read[t].arrive()
                yield
                if turn:
                    while not o_done[t][turn - 1 & 1].passed(turn - 1 >> 1):
                        yield
                p_full[t].arrive()
                turn += 1
                yield
                i = at[t](i + 1)
            if first < z:
                while not o_done[t][turn - 1 & 1].passed(turn - 1 >> 1):
                    yield
                o_empty[t].arrive()
                yield
            base += z - a

    bars = [b for group in (k_full, k_empty, v_full, v_empty, s_full, s_read, p_full, o_empty, q_full, q_empty, *o_done)
            for b in group]
    alive, idle = [loads(), queries(), scores(), values(), rows(0), rows(1)], 0
    while alive:
        p = rng.choice(alive)
        before = [b.phase for b in bars]
        try:
            next(p)
        except StopIteration:
            alive.remove(p)
            idle = 0
            continue
        idle = 0 if before != [b.phase for b in bars] else idle + 1
        assert idle < 2000, "a wait that nothing ends"


@pytest.mark.parametrize("seed", range(4))
def test_schedule(seed):
    rng = random.Random(seed)
    for _ in range(150):
        group = rng.choice([1, 1, 2, 3, 4, 5, 7, 8, 16, 17, 40, 128, 200, 1000])
        window = rng.choice([0, rng.randint(1, 70), rng.randint(1, 400), rng.randint(1, 1500)])
        sinks = rng.choice([0, 1, 4, rng.randint(0, 300), rng.randint(0, 1000)])
        items = []
        for _ in range(rng.randint(1, 4)):
            part = rng.choice([None, None, (0, 2), (1, 2), (1, 3)])
            item = spans(rng.choice([rng.randint(-50, 300), rng.randint(0, 1500)]),
                         rng.choice([ROWS, rng.randint(1, ROWS)]), group, rng.randrange(group), window, sinks, part)
            if item:
                items.append(item)
        for stages in (1, 2, 4):
            run(items, stages, rng)
