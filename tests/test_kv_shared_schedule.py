"""How the work over shared and own keys is cut into runs (csrc/kv_shared.cuh, Runs), on the CPU: a model of its 32-bit
arithmetic over random groups, sequences, rows, workers and coarse counts.  Every unit's key tiles are covered once and in
order, its parts lie side by side in slots that no other unit has, and the first slot and the number of parts that the join
reads are those that were written."""
from __future__ import annotations

import random

import pytest


def tiles(keys, begin, end):
    if end <= begin:
        return 0
    return (end - begin + keys - 1) // keys if keys == 16 else (end - 1) // keys - begin // keys + 1


def runs(rows_of_unit, keys, lead, elements, group, heads, workers, least, coarse):
    """elements: (own, tokens, begin, end); the slots used."""
    lead >>= coarse

    def blocks_of(e):
        return (e[1] * group + rows_of_unit - 1) // rows_of_unit if e[3] > e[2] else 0

    def tiles_of(e, b):
        rows = min(e[1] * group, (b + 1) * rows_of_unit)
        return tiles(keys, e[2], e[3] - e[1] + (rows - 1) // group + 1 if e[0] else e[3])

    def counted(n):
        return max(1, (n + (1 << coarse) - 1) >> coarse) + lead

    row, upto, units_upto = [], 0, 0
    for number, e in enumerate(elements):
        blocks = blocks_of(e)
        paired = e[0] and blocks > 1
        pairs = (blocks + 1) // 2 if paired else blocks
        work = counted(tiles_of(e, blocks - 1)) + (counted(tiles_of(e, 0)) if paired else 0) if blocks else 0
        upto += pairs * heads * work
        side = 2 if paired else 1
        units_upto += side * pairs * heads
        row.append((number, e, blocks, pairs, work, upto, units_upto, side))
    length = max(max(1, least >> coarse), (upto + workers - 1) // workers)
    assert upto < 1 << 31
    covered, parts, slots = {}, {}, set()
    for w in range(workers):
        x = min(w * length, upto)
        end = min(x + length, upto)
        while x < end:
            number, e, blocks, pairs, each, last, units_last, side = next(i for i in row if x < i[5])
            units = pairs * heads
            into = x - (last - units * each)
            at, off = divmod(into, each)
            pair, g = divmod(at, heads)
            block = blocks - 1 - pair if e[0] else pair
            n, which = tiles_of(e, block), 0
            of_unit = min(counted(n), each) if e[0] and blocks > 1 and block != pair else each
            if off >= of_unit:
                off -= of_unit
                of_unit = each - of_unit
                block, which = pair, 1
                n = tiles_of(e, block)
            unit_x = x - off
            key_x, to = unit_x + lead, min(end, unit_x + of_unit)
            if to <= key_x:  # the run ends in the unit's start
                break
            first = x <= key_x
            a = 0 if first else min((x - key_x) << coarse, n)
            b = n if to == unit_x + of_unit else min((to - key_x) << coarse, n)
            slot = w + units_last - side * units + side * at + which
            assert slot not in slots
            slots.add(slot)
            covered.setdefault((number, block, g), []).append((a, b, slot))
            if first:
                assert (number, block, g) not in parts
                parts[number, block, g] = slot, (unit_x + of_unit - 1) // length - w + 1
            x = to
    for number, e, blocks, *_ in row:
        for b in range(blocks):
            for g in range(heads):
                first, count = parts[number, b, g]
                pieces = covered[number, b, g]
                assert [p[2] for p in pieces] == list(range(first, first + count))
                at = 0
                for begin, end, _ in pieces:
                    assert begin == at
                    at = end
                assert at == tiles_of(e, b)
    return slots, units_upto


@pytest.mark.parametrize("seed", range(8))
def test_runs(seed):
    rng = random.Random(seed)
    for _ in range(100):
        group, heads = rng.choice([1, 2, 3, 5, 8, 17, 40, 300]), rng.choice([1, 2, 3, 8])
        rows_of_unit, keys = rng.choice([(16, 16), (256, 128)])
        elements = []
        for _ in range(rng.randint(1, 9)):
            own, tokens = rng.random() < 0.6, rng.choice([0, 1, 1, 2, 5, 40, 300])
            begin = rng.choice([0, 5, 100, 130]) if own else 0
            # all that is shared is before a sequence's first new token, but for one
            end = (begin + max(tokens - 1, 0) + rng.choice([0, 1, 7, 200])) if own else rng.choice([0, 1, 50, 700])
            elements.append((own, tokens, begin, end))
        workers = rng.choice([1, 3, 148, 592])
        slots, units = runs(rows_of_unit, keys, rng.choice([0, 3]), elements, group, heads, workers, rng.choice([1, 4]),
                            rng.choice([0, 0, 0, 1, 3]))
        assert not slots or max(slots) < workers + units
        # the host's bound on the units' numbers
        total = sum(e[1] for e in elements)
        assert units <= (total * group // rows_of_unit + 2 * len(elements)) * heads
