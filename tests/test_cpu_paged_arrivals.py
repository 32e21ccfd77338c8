"""What the roles of the wide form of attention over pages (csrc/paged_attention_many.cuh) read from memory that others write, without a GPU: every warp of rows by itself, the
issuing warps, the tensor core behind them and the copies as coroutines of unlike speeds. Barriers count arrivals and are waited for by the parity of a phase. Whoever reads a place of
the ring or the marks of values that are not finite must find what was written for the unit at hand; nothing may wait for ever; a wait must not take one phase for another.

The model can be told to do without a rule of the kernel's, and has to fail then."""
import os
import random
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llm.metal_b200", "csrc", "paged_attention_many.cuh")
UNIT = 64


def source():
    with open(SOURCE) as f:
        return re.sub(r"\s+", " ", re.sub(r"//[^\n]*", "", f.read()))


class Barrier:
    def __init__(self, arrivals=1):
        self.arrivals, self.count, self.phase = arrivals, 0, 0

    def arrive(self, n=1):
        self.count += n
        assert self.count <= self.arrivals, "more arrivals than the phase takes"
        if self.count == self.arrivals:
            self.count, self.phase = 0, self.phase + 1

    def wait(self, phase):
        """For the end of this phase, by its parity."""
        while (self.phase & 1) == (phase & 1):
            yield
        assert self.phase == phase + 1, "one phase taken for another"


class Piece:
    def __init__(self, number, rng, slots):
        self.number = number
        while True:
            G, rows = rng.choice([1, 4, 5]), rng.choice([5, 8, 9, 40, 64, 70, 128, 200, 256])
            nr = rows * G
            if nr <= 32:
                continue
            self.t, own = rng.randrange((nr + 255) // 256), rng.random() < 0.7
            keys = rows + rng.randrange(600) if own else rng.randint(1, 900)
            before = rng.choice([0, 64, 100, 300]) if own and nr >= 128 else 0
            seen = lambda i: keys - rows + i // G + 1 if own else keys       # noqa: E731
            self.first = -(-before // UNIT)                      # units before the own keys
            units = self.first + -(-seen(min((self.t + 1) * 256, nr) - 1) // UNIT)
            k0 = rng.randrange(units)
            self.n = rng.randint(1, units - k0)
            self.halves = min(256, nr - self.t * 256) <= 128
            self.ahead = 4 if self.halves and slots >= 7 else 2
            self.lead = min(self.n, self.ahead)
            if self.halves:
                self.units = [(self.n + 1) // 2, self.n // 2]
            else:
                self.units = [max(0, min(self.n, self.first + -(-seen(self.t * 256 + 127) // UNIT) - k0)), self.n]
            own_all = seen(self.t * 256)
            # units of which not all rows see all keys, and those with a value among them that is not finite
            self.hidden = [((u + 1) * UNIT > before) if u < self.first else ((u - self.first + 1) * UNIT > own_all) for u in range(k0, k0 + self.n)]
            self.special = [own and rng.random() < 0.5 for _ in range(self.n)]
            self.order = []                                      # what passes through the ring: (unit, values)
            for j in range(-self.lead, self.n):
                if j >= 0:
                    self.order.append((j, True))
                if j + self.lead < self.n:
                    self.order.append((j + self.lead, False))
            return

    def values(self, j):
        at = self.lead + j + min(j, self.n - self.lead)
        assert self.order[at] == (j, True)
        return at


def run(pieces, slots, rng, buffers=2, freed_first=True):
    full, empty = [Barrier() for _ in range(slots)], [Barrier(2) for _ in range(slots)]
    holds, flying = [None] * slots, {}                           # the item that lies in a place; copies on their way and how long they take: some are late
    queues = [[], []]                                            # what the tensor core has been given by each issuing warp
    queries, done, both = [Barrier(4), Barrier(4)], Barrier(2), Barrier(8)
    scores, sums = ([[Barrier(), Barrier()] for _ in range(2)] for _ in range(2))
    weights, alone = [[Barrier(4), Barrier(4)] for _ in range(2)], [Barrier(4), Barrier(4)]
    marks = [[None, None] for _ in range(6)]
    starts = [0]
    for p in pieces:
        starts.append(starts[-1] + 2 * p.n)

    def copies():
        for item in range(starts[-1]):
            slot = item % slots
            yield from empty[slot].wait(item // slots - 1)
            yield
            assert not any(kind == "read" and at % slots == slot for q in queues for kind, at, _ in q), "written while it is read"
            holds[slot] = None
            flying[item] = int(10 ** rng.uniform(0, 2.5))

    def landing():
        while True:
            for item in list(flying):
                flying[item] -= 1
                if not flying[item]:
                    del flying[item]
                    holds[item % slots] = item
                    full[item % slots].arrive()
            yield

    def tensor(s):
        while True:
            if queues[s]:
                kind, x, n = queues[s].pop(0)
                if kind == "read":
                    assert holds[x % slots] == x, "another unit's keys or values"
                else:
                    x.arrive(n)
            yield

    def products(s):
        used = [0, 0]
        for turn, p in enumerate(pieces):
            for q in queries:
                yield from q.wait(turn)
            n, mine = p.n, p.units[s]
            for at, (unit, values) in enumerate(p.order):
                item = starts[turn] + at
                slot = item % slots
                if p.halves and unit & 1 != s:
                    continue
                if p.halves and freed_first:
                    yield from empty[slot].wait(item // slots - 1)
                yield from full[slot].wait(item // slots)
                if not p.halves and unit >= mine:
                    empty[slot].arrive()
                    continue
                place = (unit >> 1 if p.halves else unit) & 1
                if values:
                    yield from weights[s][place].wait(used[place])
                    used[place] += 1
                queues[s] += [("read", item, 0), ("commit", (sums if values else scores)[s][place], 1)] + [("commit", empty[slot], 1)] * (2 if p.halves else 1)
                yield
            queues[s].append(("commit", done, 1))

    def rows(s, w):
        seen_alone = seen_both = 0
        got, before = [0, 0], [0, 0]
        for turn, p in enumerate(pieces):
            mine = p.units[s]
            yield
            queries[s].arrive()

            def settled(j):
                if j:
                    i = j - 1
                    yield from sums[s][i & 1].wait(before[i & 1] + i // 2)

            for j in range(mine):
                unit, place = 2 * j + s if p.halves else j, j & 1
                yield from scores[s][place].wait(got[place])
                got[place] += 1
                yield
                if rng.random() < 0.3:                           # a larger score: the sums are rescaled
                    yield from settled(j)
                if p.hidden[unit]:
                    item = starts[turn] + p.values(unit)
                    if p.halves and freed_first:
                        yield from empty[item % slots].wait(item // slots - 1)
                    yield from full[item % slots].wait(item // slots)
                    assert holds[item % slots] == item, "values of another unit"
                    together = not p.halves and unit < p.units[0]
                    if together:
                        index = 4 + (seen_both & 1)
                    else:
                        index = 2 * s + (seen_alone & 1 if buffers == 2 else 0)
                    looks = not together or s == 0
                    if looks and w < 2:
                        marks[index][w] = (turn, unit)

                    def meet():
                        nonlocal seen_alone, seen_both
                        bar, phase = (both, seen_both) if together else (alone[s], seen_alone)
                        bar.arrive()
                        if together:
                            seen_both += 1
                        else:
                            seen_alone += 1
                        yield from bar.wait(phase)

                    yield from meet()
                    yield
                    assert marks[index] == [(turn, unit)] * 2, "marks of another unit"
                    if p.special[unit]:
                        yield from settled(j)
                        yield
                        assert marks[index] == [(turn, unit)] * 2 and holds[item % slots] == item, "marks of another unit"
                        yield from meet()
                        yield
                        yield from meet()
                weights[s][place].arrive()
            yield from settled(mine)
            yield from done.wait(turn)
            before[0] += (mine + 1) // 2
            before[1] += mine // 2

    live = {"copies": copies(), "landing": landing(), **{("tensor", s): tensor(s) for s in range(2)}, **{("products", s): products(s) for s in range(2)},
            **{("rows", s, w): rows(s, w) for s in range(2) for w in range(4)}}
    every = full + empty + queries + [done, both] + alone + [b for kind in (scores, weights, sums) for pair in kind for b in pair]
    names, speed = list(live), [10 ** rng.uniform(-2, 0) for _ in live]
    left, idle, last = 11, 0, None                               # (the tensor core and the landing of copies have no end)
    while left:
        for name in rng.choices(names, speed, k=64):
            if name in live:
                try:
                    next(live[name])
                except StopIteration:
                    del live[name]
                    left -= 1
        state = [(b.phase, b.count) for b in every], sum(flying.values()), [len(q) for q in queues], left
        idle, last = (idle + 1, last) if state == last else (0, state)
        assert idle < 500, f"{sorted(map(str, live))} wait for ever"


def runs(n, slots, seed, **rules):
    for k in range(n):
        rng = random.Random(1000 * seed + k)
        run([Piece(i, rng, slots) for i in range(rng.randint(1, 4))], slots, rng, **rules)


@pytest.mark.parametrize("slots", [6, 7, 8, 9, 10, 12])
def test_everyone_reads_what_was_written_for_the_unit(slots):
    runs(120, slots, slots)


@pytest.mark.parametrize("slots", [6, 8, 9])
def test_waiting_for_the_own_copy_alone_is_not_enough(slots):
    """Where the other stream's keys have yet to land in the place before, its barrier has the parity of an earlier phase's end."""
    with pytest.raises(AssertionError, match="one phase taken for another|another unit"):
        runs(3000, slots, 2, freed_first=False)


def test_one_buffer_of_marks_is_not_enough():
    with pytest.raises(AssertionError, match="marks of another unit"):
        runs(400, 9, 1, buffers=1)


def test_the_kernel_waits_for_the_place_first():
    s = source()
    assert "(!halves || wait_or_abort(&empty_bar[slot], phase ^ 1, abort_flag)) && wait_or_abort(&full_bar[slot], phase, abort_flag)" in s
    assert s.count("is_there(") == 3 and s.count("&full_bar[") == 5      # by rows, for scores and for sums; besides: set up, filled twice, passed on


def test_the_kernel_has_two_buffers_of_marks():
    s = source()
    assert "special_sh[6][2]" in s and "found = special_sh[both ? 4 + both_phase : 2 * s + alone_phase]" in s
