"""Who waits for whom in the wide form of attention over pages (csrc/paged_attention_many.cuh), without a GPU: the copying warp, the two issuing warps and the two
streams of rows as coroutines over barriers that count arrivals and are waited for by the parity of a phase, in random order. Nothing may wait for
ever, no barrier may be given more arrivals than it takes, and a wait that looks at a parity must not be two phases late."""
import random

import pytest

UNIT = 64


class Barrier:
    def __init__(self, arrivals=1):
        self.arrivals, self.count, self.phase = arrivals, 0, 0

    def arrive(self, n=1):
        self.count += n
        assert self.count <= self.arrivals, "more arrivals than the phase takes"
        if self.count == self.arrivals:
            self.count, self.phase = 0, self.phase + 1

    def wait(self, parity):
        while (self.phase & 1) == parity:
            yield


class Ring:
    """A role's place in the ring."""

    def __init__(self, slots):
        self.slots, self.slot, self.parity = slots, 0, 0

    def next(self):
        self.slot += 1
        if self.slot == self.slots:
            self.slot, self.parity = 0, self.parity ^ 1


def streams(p, slots):
    """Every other unit to a stream, or the units of both; how many units of keys come before values."""
    halves = min(256, p["nr"] - p["t"] * 256) <= 128
    n, lead = p["n"], min(p["n"], 4 if halves and slots >= 7 else 2)
    if halves:
        return True, [(n + 1) // 2, n // 2], lead
    seen = p["keys"] - p["rows"] + (p["t"] * 256 + 127) // p["G"] + 1 if p["own"] else p["keys"]
    return False, [max(0, min(n, -(-seen // UNIT) - p["k0"])), n], lead


def run(pieces, slots, rng):
    full, empty = [Barrier() for _ in range(slots)], [Barrier(2) for _ in range(slots)]
    queries, done = [Barrier(), Barrier()], Barrier(2)
    scores, weights, sums = ([[Barrier(), Barrier()] for _ in range(2)] for _ in range(3))
    alone, both = [Barrier(), Barrier()], Barrier(2)

    def copies():
        at = Ring(slots)
        for p in pieces:
            for _ in range(2 * p["n"]):
                yield from empty[at.slot].wait(at.parity ^ 1)
                yield
                full[at.slot].arrive()
                at.next()

    def products(s):
        at, turn, parity = Ring(slots), 0, [0, 0]
        for p in pieces:
            halves, units, lead = streams(p, slots)
            n, mine = p["n"], units[s]
            for q in queries:
                yield from q.wait(turn & 1)
            turn += 1

            def step(kind, place):
                yield from full[at.slot].wait(at.parity)
                if kind == "pass":
                    empty[at.slot].arrive()
                    return
                if kind == "sums":
                    yield from weights[s][place].wait(parity[place])
                    parity[place] ^= 1
                (scores if kind == "scores" else sums)[s][place].arrive()
                empty[at.slot].arrive(2 if halves else 1)

            for j in range(-lead, n):                          # values j, then keys j + lead
                for kind, unit in ([("sums", j)] if j >= 0 else []) + ([("scores", j + lead)] if j + lead < n else []):
                    if halves:
                        if unit & 1 == s:
                            yield from step(kind, unit >> 1 & 1)
                    else:
                        yield from step(kind if unit < mine else "pass", unit & 1)
                    at.next()
            done.arrive()

    def rows(s):
        turn = item = seen_alone = seen_both = 0
        parity, before = [0, 0], [0, 0]
        for p in pieces:
            halves, units, lead = streams(p, slots)
            n, mine = p["n"], units[s]
            yield
            queries[s].arrive()

            def settled(j):
                if j:
                    i = j - 1
                    yield from sums[s][i & 1].wait((before[i & 1] + i // 2) & 1)
                    assert sums[s][i & 1].phase >= before[i & 1] + i // 2 + 1, "taken for a later phase"

            for j in range(mine):
                unit, place = 2 * j + s if halves else j, j & 1
                yield from scores[s][place].wait(parity[place])
                parity[place] ^= 1
                yield
                if rng.random() < 0.3:                          # a larger score: the sums are rescaled
                    yield from settled(j)
                if (p["k0"] + unit + 1) * UNIT > p["limit"]:    # some rows do not see all of these keys: the values are looked at
                    value = item + lead + unit + min(unit, n - lead)
                    yield from full[value % slots].wait(value // slots & 1)
                    assert full[value % slots].phase >= value // slots + 1
                    if not halves and unit < units[0]:
                        both.arrive()
                        yield from both.wait(seen_both)
                        seen_both ^= 1
                    else:
                        alone[s].arrive()
                        yield from alone[s].wait(seen_alone)
                        seen_alone ^= 1
                weights[s][place].arrive()
            yield from settled(mine)
            yield from done.wait(turn & 1)
            turn, item = turn + 1, item + 2 * n
            before[0] += (mine + 1) // 2
            before[1] += mine // 2

    live = {"copies": copies(), "products 0": products(0), "products 1": products(1), "rows 0": rows(0), "rows 1": rows(1)}
    every = full + empty + queries + [done, both] + alone + [b for kind in (scores, weights, sums) for pair in kind for b in pair]
    idle, last = 0, None
    while live:
        name = rng.choice(list(live))
        try:
            next(live[name])
        except StopIteration:
            del live[name]
            idle = 0
        state = [(b.phase, b.count) for b in every]
        idle, last = (idle + 1, last) if state == last else (0, state)
        assert idle < 5000, f"{sorted(live)} wait for ever"


@pytest.mark.parametrize("slots", [6, 7, 9, 12])              # 6: the most requests and groups, hd 128; 9: few of them; 12: hd 64
def test_every_wait_ends(slots):
    rng = random.Random(slots)
    for _ in range(250):
        pieces = []
        for _ in range(rng.randint(1, 5)):
            G, rows = rng.choice([1, 4, 5]), rng.choice([5, 8, 9, 40, 64, 70, 200])
            if rows * G <= 32:
                continue
            t, own = rng.randrange((rows * G + 255) // 256), rng.random() < 0.6
            keys = rows + rng.randrange(600) if own else rng.randint(1, 900)
            seen = keys - rows + (min((t + 1) * 256, rows * G) - 1) // G + 1 if own else keys
            units = -(-seen // UNIT)
            k0 = rng.randrange(units)
            pieces.append(dict(n=rng.randint(1, units - k0), nr=rows * G, t=t, own=own, keys=keys, rows=rows, G=G, k0=k0, limit=keys - rows + t * 256 // G + 1 if own else keys))
        run(pieces, slots, rng)
