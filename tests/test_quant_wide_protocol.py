"""The barriers between the roles of the many-slot attention kernel (csrc/kernels/quant_wide.cu), played on the CPU.

Copy, converter, matrix and softmax warps run at random paces, bulk copies land and products end in random order, and
every wait asserts that what it stands for has happened: a wait looks at the parity of a phase alone, so a barrier that
may be two phases ahead would let it through.  The numbers of barriers, arrivals and kept units are the source's own.
"""

import os
import random
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
TEXT = open(os.path.join(ROOT, "csrc", "kernels", "quant_wide.cu")).read()


def constant(name):
    return int(re.search(rf"\b{name} = (\d+)[,;]", TEXT).group(1))


BLOCKS = 4                                   # of a tile
SOFT, CONV, MAX_RAW = constant("SOFT") // 32, constant("CONV") // 32, constant("MAX_RAW")


def test_the_source_is_what_is_played():
    for line in ("constexpr int UNITS = MAX_RAW + 2;", "constexpr int TBLOCKS = WIDE_KEYS / TOK;", "mbar_init(&s.raw_empty[i], TBLOCKS);",
                 "mbar_init(&s.k_full[i], TBLOCKS);", "mbar_init(&s.v_full[i], TBLOCKS);", "mbar_init(&s.s_full[i], 1);",
                 "mbar_init(&s.p_full[i], SOFT / 32);", "mbar_init(&s.o_full[i], 1);", "mbar_init(&s.raw_full[i], 1);",
                 "mbar_init(&s.k_empty[i], 1);", "mbar_init(&s.v_empty[i], 1);", "mbar_init(&s.q_full, SOFT / 32);",
                 "uint64_t raw_full[4], raw_empty[MAX_RAW];", "k_full[2], v_full[2], k_empty[4], v_empty[4], s_full[2], p_full[2], o_full[2], q_full;",
                 "wait_for(s, &s.raw_full[i & 3], (i >> 2) & 1, a.err)", "wait_for(s, &s.k_empty[(i - 2) & 3], ((i - 2) >> 2) & 1, a.err)",
                 "wait_for(s, &s.v_empty[(i - 2) & 3], ((i - 2) >> 2) & 1, a.err)", "wait_for(s, &s.k_full[b], (i >> 1) & 1, a.err)",
                 "wait_for(s, &s.v_full[b], (i >> 1) & 1, a.err)", "wait_for(s, &s.p_full[b], (i >> 1) & 1, a.err)",
                 "wait_for(s, &s.s_full[b], (i >> 1) & 1, a.err)", "wait_for(s, &s.o_full[b], ((i >> 1) - 1) & 1, a.err)",
                 "wait_for(s, &s.o_full[b ^ 1], ((i - 1) >> 1) & 1, a.err)", "wait_for(s, &s.raw_empty[st], phase, a.err)"):
        assert line in TEXT, line
    assert (SOFT, CONV, MAX_RAW) == (16, 14, 4)


class Barrier:
    def __init__(self, arrivals):
        self.arrivals, self.count, self.phase = arrivals, 0, 0

    def arrive(self):
        self.count += 1
        if self.count == self.arrivals:
            self.count, self.phase = 0, self.phase + 1

    def passed(self, parity):   # as a try_wait on the parity
        return (self.phase & 1) != parity


class Play:
    """One CTA that walks `pieces` (tiles of each) with `ring` places for raw tiles, `units` kept units and
    `depth` barriers in turn that say an image is free."""

    def __init__(self, pieces, ring, units, seed, depth=4):
        self.pieces, self.ring, self.units, self.rng, self.seed, self.depth = pieces, ring, units, random.Random(seed), seed, depth
        bars = lambda n, arrivals: [Barrier(arrivals) for _ in range(n)]  # noqa: E731
        self.raw_full, self.raw_empty = bars(4, 1), bars(ring, BLOCKS)
        self.k_full, self.v_full, self.k_empty, self.v_empty = bars(2, BLOCKS), bars(2, BLOCKS), bars(depth, 1), bars(depth, 1)
        self.s_full, self.p_full, self.o_full, self.q_full = bars(2, 1), bars(2, SOFT), bars(2, 1), Barrier(SOFT)
        self.copies, self.landed = [], set()            # under way; tiles
        self.products, self.scores, self.outputs = [], 0, 0   # in order; finished
        self.read = [0] * SOFT                          # tiles whose units a softmax warp has read
        self.named = {}

    def copy(self):
        place, parity = 0, 1
        for i in range(sum(self.pieces)):
            while not self.raw_empty[place].passed(parity):
                yield True
            self.copies.append(i)
            place += 1
            if place == self.ring:
                place, parity = 0, parity ^ 1
            yield False

    def matrix(self):
        def score(i):
            while not self.k_full[i & 1].passed((i >> 1) & 1):
                yield True
            while i >= 2 and not self.o_full[i & 1].passed(((i >> 1) - 1) & 1):
                yield True
            assert i < 2 or self.outputs >= i - 1, "S takes the place of weights that are still read"
            self.products.append(("S", [self.k_empty[i % self.depth], self.s_full[i & 1]]))

        def output(i):
            while not self.v_full[i & 1].passed((i >> 1) & 1):
                yield True
            while not self.p_full[i & 1].passed((i >> 1) & 1):
                yield True
            assert min(self.read) > i, "weights of a tile that are not there"
            self.products.append(("O", [self.v_empty[i % self.depth], self.o_full[i & 1]]))

        i = 0
        for queries, n in enumerate(self.pieces):
            while not self.q_full.passed(queries & 1):
                yield True
            yield from score(i)
            for t in range(n):
                if t + 1 < n:
                    yield from score(i + 1)
                yield from output(i)
                i += 1
                yield False

    def convert(self, w):
        for at in range(w, sum(self.pieces) * BLOCKS, CONV):
            i = at // BLOCKS
            while not self.raw_full[i & 3].passed((i >> 2) & 1):
                yield True
            assert i in self.landed, "a tile that has not landed"
            assert i < self.units or min(self.read) > i - self.units, "units that a softmax still reads"
            yield False
            while i >= 2 and not self.k_empty[(i - 2) % self.depth].passed((i - 2) // self.depth & 1):
                yield True
            assert i < 2 or self.scores >= i - 1, "K's image is still read"
            yield False
            self.k_full[i & 1].arrive()
            while i >= 2 and not self.v_empty[(i - 2) % self.depth].passed((i - 2) // self.depth & 1):
                yield True
            assert i < 2 or self.outputs >= i - 1, "V's image is still read"
            yield False
            self.raw_empty[i % self.ring].arrive()
            self.v_full[i & 1].arrive()

    def together(self, key):   # the four warps of the same slots
        self.named[key] = self.named.get(key, 0) + 1
        while self.named[key] < 4:
            yield True

    def softmax(self, w):
        quarter, i = w & 3, 0
        for piece, n in enumerate(self.pieces):
            busy = quarter < random.Random(self.seed * 77 + piece).randint(1, 4)
            yield from self.together(("query", piece, quarter))
            assert self.outputs + sum(k == "O" for k, _ in self.products) >= i and self.scores >= i, "queries that are still read"
            self.q_full.arrive()
            yield False
            for t in range(n):
                while not self.s_full[i & 1].passed((i >> 1) & 1):
                    yield True
                assert self.scores > i, "scores that are not there"
                yield False
                if busy:
                    moves = t == 0 or random.Random(self.seed * 1000003 + i * 4 + quarter).random() < 0.3
                    for turn in range(4 if moves else 1):
                        yield from self.together(("reference", turn, i, quarter))
                    if moves and t > 0:
                        while not self.o_full[~i & 1].passed(((i - 1) >> 1) & 1):
                            yield True
                        assert self.outputs == i and not any(k == "O" for k, _ in self.products), "O is written while it is scaled"
                yield False
                i += 1
                self.read[w] = i
                self.p_full[~i & 1].arrive()
            while not self.o_full[(i - 1) & 1].passed(((i - 1) >> 1) & 1):
                yield True
            assert self.outputs >= i, "a record of an O that is not whole"
            yield from self.together(("record", piece, quarter))

    def run(self):
        rng = self.rng
        live = {"copy": self.copy(), "matrix": self.matrix()}
        live |= {("convert", w): self.convert(w) for w in range(CONV)} | {("softmax", w): self.softmax(w) for w in range(SOFT)}
        pace, idle = {}, 0
        while live:
            if rng.random() < 0.0005:
                pace.clear()
            names = list(live)
            for x in names:
                pace.setdefault(x, rng.choice([0.02, 0.3, 1, 1]))
            name = rng.choices(names, [pace[x] for x in names])[0]
            if self.copies and rng.random() < 0.3:
                i = self.copies.pop(rng.randrange(len(self.copies)))
                self.landed.add(i)
                self.raw_full[i & 3].arrive()
                idle = 0
            if self.products and rng.random() < 0.1:
                kind, bars = self.products.pop(0)
                if kind == "S":
                    self.scores += 1
                else:
                    self.outputs += 1
                for b in bars:
                    b.arrive()
                idle = 0
            try:
                idle = idle + 1 if next(live[name]) else 0
            except StopIteration:
                del live[name]
                idle = 0
            assert idle < 100000 or self.copies or self.products, f"all wait: {list(live)}"


def pieces_of(seed):
    rng = random.Random(seed)
    return [rng.randint(1, 20) for _ in range(3)]


@pytest.mark.parametrize("ring", range(2, MAX_RAW + 1))
@pytest.mark.parametrize("seed", range(3))
def test_every_wait_means_its_phase(ring, seed):
    Play(pieces_of(seed), ring, MAX_RAW + 2, seed).run()


@pytest.mark.parametrize("change", [dict(units=MAX_RAW + 1), dict(depth=2)])
def test_too_few_are_noticed(change):
    """What is played can fail: a unit less than the source keeps, and two barriers in turn for the images."""
    for seed in range(30):
        try:
            Play(**{**dict(pieces=[12, 12], ring=MAX_RAW, units=MAX_RAW + 2, seed=seed), **change}).run()
        except AssertionError:
            return
    raise AssertionError("not noticed")
