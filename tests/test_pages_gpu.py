"""The page pool against a sequential model of it: tables, counts, lengths and page data are
compared exactly after every call."""

import random

import pytest
import torch

from zstep_b200.ops.pages import PagePool

pytestmark = pytest.mark.gpu
PAGE = 16


class Model:
    """One request after the other, in Python."""

    def __init__(self, pages, slots, width, caches):
        self.ref = [1] + [0] * (pages - 1)
        self.len = [0] * slots
        self.table = [[0] * width for _ in range(slots)]
        self.caches = [c.clone() for c in caches]

    def fresh(self):
        p = self.ref.index(0)
        self.ref[p] = 1
        return p

    def copy(self, moves):
        for s, d in moves:
            for c in self.caches:
                c[:, d] = c[:, s]

    def fork(self, parents, children, share):
        moves = []
        for p, c, s in zip(parents, children, share):
            self.len[c] = self.len[p]
            for j in range(-(-self.len[p] // PAGE)):
                src = self.table[p][j]
                if (j + 1) * PAGE <= min(s, self.len[p]):
                    self.table[c][j] = src
                    self.ref[src] += 1
                else:
                    self.table[c][j] = self.fresh()
                    moves.append((src, self.table[c][j]))
        self.copy(moves)

    def extend(self, slots, lens):
        moves, left, grow = [], [], []
        for s, n in zip(slots, lens):   # what is copied is decided before anything changes
            grow.append(n > self.len[s] and self.len[s] % PAGE and self.ref[self.table[s][self.len[s] // PAGE]] > 1)
        for s, n, cow in zip(slots, lens, grow):
            if n <= self.len[s]:
                continue
            if cow:
                j = self.len[s] // PAGE
                left.append(self.table[s][j])
                self.table[s][j] = self.fresh()
                moves.append((left[-1], self.table[s][j]))
            for j in range(-(-self.len[s] // PAGE), -(-n // PAGE)):
                self.table[s][j] = self.fresh()
            self.len[s] = n
        for p in left:
            self.ref[p] -= 1
        self.copy(moves)

    def truncate(self, slots, lens):
        for s, n in zip(slots, lens):
            for j in range(-(-n // PAGE), -(-self.len[s] // PAGE)):
                self.ref[self.table[s][j]] -= 1
                self.table[s][j] = 0
            self.len[s] = min(n, self.len[s])

    def compact(self):
        live = [p for p, r in enumerate(self.ref) if r]
        moves = list(zip([p for p in live if p >= len(live)], [p for p in range(len(live)) if not self.ref[p]]))
        self.copy(moves)
        to = dict(moves)
        self.table = [[to.get(p, p) for p in row] for row in self.table]
        for s, d in moves:
            self.ref[d], self.ref[s] = self.ref[s], 0


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make(pages, slots, width, shapes=((2, 1, PAGE, 256), (2, 1, PAGE, 256)), dtype=torch.bfloat16, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    caches = [torch.randint(-100, 100, (s[0], pages, *s[1:]), generator=g, device="cuda").to(dtype) for s in shapes]
    model = Model(pages, slots, width, caches)
    return PagePool(caches, slots, width, PAGE), model


def same(pool, m):
    torch.cuda.synchronize()
    assert pool.refcount.tolist() == m.ref
    assert pool.seq_len.tolist() == m.len
    assert pool.page_table.tolist() == m.table
    free = [(int(pool.free_bits[p // 32]) >> (p % 32)) & 1 for p in range(len(m.ref))]
    assert free == [int(r == 0) for r in m.ref]
    assert not int(pool.free_bits[-1]) >> ((len(m.ref) - 1) % 32 + 1) or len(m.ref) % 32 == 0
    for a, b in zip(pool.caches, m.caches):
        assert torch.equal(a, b)


def both(pool, m, name, *args):
    getattr(pool, name)(*(ints(a) for a in args))
    if name == "free":
        m.truncate(args[0], [0] * len(args[0]))
    else:
        getattr(m, name)(*args)
    pool.check()
    same(pool, m)


@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 32, 100])
def test_fork_extend_truncate_at_page_ends(length):
    pool, m = make(80, 8, 12)
    if length:
        both(pool, m, "extend", [3], [length])
    both(pool, m, "fork", [3, 3, 3], [0, 7, 5], [length, length // 2, 0])
    both(pool, m, "extend", [0, 3, 5], [length + 1, length + 16, length + 17])
    both(pool, m, "truncate", [0, 7], [max(0, length - 1), length // 3])
    both(pool, m, "free", [3, 5])
    both(pool, m, "compact")


def test_copy_on_write_of_a_page_that_others_still_use():
    """A cut sequence ends inside a shared page: growing it copies that page first."""
    pool, m = make(40, 4, 8)
    both(pool, m, "extend", [0], [60])
    both(pool, m, "fork", [0, 0], [1, 2], [60, 60])
    both(pool, m, "truncate", [1, 2], [20, 40])
    both(pool, m, "extend", [1, 2], [25, 41])
    both(pool, m, "extend", [0], [61])
    # two slots with one partly filled page that is theirs alone: each copies, the page is free then
    both(pool, m, "free", [0])
    both(pool, m, "fork", [1], [3], [16])
    both(pool, m, "truncate", [1, 3], [9, 9])
    both(pool, m, "extend", [1, 3], [10, 17])


@pytest.mark.parametrize("seed,pages,slots,width,shapes,dtype", [
    (1, 64, 9, 7, ((2, 1, PAGE, 256), (2, 1, PAGE, 256)), torch.bfloat16),
    (2, 257, 40, 11, ((3, 2, PAGE, 256), (1, PAGE, 24)), torch.bfloat16),      # page sizes that end inside a copy piece
    (3, 2000, 70, 40, ((1, 8),), torch.float32),
    (4, 33, 5, 9, ((2, 5, 16),) * 8, torch.uint8),
])
def test_random_lives(seed, pages, slots, width, shapes, dtype):
    r = random.Random(seed)
    pool, m = make(pages, slots, width, shapes, dtype, seed)
    for _ in range(60):
        full = [s for s in range(slots) if m.len[s]]
        empty = [s for s in range(slots) if not m.len[s]]
        room = m.ref.count(0)
        op = r.choice(["fork", "extend", "extend", "truncate", "free", "compact"])
        if op == "fork" and full and empty:
            k = min(len(empty), r.randint(1, 6))
            parents = [r.choice(full) for _ in range(k)]
            share = [r.randint(0, width * PAGE) for _ in range(k)]
            if sum(-(-m.len[p] // PAGE) for p in parents) <= room:
                both(pool, m, "fork", parents, r.sample(empty, k), share)
        elif op == "extend":
            pick = r.sample(range(slots), r.randint(1, slots))
            lens = [min(width * PAGE, m.len[s] + r.randint(0, 40)) for s in pick]
            if sum(-(-n // PAGE) - m.len[s] // PAGE for s, n in zip(pick, lens)) <= room:
                both(pool, m, "extend", pick, lens)
        elif op == "truncate":
            pick = r.sample(range(slots), r.randint(1, slots))
            both(pool, m, "truncate", pick, [r.randint(0, m.len[s] + 3) for s in pick])
        elif op == "free" and full:
            both(pool, m, "free", r.sample(full, r.randint(1, (len(full) + 1) // 2)))
        elif op == "compact":
            both(pool, m, "compact")


def test_more_requests_than_threads():
    """3000 slots: several rounds of the planning block."""
    slots = 3000
    pool, m = make(9000, slots, 3, ((1, 16),), torch.float32)
    both(pool, m, "extend", list(range(1400)), [1 + i % 48 for i in range(1400)])
    both(pool, m, "fork", list(range(1400)), list(range(1500, 2900)), [48 if i % 3 else 16 for i in range(1400)])
    both(pool, m, "free", list(range(0, 1400, 2)))
    both(pool, m, "compact")


def test_too_few_pages_changes_nothing():
    pool, m = make(10, 6, 8)
    both(pool, m, "extend", [0], [100])
    for call in (lambda: pool.fork(ints([0, 0]), ints([1, 2]), ints([0, 96])), lambda: pool.extend(ints([3, 4]), ints([16, 48]))):
        call()
        with pytest.raises(RuntimeError, match="too few"):
            pool.check()
        same(pool, m)
    both(pool, m, "extend", [3], [32])   # exactly what is left
    assert m.ref.count(0) == 0


@pytest.mark.parametrize("call", [
    lambda p: p.fork(ints([0]), ints([0])),               # child not empty
    lambda p: p.fork(ints([0, 0]), ints([2, 2])),         # child twice
    lambda p: p.fork(ints([9]), ints([2])),
    lambda p: p.fork(ints([0]), ints([-1])),
    lambda p: p.fork(ints([0]), ints([2]), ints([-5])),
    lambda p: p.extend(ints([0, 0]), ints([50, 60])),     # slot twice
    lambda p: p.extend(ints([6]), ints([5])),
    lambda p: p.extend(ints([1]), ints([8 * PAGE + 1])),  # longer than a table row
    lambda p: p.extend(ints([1]), ints([-1])),
])
def test_bad_requests_change_nothing(call):
    pool, m = make(40, 6, 8)
    both(pool, m, "extend", [0], [40])
    call(pool)
    with pytest.raises(RuntimeError, match="cannot serve"):
        pool.check()
    same(pool, m)
    both(pool, m, "fork", [0], [2], [40])


def test_bad_truncate_and_copy_requests_are_reported():
    pool, m = make(40, 6, 8)
    both(pool, m, "extend", [0], [40])
    for call in (lambda: pool.free(ints([6])), lambda: pool.truncate(ints([0]), ints([-1])),
                 lambda: pool.copy(ints([1]), ints([40])), lambda: pool.copy(ints([-1]), ints([5]))):
        call()
        with pytest.raises(RuntimeError):
            pool.check()
        same(pool, m)


def test_a_slot_cut_twice_in_one_call_ends_at_the_shorter_length():
    pool, m = make(40, 6, 8)
    both(pool, m, "extend", [0, 1], [100, 50])
    pool.truncate(ints([0, 1, 0, 0]), ints([70, 50, 20, 90]))
    m.truncate([0], [20])
    pool.check()
    same(pool, m)


@pytest.mark.parametrize("huge", [2 ** 31 - 1, 2 ** 31 - PAGE, 2 ** 31 - PAGE + 1])
def test_lengths_whose_pages_pass_32_bits(huge):
    """A cut to more than a slot holds has no effect, however much more; growth to that is refused."""
    pool, m = make(40, 4, 8)
    both(pool, m, "extend", [1, 3], [100, 128])
    pool.truncate(ints([1, 3, 0]), ints([huge] * 3))
    pool.check()
    same(pool, m)
    pool.extend(ints([1]), ints([huge]))
    with pytest.raises(RuntimeError):
        pool.check()
    same(pool, m)
    both(pool, m, "fork", [1], [0], [huge])
    pool.check()
    same(pool, m)


def test_copy_and_adopt():
    pool, m = make(50, 4, 6, ((2, 1, PAGE, 256), (3, PAGE, 40)))
    table = [[7, 9, 0], [7, 30, 49], [0, 0, 0], [12, 0, 0]]
    pool.adopt(ints([20, 48, 0, 3]), ints(table))
    m.len, m.table = [20, 48, 0, 3], [t + [0] * 3 for t in table]
    for p in (7, 9, 7, 30, 49, 12):
        m.ref[p] += 1
    same(pool, m)
    pool.copy(ints([7, 0, 49, 12]), ints([1, 5, 2, 3]))
    m.copy([(7, 1), (49, 2), (12, 3)])
    pool.check()
    same(pool, m)
    both(pool, m, "compact")
    both(pool, m, "extend", [2], [33])
    for lens, t in (([20, 0, 0, 0], [[7, 50, 0]] + [[0] * 3] * 3), ([49, 0, 0, 0], [[1, 2, 3]] + [[0] * 3] * 3),
                    ([17, 0, 0, 0], [[1, 0, 0]] + [[0] * 3] * 3)):
        with pytest.raises(ValueError):
            pool.adopt(ints(lens), ints(t))


def test_calls_in_a_graph_and_on_another_stream():
    pool, m = make(60, 6, 8)
    both(pool, m, "extend", [0], [35])
    start = pool.state.clone()
    kids, lens, zero = ints([1, 2, 3]), ints([40, 41, 36]), ints([0, 0, 0])

    def step():
        pool.state.copy_(start)
        pool.fork(zero, kids)
        pool.extend(kids, lens)
        pool.truncate(kids, zero + 34)
        pool.compact()

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    s.synchronize()
    m.fork([0, 0, 0], [1, 2, 3], [35] * 3)
    m.extend([1, 2, 3], [40, 41, 36])
    m.truncate([1, 2, 3], [34] * 3)
    m.compact()
    same(pool, m)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    g.replay()
    g.replay()
    pool.check()
    same(pool, m)


def test_adopt_refuses_lengths_below_zero():
    """Such a slot could neither be filled nor cut nor freed."""
    pool, m = make(20, 3, 4)
    both(pool, m, "extend", [1], [20])
    with pytest.raises(ValueError, match="negative"):
        pool.adopt(ints([0, -1, 5]), ints([[0], [0], [3]]))
    same(pool, m)
    for call in (lambda: pool.free(None), lambda: pool.fork(None, None), lambda: pool.copy(ints([1]), None)):
        with pytest.raises(ValueError):   # not taken for a call without requests
            call()
    same(pool, m)


def test_large_caches():
    """Page offsets that pass 2^31 elements and 2^32 bytes."""
    pages = (1 << 32) // (PAGE * 256 * 2) + 70
    cache = torch.zeros(1, pages, 1, PAGE, 256, dtype=torch.bfloat16, device="cuda")
    pool = PagePool([cache], 3, 4, PAGE)
    pool.adopt(ints([20, 0, 0]), ints([[pages - 1, pages - 2, 0, 0], [0] * 4, [0] * 4]))
    cache[0, pages - 1], cache[0, pages - 2] = 3.0, 5.0
    pool.fork(ints([0]), ints([1]), ints([0]))
    pool.free(ints([0]))
    pool.compact()
    pool.check()
    assert pool.page_table[1, :2].tolist() == [1, 2] and pool.refcount[:4].tolist() == [1, 1, 1, 0]
    assert (cache[0, 1] == 3.0).all() and (cache[0, 2] == 5.0).all()


def test_refusals():
    c = torch.zeros(2, 10, 16, dtype=torch.float32, device="cuda")
    for caches, slots, width in (([], 2, 2), ([c, c[:, :5]], 2, 2), ([c], 0, 2), ([c], 2, 0), ([c[:, :1]], 2, 2)):
        with pytest.raises(ValueError):
            PagePool(caches, slots, width)
    pool = PagePool([c], 3, 4)
    for call in (lambda: pool.fork(ints([0]), None), lambda: pool.extend(ints([0]), None), lambda: pool.truncate(ints([0]), None),
                 lambda: pool.fork(ints([0, 1]), ints([2])), lambda: pool.free(ints([0]).long()), lambda: pool.free(torch.zeros(1, dtype=torch.int32)),
                 lambda: pool.extend(ints([0, 1, 2, 2]), ints([1, 1, 1, 1])), lambda: pool.free(ints([0, 1, 2, 2])[::2])):
        with pytest.raises((ValueError, RuntimeError)):
            call()
    odd = PagePool([torch.zeros(2, 10, 3, dtype=torch.float32, device="cuda")], 3, 4)
    with pytest.raises(RuntimeError, match="16 bytes"):
        odd.free(ints([0]))
    pool.fork(ints([]), ints([]))
    pool.free(ints([]))
    pool.check()
