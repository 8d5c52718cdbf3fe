"""Attention over shared pages against a 64-bit reference that reads every row's own pages.

Tolerance of an output y = gate * sum(p v), from the roundings that a kernel may make: weights
rounded to bf16 (2^-9 of each, so 2^-9 * A in the sum, A = gate * sum(p |v|)), the same roundings
in the normaliser (2^-9 |y|), the output's own (2^-9 |y|), and 32-bit arithmetic (1e-4 A)."""

import math

import pytest
import torch

from zstep_b200.ops import mx
from zstep_b200.ops.kv_layout import swizzle_pages
from zstep_b200.ops.shared_prefix import SharedPrefixPlan

gpu = pytest.mark.gpu
PAGE, D = 16, 256


def _pages(n):
    return -(-n // PAGE)


class Batch:
    """Sequences (prefix pages from a shared list, own tokens) with rows; caches of random values
    whose rows behind every sequence's end, and whose unused pages, hold `poison`."""

    def __init__(self, hq, hkv, prefixes, seqs, seed=0, poison=float("nan"), scale=1.0):
        """prefixes: pages of each shared prefix; seqs: (prefix or None, total tokens, row lengths)."""
        g = torch.Generator().manual_seed(seed)
        self.hq, self.hkv = hq, hkv
        need = sum(prefixes) + sum(_pages(n) - (prefixes[p] if p is not None else 0) for p, n, _ in seqs)
        ids = (torch.randperm(need + 3, generator=g) + 1).tolist()
        shared = [[ids.pop() for _ in range(k)] for k in prefixes]
        total = need + 4
        self.k = torch.full((total, hkv, PAGE, D), poison)
        self.v = torch.full((total, hkv, PAGE, D), poison)
        width = max(_pages(n) for _, n, _ in seqs) + 2
        self.table = torch.zeros(len(seqs), width, dtype=torch.int32)
        self.slots, self.lens, self.rows_of, filled = [], [], {}, set()
        for s, (p, n, rows) in enumerate(seqs):
            have = shared[p] if p is not None else []
            pages = have + [ids.pop() for _ in range(_pages(n) - len(have))]
            self.table[s, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
            for j, pg in enumerate(pages):
                m = min(PAGE, n - j * PAGE)
                if pg not in filled:
                    filled.add(pg)
                    self.k[pg, :, :m] = torch.randn(hkv, m, D, generator=g) * scale
                    self.v[pg, :, :m] = torch.randn(hkv, m, D, generator=g)
            for x in rows:
                self.rows_of.setdefault(p, []).append(len(self.lens))
                self.slots.append(s)
                self.lens.append(x)
        self.k, self.v = self.k.to(torch.bfloat16), self.v.to(torch.bfloat16)
        rows = len(self.lens)
        self.q = torch.randn(rows, hq, D, generator=g).to(torch.bfloat16)
        self.gate = torch.randn(rows, hq, D, generator=g).to(torch.bfloat16)
        self.prefixes = [(self.rows_of[p], k) for p, k in enumerate(prefixes) if p in self.rows_of]

    def plan(self):
        return SharedPrefixPlan.from_prefixes(self.slots, self.prefixes, self.hq, self.hkv)

    def device(self):
        return dict(q=self.q.cuda(), gate=self.gate.cuda(), k_cache=swizzle_pages(self.k).cuda(),
                    v_cache=swizzle_pages(self.v).cuda(), page_table=self.table.cuda(),
                    seq_lens=torch.tensor(self.lens, dtype=torch.int32).cuda())

    def want(self, gated=True, sm=1 / 16):
        """(outputs, A) in 64 bits."""
        rows, group = len(self.lens), self.hq // self.hkv
        out = torch.zeros(rows, self.hq, D, dtype=torch.float64)
        mag = torch.zeros_like(out)
        for r, (s, n) in enumerate(zip(self.slots, self.lens)):
            if n == 0:
                continue
            pg = self.table[s, :_pages(n)].long()
            k = self.k[pg].double().permute(1, 0, 2, 3).reshape(self.hkv, -1, D)[:, :n]
            v = self.v[pg].double().permute(1, 0, 2, 3).reshape(self.hkv, -1, D)[:, :n]
            p = torch.softmax(torch.bmm(self.q[r].double().view(self.hkv, group, D), k.transpose(1, 2)) * sm, -1)
            out[r], mag[r] = torch.bmm(p, v).view(self.hq, D), torch.bmm(p, v.abs()).view(self.hq, D)
        gate = torch.sigmoid(self.gate.double()) if gated else 1.0
        return (out * gate).view(rows, -1), (mag * gate).view(rows, -1)


def run(b, plan=None, gate=True, sm=1 / 16, **kw):
    d = b.device()
    plan = plan or b.plan()
    plan.update(d["seq_lens"])
    out = plan.attend(d["q"], d["gate"] if gate else None, d["k_cache"], d["v_cache"], d["page_table"], d["seq_lens"], sm, **kw)
    torch.cuda.synchronize()
    plan.check()
    return out


def near(out, want):
    y, a = want
    tol = 2.0 ** -9 * (a + 2 * y.abs()) + 1e-4 * a + 1e-30
    bad = (out.cpu().double() - y).abs() > tol
    worst = ((out.cpu().double() - y).abs() / tol).max()
    assert not bad.any(), f"{int(bad.sum())} values off, worst {float(worst):.2f} of the tolerance"
    assert torch.isfinite(out).all()


def seq(prefix, base, own, rows=1):
    """A sequence of `base` shared tokens and `own` more, whose last `rows` tokens are its rows."""
    n = base + own
    return prefix, n, [n - rows + 1 + j for j in range(rows)]


CASES = {
    "one_token": (16, 2, [], [seq(None, 0, 1)]),
    "one_row_short": (16, 2, [], [seq(None, 0, 15)]),
    "two_samples": (16, 2, [3], [seq(0, 48, 1), seq(0, 48, 17)]),
    "ends": (8, 1, [4], [seq(0, 64, n) for n in (1, 15, 16, 17, 63, 64, 65, 128, 129)]),
    "odd_groups": (16, 2, [1, 7, 12], [seq(i % 3, [16, 112, 192][i % 3], 1 + 13 * i) for i in range(11)]),
    "mixed_with_unshared": (16, 2, [5], [seq(0, 80, 3), seq(None, 0, 100), seq(0, 80, 40), seq(None, 0, 1)]),
    "verify_rows": (16, 2, [6, 9], [seq(i % 2, [96, 144][i % 2], 4 + 7 * i, 4) for i in range(9)]),
    "many_rows": (16, 2, [10], [seq(0, 160, 1 + (5 * i) % 37) for i in range(70)]),
    "one_head_each": (2, 2, [4], [seq(0, 64, 9 + i) for i in range(5)]),
    "group_2": (2, 1, [40], [seq(0, 640, 3 + i) for i in range(67)]),
    "group_3": (6, 2, [5], [seq(0, 80, 1 + i) for i in range(7)]),
    "group_16": (16, 1, [8], [seq(0, 128, 30 + i) for i in range(9)]),
    "group_64": (64, 1, [8], [seq(0, 128, 5 + i) for i in range(5)]),
    "long": (16, 2, [300], [seq(0, 4800, 1 + 50 * i) for i in range(6)]),
    "more_units_than_sms": (16, 2, [9, 30], [seq(i % 2, [144, 480][i % 2], 1 + (37 * i) % 230) for i in range(150)]),
    "many_fragments_of_128_slots": (16, 2, [30] * 24, [seq(i % 24, 480, 1 + (7 * i) % 90, 1 + i % 3) for i in range(250)]),
    "long_alone": (16, 2, [], [seq(None, 0, 5000)]),
}


@gpu
@pytest.mark.parametrize("name", CASES)
def test_matches_64_bits(name):
    hq, hkv, prefixes, seqs = CASES[name]
    b = Batch(hq, hkv, prefixes, seqs, seed=len(name))
    near(run(b), b.want())


@gpu
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), float("-inf"), -3.0e38])
def test_values_behind_the_mask_do_not_count(poison):
    """Rows of the last page behind a sequence's end, and pages that no row sees."""
    b = Batch(16, 2, [3], [seq(0, 48, 5), seq(0, 48, 16), seq(0, 48, 29, 2)], seed=4, poison=poison)
    near(run(b), b.want())


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_value_that_only_another_row_sees_does_not_count(bad):
    """Draft rows: the last row's own token is not finite, the rows before it do not see it."""
    b = Batch(16, 2, [3], [seq(0, 48, 21, 4), seq(0, 48, 8, 1)], seed=5)
    for x in (b.k, b.v):
        x[b.table[0, 68 // PAGE], :, 68 % PAGE] = bad
    out = run(b).cpu().double()
    y, a = b.want()
    seen = [r for r, n in enumerate(b.lens) if not (b.slots[r] == 0 and n == 69)]
    tol = 2.0 ** -9 * (a + 2 * y.abs()) + 1e-4 * a
    assert ((out - y).abs() <= tol)[seen].all()
    assert not torch.isfinite(out[[r for r in range(len(b.lens)) if r not in seen]]).all()


@gpu
@pytest.mark.parametrize("hq,hkv,pages,seqs", [
    (16, 2, 128, [seq(0, 2048, 20 + 19 * i) for i in range(20)]),
    (16, 2, 60, [seq(0, 960, 5 + 11 * i, 4) for i in range(9)]),
    (2, 1, 100, [seq(0, 1600, 7 + 31 * i) for i in range(12)]),
    (8, 1, 400, [seq(0, 6400, 300), seq(0, 6400, 1)]),
    (16, 2, 1600, [seq(0, 25600, 1 + 5 * i) for i in range(32)]),    # many tiles one after the other in a CTA
    (64, 1, 800, [seq(0, 12800, 1 + 9 * i) for i in range(24)]),
])
def test_no_more_is_lost_than_the_rounding_of_the_outputs(hq, hkv, pages, seqs):
    """Rounding to bf16 moves an output by at most 2^-9 of itself and, over outputs of every mantissa, by 0.85 of
    that in the norm, so 2^-9 of the norm leaves half as much again for all that comes before it: scores in 32 bits
    (2^-20 of a weight) are far below, weights rounded to bf16 (0.85 * 2^-9 of each, which keyed values of either
    sign pass on to the output unaveraged: 1.2 * 2^-9 in all) are above."""
    b = Batch(hq, hkv, [pages], seqs, seed=20)
    y, _ = b.want()
    assert (run(b).cpu().double() - y).norm() <= 2.0 ** -9 * y.norm()


def near_where_finite(out, want):
    y, a = want
    out = out.cpu().double()
    assert torch.equal(out.isnan(), y.isnan())
    tol = 2.0 ** -9 * (a + 2 * y.abs()) + 1e-4 * a + 1e-30
    assert ((out - y).abs() <= tol)[~y.isnan()].all()


@gpu
@pytest.mark.parametrize("prefix", [3, 200])
def test_scores_that_are_all_nan_are_not_taken_for_no_keys(prefix):
    """A query row of NaN; a NaN key that is the only one of its record, beside records of finite ones."""
    n = prefix * PAGE
    b = Batch(16, 2, [prefix], [seq(0, n, 5), seq(0, n, 1), seq(0, n, 40), (0, n + 7, [0, n + 7])], seed=18)
    b.q[2] = float("nan")
    b.q[0, 3] = float("nan")
    b.k[b.table[1, prefix], 1, 0] = float("nan")
    y, a = b.want()
    nan = y.view(5, 16, D).isnan().all(-1)
    assert nan[0].tolist() == [h == 3 for h in range(16)] and nan[1].tolist() == [h >= 8 for h in range(16)]
    assert nan[2].all() and not nan[3:].any()
    near_where_finite(run(b), (y, a))


@gpu
@pytest.mark.parametrize("keys", [(5,), (40, 200), (527,), (900, 1033)])
def test_infinite_values_that_rows_see_stay_infinite(keys):
    """In the prefix's first tiles, in later ones, and among own tokens that not every row sees."""
    b = Batch(16, 2, [64], [seq(0, 1024, 30, 4), seq(0, 1024, 9), seq(0, 1024, 70)], seed=21)
    for i, t in enumerate(keys):
        b.v[b.table[0, t // PAGE], :, t % PAGE, 10 + i] = float("inf")
        b.v[b.table[0, t // PAGE], 1, t % PAGE, 20 + i] = float("-inf")
    y, a = b.want()
    y, n = y.view(-1, 16, D), len(keys)
    assert y[3, :, 10:10 + n].isinf().all() and y[3, 8:, 20:20 + n].isinf().all()
    assert not y.isnan().any()
    out = run(b).cpu().double().view_as(y)
    inf = y.isinf()
    assert torch.equal(out[inf], y[inf])
    tol = (2.0 ** -9 * (a.view_as(y) + 2 * y.abs()) + 1e-4 * a.view_as(y) + 1e-30)
    assert ((out - y).abs() <= tol)[~inf].all()


@gpu
def test_scores_that_are_all_minus_infinity():
    """Keys that a row sees, all with a score of -inf, are no empty mask: 0 / 0.  Beside finite ones they weigh nothing."""
    b = Batch(16, 2, [2], [(None, 33, [33]), (0, 40, [0, 40])], seed=19)
    b.q[:, :, 0] = 1.0
    for t in range(33):
        b.k[b.table[0, t // PAGE], 0, t % PAGE, 0] = float("-inf")
    b.k[b.table[1, 2], :, 3, 0] = float("-inf")
    y, a = b.want()
    assert y.view(3, 16, D)[0, :8].isnan().all() and not y.view(3, 16, D)[0, 8:].isnan().any() and not y[1:].isnan().any()
    out = run(b)
    near_where_finite(out, (y, a))
    assert not out[1].any()


@gpu
def test_rows_without_keys_and_rows_inside_the_prefix():
    """Length 0 gives 0; a row shorter than its group's prefix sees that much of it."""
    b = Batch(16, 2, [6], [(0, 130, [0, 1, 16, 40, 95, 96, 97, 130]), (0, 100, [100])], seed=6)
    out = run(b)
    near(out, b.want())
    assert not out[0].any()
    z = Batch(16, 2, [2], [(0, 40, [0]), (0, 33, [0])], seed=7)
    assert not run(z).any()


@gpu
def test_short_tables_behind_the_prefix():
    """A padding row in a group (length 1, table entries behind its page never set) reads its own page only."""
    b = Batch(16, 2, [9], [seq(0, 144, 4), seq(0, 144, 40)], seed=8)
    b.table = torch.cat([b.table, torch.zeros_like(b.table[:1])])
    b.table[2, 0] = b.table[0, 0]
    b.slots.append(2)
    b.lens.append(1)
    b.q, b.gate = torch.cat([b.q, b.q[:1]]), torch.cat([b.gate, b.gate[:1]])
    b.prefixes = [([2, 0, 1], 9)]
    near(run(b), b.want())


@gpu
def test_tree_of_prefixes():
    """Three levels: a prompt that all rows share, branches, and sequences."""
    b = Batch(16, 2, [11], [seq(0, 176, 70 + 3 * i) for i in range(6)], seed=9)
    for s in (1, 2):
        b.table[s, 11:13] = b.table[0, 11:13]   # sequences 0..2 also share pages 11 and 12
    for s in (4, 5):
        b.table[s, 11:14] = b.table[3, 11:14]
    segments = [(list(range(6)), 0, 11), ([0, 1, 2], 11, 13), ([3, 4, 5], 11, 14)]
    segments += [([s], 13 if s < 3 else 14, None) for s in range(6)]
    near(run(b, SharedPrefixPlan(b.slots, segments, 16, 2)), b.want())


@gpu
def test_without_gate_and_other_scales():
    b = Batch(16, 2, [4], [seq(0, 64, 20 + i) for i in range(4)], seed=10, scale=3.0)
    near(run(b, gate=False), b.want(gated=False))
    near(run(b, sm=0.31), b.want(sm=0.31))


@gpu
def test_scores_that_grow_along_the_keys():
    """Later keys score ever higher (the running maximum moves all the time), then lower."""
    for sign in (1.0, -1.0):
        b = Batch(16, 2, [20], [seq(0, 320, 200), seq(0, 320, 77)], seed=11)
        u = torch.randn(D, generator=torch.Generator().manual_seed(1))
        b.q = (b.q.float() * 0.1 + u).to(torch.bfloat16)
        for s, n in ((0, 520), (1, 397)):
            for t in range(n):
                b.k[b.table[s, t // PAGE], :, t % PAGE] = (u * (sign * t / 40)).to(torch.bfloat16)
        near(run(b), b.want())


@gpu
def test_mxfp8_output():
    b = Batch(16, 2, [4], [seq(0, 64, 3 + i) for i in range(5)], seed=12)
    rows, width = len(b.lens), 16 * D
    q = torch.zeros(128, width, dtype=torch.uint8, device="cuda")
    sf = torch.zeros(mx.atoms_bytes(128, width), dtype=torch.uint8, device="cuda")
    out = torch.empty(rows, width, dtype=torch.bfloat16, device="cuda")
    run(b, out=out, out_q=q, out_sf=sf)
    got = mx.dequantize(q[:rows].cpu(), mx.codes_from_atoms(sf.cpu(), rows, width)).double()
    y = out.cpu().double()
    amax = y.abs().view(rows, -1, 32).amax(-1, keepdim=True).expand(-1, -1, 32).reshape(rows, width)
    # e4m3 has 3 mantissa bits (2^-4 of a value), its smallest step is 2^-9 of a scale that is at
    # most 2 * amax / 448; `out` itself is rounded by 2^-9.
    assert ((got - y).abs() <= (2.0 ** -4 + 2.0 ** -8) * y.abs() + amax * 2 / 448 * 2.0 ** -10).all()


@gpu
def test_growing_lengths_streams_and_graphs():
    """One plan while its sequences grow: on a stream of its own, and replayed from a CUDA graph."""
    b = Batch(16, 2, [8], [seq(0, 128, 300) for _ in range(5)], seed=13)
    plan, d = b.plan(), b.device()
    lens = torch.zeros(5, dtype=torch.int32, device="cuda")
    out = torch.empty(5, 16 * D, dtype=torch.bfloat16, device="cuda")
    args = (d["q"], d["gate"], d["k_cache"], d["v_cache"], d["page_table"], lens, 1 / 16)

    def step():
        plan.update(lens)
        plan.attend(*args, out=out)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    s.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    for k in (1, 100, 160, 299):
        b.lens = [128 + k, 128, 130 + k // 2, 17, 0]
        lens.copy_(torch.tensor(b.lens, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        plan.check()
        near(out, b.want())


@gpu
def test_two_calls_give_the_same_bits():
    b = Batch(16, 2, [30], [seq(0, 480, 1 + 31 * i) for i in range(12)], seed=14)
    plan = b.plan()
    assert torch.equal(run(b, plan), run(b, plan))


@gpu
def test_many_pieces_of_one_tile():
    """Hundreds of sequences within one tile: every warp gets a new piece with every tile."""
    b = Batch(16, 2, [], [seq(None, 0, 1 + (7 * i) % 64) for i in range(700)], seed=17)
    plan, d = b.plan(), b.device()
    out = run(b, plan)
    near(out, b.want())
    again = torch.empty_like(out)
    for _ in range(50):
        plan.update(d["seq_lens"])
        plan.attend(d["q"], d["gate"], d["k_cache"], d["v_cache"], d["page_table"], d["seq_lens"], 1 / 16, out=again)
        assert torch.equal(out, again)
    plan.check()


@gpu
def test_page_beyond_four_gigabytes_of_elements():
    """A page whose element offset passes 2^32 (and byte offset 2^33)."""
    hq, hkv = 2, 1
    pages = (1 << 32) // (PAGE * D) + 5
    b = Batch(hq, hkv, [2], [seq(0, 32, 9), seq(0, 32, 20)], seed=15)
    small = b.device()
    k = torch.empty(pages, hkv, PAGE, D, dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    n = b.k.shape[0]
    k[pages - n:], v[pages - n:] = small["k_cache"], small["v_cache"]
    plan = b.plan()
    plan.update(small["seq_lens"])
    table = small["page_table"] + (pages - n)
    out = plan.attend(small["q"], small["gate"], k, v, table, small["seq_lens"], 1 / 16)
    plan.check()
    near(out, b.want())


@gpu
def test_bad_pages_and_arguments_are_reported():
    b = Batch(16, 2, [2], [seq(0, 32, 9), seq(0, 32, 20)], seed=16)
    d, plan = b.device(), b.plan()
    args = dict(gate=d["gate"], k_cache=d["k_cache"], v_cache=d["v_cache"], page_table=d["page_table"],
                seq_lens=d["seq_lens"], sm_scale=1 / 16)
    for wrong in (dict(q=d["q"][:, :8].contiguous()), dict(q=d["q"].float()), dict(q=d["q"].transpose(0, 1)),
                  dict(gate=d["gate"][:1].contiguous()), dict(k_cache=d["k_cache"][:, :1].contiguous()), dict(v_cache=d["v_cache"][:3]),
                  dict(page_table=d["page_table"][:1]), dict(page_table=d["page_table"].long()),
                  dict(seq_lens=d["seq_lens"].long()), dict(seq_lens=d["seq_lens"][:1]),
                  dict(out=torch.empty(1, 8, dtype=torch.bfloat16, device="cuda")),
                  dict(out_q=torch.empty(2, 16 * D, dtype=torch.uint8, device="cuda"))):
        with pytest.raises((ValueError, RuntimeError)):
            plan.attend(**{**args, "q": d["q"], **wrong})
    for page in (-1, b.k.shape[0]):   # the kernel checks page ids itself
        table = d["page_table"].clone()
        table[1, 2] = page
        plan.update(d["seq_lens"])
        plan.attend(d["q"], **{**args, "page_table": table})
        with pytest.raises(RuntimeError):
            plan.check()
    plan.update(d["seq_lens"])
    plan.attend(d["q"], **args)
    plan.check()


@pytest.mark.parametrize("slots,segments,hq,hkv,what", [
    ([0, 1], [([0, 1], 0, 2), ([0], 2, None)], 16, 2, "end at None"),
    ([0, 1], [([0, 1], 0, 2), ([0, 1], 3, None)], 16, 2, "follow"),
    ([0], [([0], 1, None)], 16, 2, "follow"),
    ([0], [([0], 0, None), ([0], 0, None)], 16, 2, "follow"),
    ([0], [([0, 1], 0, None)], 16, 2, "outside"),
    ([0], [([0], 0, 0), ([0], 0, None)], 16, 2, "empty"),
    ([0], [([], 0, 3), ([0], 0, None)], 16, 2, "needs rows"),
    ([-1], [([0], 0, None)], 16, 2, "negative"),
    ([0], [([0], 0, None)], 15, 2, "q heads"),
    ([0], [([0], 0, None)], 130, 2, "q heads"),
])
def test_plans_that_are_refused(slots, segments, hq, hkv, what):
    with pytest.raises(ValueError, match=what):
        SharedPrefixPlan(slots, segments, hq, hkv, device="cpu")


def test_a_row_in_two_groups_is_refused():
    with pytest.raises(ValueError, match="two groups"):
        SharedPrefixPlan.from_prefixes([0, 1], [([0, 1], 2), ([1], 3)], 16, 2, device="cpu")
