"""How near the quantised attention is to the 64-bit result, and what a row may depend on: limits that a dropped key or a
score 2 % off do not pass (tests/test_quant_oracle.py), for every grouping of rows."""

import numpy as np
import pytest
import torch

from tests.quant_oracle import LIMIT, attention, distance, held
from zstep_b200.ops.quant_cache import QuantAttention, QuantCache

pytestmark = pytest.mark.gpu
DEV = "cuda"
FORMS = [(64, 4), (128, 4), (256, 4), (64, 8), (128, 8), (256, 8)]


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def keys_of(n, heads, dim, dtype, seed):
    """Keys and values whose channels have offsets and sizes of their own."""
    g = gen(seed)
    size = torch.exp(0.5 * torch.randn(heads, dim, generator=g, device=DEV))
    k = size * (torch.randn(n, heads, dim, generator=g, device=DEV) + torch.randn(heads, dim, generator=g, device=DEV))
    return k.to(dtype), (0.7 * torch.randn(n, heads, dim, generator=g, device=DEV)).to(dtype)


class Held:
    """Sequences of these keys and values in a cache, their pages in any order."""

    def __init__(self, ks, vs, bits, page=16):
        n = [len(k) for k in ks]
        need = [-(-x // page) for x in n]
        ids = torch.randperm(sum(need), generator=torch.Generator().manual_seed(1)) + 1
        table = torch.zeros(len(ks), max(need) + 1, dtype=torch.int32)
        for i, part in enumerate(ids.split(need)):
            table[i, :need[i]] = part
        self.table, self.ks, self.vs, self.bits = table.to(DEV), ks, vs, bits
        self.cache = QuantCache(1, sum(need) + 1, ks[0].shape[1], ks[0].shape[2], bits=bits, page_size=page)
        at = i32(np.repeat(np.arange(len(n)), n).tolist()), i32([p for x in n for p in range(x)])
        self.cache.write(0, torch.cat(ks), torch.cat(vs), self.table, *at)
        self.cache.check()

    def attend(self, q, counts, lens, scale, gate=None):
        """counts[s] rows of sequence s, each with its length; alone where counts is None (row r of sequence r)."""
        each = [1] * len(self.ks) if counts is None else counts
        slots = i32([s for s, c in enumerate(each) for _ in range(c)])
        starts = None if counts is None else i32([0] + list(np.cumsum(counts)))
        plan = QuantAttention(self.cache, q.shape[1], max_rows=len(q), max_seqs=len(each), max_seq_rows=max(each))
        plan.update(slots, i32(lens), starts)
        out = plan.attend(0, q, self.table, scale, gate=gate)
        plan.check()
        return out.view(q.shape)

    def exact(self, q, counts, lens, scale, gate=None):
        out, r = [], 0
        for s, c in enumerate([1] * len(self.ks) if counts is None else counts):
            part = slice(r, r + c)
            out.append(attention(q[part], held(self.ks[s], self.bits), held(self.vs[s], self.bits), lens[part], scale,
                                 None if gate is None else gate[part]))
            r += c
        return torch.cat(out)


# ------------------------------------------------------------------------------------ precision
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows", [1, 2, 5, 9, 40, 150])
@pytest.mark.parametrize("dim,bits", FORMS)
def test_precision_of_every_grouping(dim, bits, rows, dtype):
    """8 to 1200 query slots of a sequence, on all variants, with a gate: the rounding of the output's type decides."""
    seqs = [rows + 3, 301, 160]
    kv = [keys_of(n, 2, dim, dtype, 7 * i + dim) for i, n in enumerate(seqs)]
    c = Held([k for k, _ in kv], [v for _, v in kv], bits)
    counts = [rows, max(1, rows - 1), rows]
    lens = [n - m + 1 + i for n, m in zip(seqs, counts) for i in range(m)]
    lens[1::7] = [max(1, n - 60) for n in lens[1::7]]   # not all of them causal
    q = torch.randn(sum(counts), 16, dim, generator=gen(rows), device=DEV).to(dtype)
    gate = torch.randn(q.shape, generator=gen(rows + 1), device=DEV).to(dtype)
    got = c.attend(q, counts, lens, dim ** -0.5, gate)
    assert distance(got, c.exact(q, counts, lens, dim ** -0.5, gate)) < LIMIT


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,bits", FORMS)
def test_precision_of_mixed_steps(dim, bits, dtype):
    """Single tokens, sequences without rows or keys, verify rows and chunks in one step; the rest of the cache is poisoned."""
    seqs, counts = [1200, 40, 16, 333, 200, 1, 64], [1, 37, 0, 2, 130, 1, 1]
    kv = [keys_of(n, 2, dim, dtype, 11 * i + dim) for i, n in enumerate(seqs)]
    c = Held([k for k, _ in kv], [v for _, v in kv], bits, page=64)
    behind = [(s, p) for s, n in enumerate(seqs) for p in range(n, -(-n // 64) * 64)]
    nan = torch.full((len(behind), 2, dim), float("nan"), dtype=dtype, device=DEV)
    c.cache.write(0, nan, nan, c.table, i32([s for s, _ in behind]), i32([p for _, p in behind]))
    lens = [n - m + 1 + i for n, m in zip(seqs, counts) for i in range(m)]
    lens[-1] = 0
    q = torch.randn(sum(counts), 16, dim, generator=gen(dim), device=DEV).to(dtype)
    got, want = c.attend(q, counts, lens, dim ** -0.5), c.exact(q, counts, lens, dim ** -0.5)
    at = 0
    for m in counts[:-1]:
        assert m == 0 or distance(got[at:at + m], want[at:at + m]) < LIMIT
        at += m
    assert not got[-1].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("dim", [64, 128])
def test_precision_of_long_sequences(dim, bits, dtype):
    """60 000 keys whose channels have large offsets: what every product cuts from a sum adds up with the keys, and must not
    show beside the output's rounding, in the dims of either half of a byte."""
    n = 60000
    g = gen(dim)
    k = torch.randn(n, 2, dim, generator=g, device=DEV) + 4 * torch.randn(2, dim, generator=g, device=DEV)
    v = 0.7 * torch.randn(n, 2, dim, generator=g, device=DEV)
    c = Held([k.to(dtype)], [v.to(dtype)], bits)
    q = torch.randn(4, 16, dim, generator=g, device=DEV).to(dtype)
    got, want = c.attend(q, [4], [n] * 4, dim ** -0.5), c.exact(q, [4], [n] * 4, dim ** -0.5)
    for half in (slice(0, None, 2), slice(1, None, 2)):
        assert distance(got[..., half], want[..., half]) < LIMIT


@pytest.mark.parametrize("per", [1, 6])
@pytest.mark.parametrize("bits", [4, 8])
def test_precision_of_small_groups_of_v(bits, per):
    """V whose second group is 2^8 smaller: each group's error is its own."""
    dim, n = 128, 200
    k, v = keys_of(n, 1, dim, torch.bfloat16, 5)
    v[..., 64:] *= 2.0 ** -8
    c = Held([k], [v], bits)
    q = torch.randn(per, 16, dim, generator=gen(2), device=DEV).to(torch.bfloat16)
    got, want = c.attend(q, [per], [n] * per, 0.09), c.exact(q, [per], [n] * per, 0.09)
    for part in (slice(0, 64), slice(64, 128)):
        assert distance(got[..., part], want[..., part]) < LIMIT


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("per", [1, 2, 6, 40])
@pytest.mark.parametrize("bits", [4, 8])
def test_precision_of_groups_of_many_sizes(bits, per, dtype):
    """V whose four groups are 1, 2^-4, 2^-8 and 2^-12 times as large: each one's error is its own.  (f16 outputs of the
    last would be subnormal: V is larger there.)"""
    dim, n = 256, 200
    k, v = keys_of(n, 1, dim, dtype, 5)
    v = v.float() * torch.tensor([1, 2.0 ** -4, 2.0 ** -8, 2.0 ** -12], device=DEV).repeat_interleave(64)
    c = Held([k], [(v * 2.0 ** 12).to(dtype)], bits)
    q = torch.randn(per, 16, dim, generator=gen(2), device=DEV).to(dtype)
    got, want = c.attend(q, [per], [n] * per, 0.06), c.exact(q, [per], [n] * per, 0.06)
    for part in range(0, dim, 64):
        assert distance(got[..., part:part + 64], want[..., part:part + 64]) < LIMIT, part


# ------------------------------------------------------------------- what rows may depend on
def larger(x, at, size):
    """The same rows, but the one at `at` is `size` times as large."""
    y = x.clone()
    y[at] = y[at] * size
    return y


def unseen_keys_change_nothing(which, dim, bits, rows):
    """A key inside the sequence that only its last row sees, ever larger: every other row's bits stay."""
    n = 120
    k, v = keys_of(n, 1, dim, torch.bfloat16, dim + rows)
    q = torch.randn(rows, 8, dim, generator=gen(rows), device=DEV).to(torch.bfloat16)
    lens = [n - rows + 1 + i for i in range(rows)]
    lens[0] = 20   # and one row far from the others
    plain = Held([k], [v], bits).attend(q, [rows], lens, 0.08)
    for size in (2.0 ** 8, 2.0 ** 14, 2.0 ** 20, 2.0 ** 60):
        c = Held([larger(k, n - 1, size) if which == "k" else k], [larger(v, n - 1, size) if which == "v" else v], bits)
        assert torch.equal(c.attend(q, [rows], lens, 0.08)[:-1], plain[:-1]), size
    c = Held([larger(k, 30, 2.0 ** 20)], [larger(v, 30, 2.0 ** 20)], bits)
    assert torch.equal(c.attend(q, [rows], lens, 0.08)[0], plain[0])


def large_keys_of_no_weight_change_little(size, dim, bits, rows):
    """Keys that all rows see with a weight of 0, K and V far larger: the others keep their precision."""
    n = 120
    k, v = keys_of(n, 1, dim, torch.bfloat16, dim + rows)
    q = torch.randn(rows, 8, dim, generator=gen(rows), device=DEV).abs().to(torch.bfloat16)
    for at in (3, 70, 71):
        k[at] = -size * (1 + k[at].float().abs()).to(torch.bfloat16)   # a score far below every other
        v[at] = v[at] * size
    c = Held([k], [v], bits)
    assert distance(c.attend(q, [rows], [n] * rows, 0.08), c.exact(q, [rows], [n] * rows, 0.08)) < LIMIT


@pytest.mark.parametrize("rows", [6, 40])
@pytest.mark.parametrize("dim,bits", FORMS)
@pytest.mark.parametrize("which", ["k", "v"])
def test_unseen_keys_of_many_rows(which, dim, bits, rows):
    unseen_keys_change_nothing(which, dim, bits, rows)


@pytest.mark.parametrize("rows", [6, 40])
@pytest.mark.parametrize("dim,bits", FORMS)
@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 20, 2.0 ** 40])
def test_large_keys_of_many_rows(size, dim, bits, rows):
    large_keys_of_no_weight_change_little(size, dim, bits, rows)


@pytest.mark.parametrize("rows", [2, 3])
@pytest.mark.parametrize("dim,bits", FORMS)
@pytest.mark.parametrize("which", ["k", "v"])
def test_unseen_keys_of_few_rows(which, dim, bits, rows):
    unseen_keys_change_nothing(which, dim, bits, rows)


@pytest.mark.parametrize("rows", [1, 2, 3])
@pytest.mark.parametrize("dim,bits", FORMS)
@pytest.mark.parametrize("size", [2.0 ** 12, 2.0 ** 20, 2.0 ** 40])
def test_large_keys_of_few_rows(size, dim, bits, rows):
    large_keys_of_no_weight_change_little(size, dim, bits, rows)


@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("dim,bits", FORMS)
@pytest.mark.parametrize("v_size", [2.0 ** -30, 1.0, 2.0 ** 30, 2.0 ** 90])
def test_scores_of_any_size(dim, bits, rows, v_size):
    """Scores of about 2^26, 2^40 and 2^80: one key of each row leads by far more than its score's error, and its V is the
    result, whatever V's size: half a step of bf16 (2^-8), and half a step of f16 (2^-11) each for a weight and a value, or 2^-16
    of the largest scale of its token, which is below 2^-2 of the largest value."""
    n = 150
    k, v = keys_of(n, 1, dim, torch.bfloat16, dim)
    v = (v.float() * v_size).to(torch.bfloat16)
    c = Held([k], [v], bits)
    for size in (2.0 ** 24, 2.0 ** 38, 2.0 ** 78):
        q = (size * torch.randn(rows, 8, dim, generator=gen(rows), device=DEV)).to(torch.bfloat16)
        x = torch.einsum("rhd,nd->rhn", q.double(), held(k, bits)[:, 0])
        lead = x.topk(2, -1).values
        sure = (lead[..., 0] - lead[..., 1]) > 2.0 ** -10 * x.abs().amax(-1)
        assert sure.float().mean() > 0.8
        got, want = c.attend(q, [rows], [n] * rows, 0.08), c.exact(q, [rows], [n] * rows, 0.08)
        err = (got.double() - want).abs()
        top = want.abs().amax(-1, keepdim=True)
        assert bool((err <= (2.0 ** -8 + 2.0 ** -10) * want.abs() + 2.0 ** -18 * top)[sure].all())


# ------------------------------------------------------------------------------ rows without keys
@pytest.mark.parametrize("rows", [1, 9, 40])
@pytest.mark.parametrize("bits", [4, 8])
def test_rows_without_keys_are_0_whatever_their_gate(bits, rows):
    """Rows of no keys and of no sequence, as padding leaves them: queries and gates of any kind, MXFP8 output too."""
    from zstep_b200.ops import mx

    dim, n = 128, 50
    k, v = keys_of(n, 2, dim, torch.bfloat16, 3)
    c = Held([k], [v], bits)
    q = torch.randn(rows + 2, 16, dim, generator=gen(rows), device=DEV).to(torch.bfloat16)
    gate = torch.randn(q.shape, generator=gen(rows + 1), device=DEV).to(torch.bfloat16)
    for r, bad in ((0, float("nan")), (rows, float("inf")), (rows + 1, float("nan"))):
        q[r], gate[r] = bad, bad
    lens = [0] + [n] * rows + [n]
    plan = QuantAttention(c.cache, 16, max_rows=rows + 2, max_seqs=1, max_seq_rows=rows + 1)
    plan.update(i32([0] * (rows + 2)), i32(lens), i32([0, rows]))   # the last two rows are of no sequence
    out = torch.full((rows + 2, 16 * dim), 7.0, dtype=torch.bfloat16, device=DEV)
    out_q = torch.full((128, 16 * dim), 9, dtype=torch.uint8, device=DEV)
    out_sf = torch.zeros(mx.atoms_bytes(rows + 2, 16 * dim), dtype=torch.uint8, device=DEV)
    plan.attend(0, q, c.table, 0.09, gate=gate, out=out, out_q=out_q, out_sf=out_sf)
    plan.check()
    got = mx.dequantize(out_q[:rows + 2], mx.codes_from_atoms(out_sf, rows + 2, 16 * dim))
    for r in (0, rows, rows + 1):
        assert not out[r].any() and not got[r].any()
    assert bool(out.isfinite().all()) and bool(got.isfinite().all())


def test_reads_into_rows_that_share_memory_are_refused():
    k, v = keys_of(20, 2, 64, torch.bfloat16, 3)
    c = Held([k], [v], 4)
    at = i32([0] * 4), i32([1, 2, 3, 4])
    one, own = torch.zeros(1, 2, 64, dtype=torch.bfloat16, device=DEV), torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=DEV)
    for shared in (one.expand(4, 2, 64), own[:, :1].expand(4, 2, 64)):
        for kw in (dict(k=shared, v=own), dict(k=own, v=shared)):
            with pytest.raises(RuntimeError, match="share memory"):
                c.cache.read(0, c.table, *at, **kw)
    # Rows to write from may be one row: a constant prefix, say.
    c.cache.write(0, one.expand(4, 2, 64), one.expand(4, 2, 64), c.table, *at)
    assert not c.cache.read(0, c.table, *at)[0].any()
    c.cache.read(0, c.table, at[0][:1], at[1][:1], k=one, v=own[:1])
    c.cache.check()
