"""The K/V cache held in 4 or 8 bits: rows written and read back, and attention over it."""

import math

import numpy as np
import pytest
import torch

from zstep_b200.ops.pages import PagePool
from zstep_b200.ops.quant_cache import QuantAttention, QuantCache

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _bf16_beside(x, up):
    """The nearest bf16 not below (up) or not above 64-bit numbers; exact down to 2^-126."""
    m, e = np.frexp(x)
    return np.ldexp((np.ceil if up else np.floor)(np.ldexp(m, 8)), e - 8)


def quantised(x, bits):
    """What a cache holds of rows [n, heads, dim], in 64 bits: values and their scales and offsets."""
    f = x.double().cpu().numpy().reshape(*x.shape[:2], -1, 64)
    z = _bf16_beside(f.min(-1, keepdims=True), False)
    s = _bf16_beside((f.max(-1, keepdims=True) - z) / (2 ** bits - 1), True)
    with np.errstate(divide="ignore", invalid="ignore"):
        n = np.where(s > 0, np.rint((f - z) / s), 0.0)
    n = np.minimum(n, 2 ** bits - 1)
    return (n * s + z).reshape(x.shape), s, z


def rows_of(n, heads, dim, dtype, seed, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    size = torch.exp(torch.randn(heads, dim, generator=g, device=DEV) * 0.5)
    return (scale * size * (torch.randn(n, heads, dim, generator=g, device=DEV) + torch.randn(heads, dim, generator=g, device=DEV))).to(dtype)


def table_of(lens, page, seed=0, spare=1):
    """Shuffled pages (from 1) for sequences of these lengths; (page_table, pages in all)."""
    need = [max(1, -(-n // page)) for n in lens]
    ids = np.random.default_rng(seed).permutation(sum(need)) + 1
    t = np.zeros((len(lens), max(need) + spare), dtype=np.int32)
    at = 0
    for i, k in enumerate(need):
        t[i, :k] = ids[at:at + k]
        at += k
    return torch.from_numpy(t).to(DEV), sum(need) + 1


def places_of(lens):
    return _i32(np.repeat(np.arange(len(lens)), lens)), _i32(np.concatenate([np.arange(n) for n in lens] + [np.zeros(0)]).astype(int))


# ------------------------------------------------------------------------------ write, read
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("bits", [4, 8])
def test_rows_read_back(bits, dim, page, dtype):
    lens, heads = [1, 17, 130], 3
    table, pages = table_of(lens, page)
    slots, pos = places_of(lens)
    k, v = rows_of(len(slots), heads, dim, dtype, 1), rows_of(len(slots), heads, dim, dtype, 2, 0.01)
    cache = QuantCache(2, pages, heads, dim, bits=bits, page_size=page)
    cache.write(1, k, v, table, slots, pos)
    got = cache.read(1, table, slots, pos, dtype=torch.float32)
    cache.check()
    for x, y in zip((k, v), got):
        want, s, z = quantised(x, bits)
        # The 32-bit sum s n + z is rounded once.
        assert np.all(np.abs(y.double().cpu().numpy() - want) <= 2.0 ** -24 * np.abs(want))
        # And what is held is within half a step and a rounding of what was written.
        step = np.repeat(s, 64, -1).reshape(x.shape)
        assert np.all(np.abs(x.double().cpu().numpy() - want) <= step * (0.5 + 2.0 ** -20))
    for t in (torch.bfloat16, torch.float16):
        for a, b in zip(cache.read(1, table, slots, pos, dtype=t), got):
            assert torch.equal(a, b.to(t))
    assert not cache.data[0].any()   # the other layer is as it was


def test_strided_rows_and_given_outputs():
    heads, dim, n = 2, 128, 21
    table, pages = table_of([n], 16)
    slots, pos = places_of([n])
    whole = rows_of(n, 3 * heads + 1, dim, torch.bfloat16, 3)
    k, v = whole[:, 1:1 + heads], whole[:, 2:2 + 2 * heads:2]
    a, b = QuantCache(1, pages, heads, dim), QuantCache(1, pages, heads, dim)
    a.write(0, k, v, table, slots, pos)
    b.write(0, k.contiguous(), v.contiguous(), table, slots, pos)
    assert torch.equal(a.data, b.data)
    out = torch.full((n, 2 * heads + 1, dim), 7.0, dtype=torch.float16, device=DEV)
    a.read(0, table, slots, pos, k=out[:, :heads], v=out[:, heads + 1:])
    want = b.read(0, table, slots, pos, dtype=torch.float16)
    assert torch.equal(out[:, :heads], want[0]) and torch.equal(out[:, heads + 1:], want[1])
    assert bool((out[:, heads] == 7).all())


@pytest.mark.parametrize("bits", [4, 8])
def test_special_groups(bits):
    """Constant, tiny, huge and non-finite groups; each spoils only itself."""
    dim, heads = 256, 1
    x = rows_of(8, heads, dim, torch.bfloat16, 4)
    x[0, 0, :64] = 0.0
    x[0, 0, 64:128] = -3.25
    x[1, 0, 5] = float("nan")
    x[2, 0, 70] = float("inf")
    x[3, 0, 200] = float("-inf")
    x[4, 0, 64:128] *= 2.0 ** -100
    x[5, 0, :64] *= 2.0 ** 100
    x[6, 0, 128:192] = 0.0
    x[6, 0, 130] = 2.0 ** -133           # the smallest bf16: N steps do not fit under it
    x[7, 0, 3] = 2.0 ** 127
    table, pages = table_of([8], 16)
    slots, pos = places_of([8])
    cache = QuantCache(1, pages, heads, dim, bits=bits)
    cache.write(0, x, x.flip(0), table, slots, pos)
    k, v = (t.double().cpu().numpy() for t in cache.read(0, table, slots, pos, dtype=torch.float32))
    bad = np.zeros((8, 1, 4), dtype=bool)
    bad[1, 0, 0] = bad[2, 0, 1] = bad[3, 0, 3] = bad[7, 0, 0] = True
    bad = np.repeat(bad, 64, -1)
    want, s, _ = quantised(x, bits)
    step = np.repeat(s, 64, -1).reshape(x.shape)
    raw = x.double().cpu().numpy()
    for got, flip in ((k, False), (v, True)):
        got = got[::-1] if flip else got
        assert np.isnan(got[bad]).all() and np.isfinite(got[~bad]).all()
        ok = ~bad
        ok[6, 0, 128:192] = False        # s is a subnormal there: looked at below
        assert np.all(np.abs(got - want)[ok] <= 2.0 ** -24 * np.abs(want)[ok])
        assert np.all(np.abs(got - raw)[ok] <= step[ok] * (0.5 + 2.0 ** -20))
        assert np.abs(got[6, 0, 128:192]).max() <= 2.0 ** -132
    assert np.all(k[0, 0, :64] == 0) and np.all(k[0, 0, 64:128] == -3.25)


def test_rows_without_a_place():
    heads, dim = 2, 64
    table, pages = table_of([16], 16)
    cache = QuantCache(1, pages, heads, dim)
    x = rows_of(4, heads, dim, torch.bfloat16, 5)
    cache.write(0, x, x, table, _i32([0, 0, 0, 0]), _i32([3, -1, -7, 4]))
    k, _ = cache.read(0, table, _i32([0, 0, 0, 0, 0]), _i32([3, 4, -1, 5, 0]), dtype=torch.float32)
    cache.check()
    want = quantised(x, 4)[0]
    assert np.allclose(k[:2].double().cpu().numpy(), want[[0, 3]], rtol=2.0 ** -23, atol=0) and not k[2:].any()
    before = cache.data.clone()
    for slots, pos, tab in (([1], [0], table), ([-1], [0], table), ([0], [32], table), ([0], [0], torch.full_like(table, pages)),
                            ([0], [0], torch.full_like(table, -1))):
        cache.write(0, x[:1], x[:1], tab, _i32(slots), _i32(pos))
        with pytest.raises(RuntimeError, match="outside the cache"):
            cache.check()
        k, v = cache.read(0, tab, _i32(slots), _i32(pos))
        assert not k.any() and not v.any()
        with pytest.raises(RuntimeError, match="outside the cache"):
            cache.check()
    cache.check()
    assert torch.equal(cache.data, before)
    cache.write(0, x[:0], x[:0], table, _i32([]), _i32([]))
    assert cache.read(0, table, _i32([]), _i32([]))[0].shape == (0, heads, dim)


# -------------------------------------------------------------------------------- attention
def filled(lens, heads, dim, bits, page=16, dtype=torch.bfloat16, seed=0, v_scale=1.0):
    """A cache of sequences of these lengths whose other tokens hold poison."""
    table, pages = table_of(lens, page, seed)
    cache = QuantCache(1, pages, heads, dim, bits=bits, page_size=page)
    every = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    all_pos = torch.arange(pages * page, dtype=torch.int32, device=DEV)
    nan = torch.full((pages * page, heads, dim), float("nan"), dtype=dtype, device=DEV)
    cache.write(0, nan, nan, every, torch.zeros_like(all_pos), all_pos)
    slots, pos = places_of(lens)
    if len(slots):
        cache.write(0, rows_of(len(slots), heads, dim, dtype, seed + 10), rows_of(len(slots), heads, dim, dtype, seed + 11, v_scale),
                    table, slots, pos)
    cache.check()
    return cache, table


def reference(cache, table, q, slots, lens, scale, gate=None):
    """Attention over what the cache holds in 64 bits, and a bound of what the kernel may be off by.

    A weight is off by: its f16 rounding (2^-11 relative, 2^-26 of the largest where it is a subnormal), and its
    score's error, which is at most 2^-19 of the sum of the magnitudes that go into it (each of some 2^4 32-bit
    additions cuts 2^-23 of them).  The output is then rounded to its type."""
    rows, hq, dim = q.shape
    kvh = cache.num_kv_heads
    out = np.zeros((rows, hq, dim))
    tol = np.zeros((rows, hq, dim))
    half_step = torch.finfo(q.dtype).eps / 2
    qn = q.double().cpu().numpy()
    for r in range(rows):
        n = int(lens[r])
        if n <= 0:
            continue
        pos = torch.arange(n, dtype=torch.int32, device=DEV)
        k, v = (t.double().cpu().numpy() for t in cache.read(0, table, torch.full_like(pos, int(slots[r])), pos, dtype=torch.float32))
        for h in range(hq):
            kk, vv = k[:, h * kvh // hq], v[:, h * kvh // hq]
            x = kk @ qn[r, h] * scale
            w = np.exp(x - x.max())
            w /= w.sum()
            o = w @ vv
            spread = np.abs(vv).max(0) + np.abs(vv).max()   # |V - z| is at most the span of its group
            # The offsets may be far larger than the values: |s n| + |z| <= 2 (max - min) + |x| of the group, at most 5 max |k|.
            delta = 2.0 ** -19 * np.abs(scale) * (np.abs(qn[r, h]).sum() * 5 * np.abs(kk).max())
            arithmetic = (2.0 ** -11 + n * 2.0 ** -26 + 2 * delta + 2.0 ** -18) * spread
            g = 1.0
            if gate is not None:
                g = 1 / (1 + np.exp(-gate[r, h].double().cpu().numpy()))
            out[r, h] = o * g
            # The gate's sigmoid: 2^-20 relative.
            tol[r, h] = arithmetic * g + (half_step + 2.0 ** -20) * np.abs(out[r, h]) + 2.0 ** -25
    return out.reshape(rows, -1), tol.reshape(rows, -1)


def check_attention(cache, table, hq, slots, lens, starts=None, dtype=torch.bfloat16, gate=False, seed=0, scale=None, plan=None):
    rows = len(slots)
    g = torch.Generator(device=DEV).manual_seed(seed + 100)
    q = torch.randn(rows, hq, cache.head_dim, generator=g, device=DEV).to(dtype)
    gt = torch.randn(rows, hq, cache.head_dim, generator=g, device=DEV).to(dtype) if gate else None
    scale = cache.head_dim ** -0.5 if scale is None else scale
    if plan is None:
        most = 1 if starts is None else max([b - a for a, b in zip(starts, starts[1:])] + [1])
        plan = QuantAttention(cache, hq, max_rows=max(rows, 1), max_seqs=max(1, rows if starts is None else len(starts) - 1), max_seq_rows=most)
    plan.update(_i32(slots), _i32(lens), None if starts is None else _i32(starts))
    got = plan.attend(0, q, table, scale, gate=gt)
    plan.check()
    want, tol = reference(cache, table, q, slots, lens, scale, gt)
    err = np.abs(got.double().cpu().numpy() - want)
    assert np.all(err <= tol), (float(np.nanmax(err / np.maximum(tol, 1e-300))), np.isnan(err).sum(), np.argwhere(~(err <= tol))[:4].tolist())
    return got


@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 1), (6, 2), (16, 2), (16, 1), (12, 12)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("bits", [4, 8])
def test_decode_rows(bits, dim, hq, hkv):
    lens = [1, 15, 16, 17, 33, 300, 0, 700]
    cache, table = filled(lens, hkv, dim, bits, seed=dim + hq)
    check_attention(cache, table, hq, list(range(len(lens))), lens, gate=hq == 16, seed=hq)


@pytest.mark.parametrize("page", [32, 128])
def test_larger_pages(page):
    lens = [5, 129, 260]
    cache, table = filled(lens, 2, 128, 4, page=page, seed=9)
    check_attention(cache, table, 8, [2, 0, 1], [260, 5, 129])


@pytest.mark.parametrize("dim,bits", [(64, 4), (128, 4), (256, 4), (64, 8), (128, 8), (256, 8)])
@pytest.mark.parametrize("per", [2, 4, 9, 40])
def test_rows_of_a_sequence(dim, bits, per):
    """Verify rows and chunks: rows of one sequence, each up to its own length, in ragged numbers."""
    lens = [per + 3, 200, 67]
    cache, table = filled(lens, 2, dim, bits, seed=per)
    counts = [per, max(1, per - 1), per]
    starts = [0, per, per + counts[1], sum(counts)]
    slots = [s for s, c in enumerate(counts) for _ in range(c)]
    seen = [lens[s] - c + 1 + i for s, c in enumerate(counts) for i in range(c)]
    check_attention(cache, table, 8, slots, seen, starts, gate=True, seed=per)


def test_many_heads_of_one_kv_head():
    """More q heads than one work unit holds, and rows whose heads are in two units."""
    cache, table = filled([90, 41], 1, 256, 4, seed=3)
    check_attention(cache, table, 160, [0, 0, 0, 1], [88, 89, 90, 41], [0, 3, 4])


def test_lengths_in_any_order_and_rows_of_no_sequence():
    cache, table = filled([100, 50, 40], 2, 128, 4, seed=5)
    starts = [0, 3, 3, 5]   # the second sequence has no rows; row 5 belongs to none
    plan = QuantAttention(cache, 4, max_rows=6, max_seqs=4, max_seq_rows=3)
    slots, seen = [0, 0, 0, 2, 2, 1], [100, 0, 7, 40, 39, 50]
    g = torch.Generator(device=DEV).manual_seed(1)
    q = torch.randn(6, 4, 128, generator=g, device=DEV).to(torch.bfloat16)
    plan.update(_i32(slots), _i32(seen), _i32(starts))
    got = plan.attend(0, q, table, 0.1)
    plan.check()
    want, tol = reference(cache, table, q[:5], slots[:5], seen[:5], 0.1)
    assert np.all(np.abs(got[:5].double().cpu().numpy() - want) <= tol) and not got[5].any() and not got[1].any()


def test_f16_and_extreme_sizes():
    cache, table = filled([130, 77], 2, 128, 4, dtype=torch.float16, seed=6)
    check_attention(cache, table, 8, [0, 1], [130, 77], dtype=torch.float16, gate=True)
    for v_scale in (2.0 ** -40, 2.0 ** 60):
        cache, table = filled([130, 77], 2, 128, 4, seed=7, v_scale=v_scale)
        q = torch.randn(2, 8, 128, device=DEV).to(torch.bfloat16)
        plan = QuantAttention(cache, 8, 2)
        plan.update(_i32([0, 1]), _i32([130, 77]))
        got = plan.attend(0, q, table, 0.09).double().cpu().numpy()
        want, tol = reference(cache, table, q, [0, 1], [130, 77], 0.09)
        assert np.all(np.abs(got - want) <= tol - 2.0 ** -25)
    # Queries of any size: the scores of the small ones are all alike, those of the large ones pick a key.
    cache, table = filled([130], 2, 128, 4, seed=8)
    for size in (2.0 ** -90, 2.0 ** 40):
        q = (size * torch.randn(1, 8, 128, device=DEV)).to(torch.bfloat16)
        plan = QuantAttention(cache, 8, 1)
        plan.update(_i32([0]), _i32([130]))
        got = plan.attend(0, q, table, 0.09).double().cpu().numpy()
        want, tol = reference(cache, table, q, [0], [130], 0.09)
        if size < 1:
            assert np.all(np.abs(got - want) <= tol)
        else:   # the winner leads by far more than its score's error
            assert np.all(np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -11 * np.abs(want).max() * 4)


def test_large_and_uneven_scores():
    """One key far above the others, early or late, and V groups of very different sizes."""
    lens, dim = [400], 128
    table, pages = table_of(lens, 16)
    cache = QuantCache(1, pages, 1, dim)
    slots, pos = places_of(lens)
    k, v = rows_of(400, 1, dim, torch.bfloat16, 1), rows_of(400, 1, dim, torch.bfloat16, 2)
    v[:, :, 64:] *= 2.0 ** -12
    for hot in (0, 399, 170):
        k2 = k.clone()
        k2[hot] *= 12
        cache.write(0, k2, v, table, slots, pos)
        check_attention(cache, table, 8, [0], lens, seed=hot)


def test_poison_and_masks():
    """NaN in K that a row sees makes the row NaN; in V only the dims of its group; behind the length nothing."""
    dim, n = 128, 50
    table, pages = table_of([n], 16)
    slots, pos = places_of([n])
    k, v = rows_of(n, 1, dim, torch.bfloat16, 1), rows_of(n, 1, dim, torch.bfloat16, 2)
    q = torch.randn(3, 4, dim, device=DEV).to(torch.bfloat16)
    plan, seen, starts = None, [39, 40, 41], [0, 3]
    for which in ("k", "v"):
        a, b = k.clone(), v.clone()
        (a if which == "k" else b)[40, 0, 70] = float("nan")   # seen by the last row alone
        cache = QuantCache(1, pages, 1, dim)
        cache.write(0, a, b, table, slots, pos)
        plan = QuantAttention(cache, 4, 3, 1, 3)
        plan.update(_i32([0, 0, 0]), _i32(seen), _i32(starts))
        got = plan.attend(0, q, table, 0.1).view(3, 4, dim)
        want, tol = reference(cache, table, q[:2], [0, 0], seen[:2], 0.1)
        assert np.all(np.abs(got[:2].double().cpu().numpy().reshape(2, -1) - want) <= tol)
        if which == "k":
            assert bool(got[2].isnan().all())
        else:
            assert bool(got[2, :, 64:].isnan().all()) and bool(got[2, :, :64].isfinite().all())
    # A query that is not finite spoils its own head only.
    cache = QuantCache(1, pages, 1, dim)
    cache.write(0, k, v, table, slots, pos)
    q[1, 2, 5] = float("inf")
    plan.cache = cache
    plan.update(_i32([0, 0, 0]), _i32(seen), _i32(starts))
    got = plan.attend(0, q, table, 0.1).view(3, 4, dim)
    assert bool(got[1, 2].isnan().all())
    got[1, 2] = 0
    assert bool(got.isfinite().all())


@pytest.mark.parametrize("dim,bits,hq", [(64, 4, 16), (128, 4, 8), (256, 4, 8), (64, 8, 16), (128, 8, 32), (256, 8, 16)])
def test_what_stands_behind_a_sequence_does_not_matter(dim, bits, hq):
    """Values of any size in the places behind a length, and other sequences' in the blocks read before."""
    lens = [1, 17, 300, 33, 5]
    table, pages = table_of(lens, 16)
    cache = QuantCache(1, pages, 1, dim, bits=bits)
    every = torch.arange(pages, dtype=torch.int32, device=DEV)[None]
    at = torch.arange(pages * 16, dtype=torch.int32, device=DEV)
    huge = rows_of(pages * 16, 1, dim, torch.bfloat16, 1, 2.0 ** 100)
    cache.write(0, huge, huge, every, torch.zeros_like(at), at)
    slots, pos = places_of(lens)
    cache.write(0, rows_of(len(slots), 1, dim, torch.bfloat16, 2), rows_of(len(slots), 1, dim, torch.bfloat16, 3), table, slots, pos)
    check_attention(cache, table, hq, list(range(5)) * 40, lens * 40)


def test_tokens_in_any_order():
    """Rows whose tokens are scattered, alone and by fours, hold what rows in order do."""
    n, dim = 64, 128
    table, pages = table_of([n], 16)
    for bits in (4, 8):
        a, b = QuantCache(1, pages, 2, dim, bits=bits), QuantCache(1, pages, 2, dim, bits=bits)
        slots, pos = places_of([n])
        k, v = rows_of(n, 2, dim, torch.bfloat16, 1), rows_of(n, 2, dim, torch.bfloat16, 2)
        a.write(0, k, v, table, slots, pos)
        for order in (torch.randperm(n, device=DEV), torch.arange(n, device=DEV).view(4, 4, 4).transpose(1, 2).reshape(-1),
                      (torch.arange(n, device=DEV) + 3) % n, torch.arange(n, device=DEV).flip(0)):
            b.data.zero_()
            for part in order.split(23):
                b.write(0, k[part], v[part], table, slots[part], pos[part])
            assert torch.equal(a.data, b.data)
            for x, y in zip(b.read(0, table, slots[order], pos[order]), a.read(0, table, slots, pos)):
                assert torch.equal(x, y[order])


def test_strided_queries_and_mxfp8():
    from zstep_b200.ops import mx

    lens, hq, dim = [130, 77, 200], 8, 256
    cache, table = filled(lens, 2, dim, 4, seed=12)
    wide = torch.randn(3, 2 * hq + 1, dim, device=DEV).to(torch.bfloat16)
    q, gate = wide[:, 0:2 * hq:2], wide[:, 1:2 * hq:2]
    plan = QuantAttention(cache, hq, 3)
    plan.update(_i32([0, 1, 2]), _i32(lens))
    out = torch.empty(3, hq * dim, dtype=torch.bfloat16, device=DEV)
    out_q = torch.empty(128, hq * dim, dtype=torch.uint8, device=DEV)
    out_sf = torch.zeros(mx.atoms_bytes(3, hq * dim), dtype=torch.uint8, device=DEV)
    plan.attend(0, q, table, 0.0625, gate=gate, out=out, out_q=out_q, out_sf=out_sf)
    same = plan.attend(0, q.contiguous(), table, 0.0625, gate=gate.contiguous())
    assert torch.equal(out, same)
    got = mx.dequantize(out_q[:3], mx.codes_from_atoms(out_sf, 3, hq * dim))
    # e4m3: half a step is 2^-4 of the value, or 2^-10 of the block's scale where it is a subnormal; bf16's rounding.
    block = out.float().abs().view(3, -1, 32).amax(-1, keepdim=True).expand(-1, -1, 32).reshape(3, -1)
    assert bool(((got - out.float()).abs() <= out.float().abs() * (2.0 ** -4 + 2.0 ** -8) + block * 2.0 ** -10).all())


def test_long_sequence_is_split_and_repeats_exactly():
    """A lone long sequence takes every SM; the result does not depend on the order they finish in."""
    n, dim = 20000, 64
    table, pages = table_of([n], 16)
    cache = QuantCache(1, pages, 1, dim)
    slots, pos = places_of([n])
    cache.write(0, rows_of(n, 1, dim, torch.bfloat16, 1), rows_of(n, 1, dim, torch.bfloat16, 2), table, slots, pos)
    first = check_attention(cache, table, 2, [0], [n - 3], seed=3)
    for _ in range(3):
        assert torch.equal(check_attention(cache, table, 2, [0], [n - 3], seed=3), first)


@pytest.mark.parametrize("dim,bits,dtype", [(64, 4, torch.bfloat16), (128, 8, torch.float16), (256, 4, torch.bfloat16), (256, 8, torch.bfloat16)])
def test_long_sequences_of_many_rows(dim, bits, dtype):
    """Five rows of eight heads over sequences long enough that every SM has dozens of tiles and several sequences."""
    lens, hkv, per = [30000, 24001, 17000], 4, 5
    cache, table = filled(lens, hkv, dim, bits, page=64, dtype=dtype, seed=dim)
    g = torch.Generator(device=DEV).manual_seed(5)
    q = torch.randn(len(lens) * per, 8 * hkv, dim, generator=g, device=DEV).to(dtype)
    slots = [s for s in range(3) for _ in range(per)]
    seen = [n - per + 1 + i for n in lens for i in range(per)]
    plan = QuantAttention(cache, 8 * hkv, max_rows=15, max_seqs=3, max_seq_rows=per)
    plan.update(_i32(slots), _i32(seen), _i32([0, 5, 10, 15]))
    got = plan.attend(0, q, table, dim ** -0.5)
    plan.check()
    rows = [0, 7, 14]
    want, tol = reference(cache, table, q[rows], [slots[r] for r in rows], [seen[r] for r in rows], dim ** -0.5)
    assert np.all(np.abs(got[rows].double().cpu().numpy() - want) <= tol)
    for _ in range(3):
        assert torch.equal(plan.attend(0, q, table, dim ** -0.5), got)


def test_many_short_sequences():
    rng = np.random.default_rng(3)
    lens = rng.integers(0, 60, 700).tolist()
    cache, table = filled(lens, 1, 64, 4, seed=2)
    check_attention(cache, table, 2, list(range(700)), lens)


def test_places_outside_are_reported():
    cache, table = filled([40], 1, 64, 4)
    q = torch.randn(1, 2, 64, device=DEV).to(torch.bfloat16)
    plan = QuantAttention(cache, 2, 4, 2, 2)
    for slots, lens, starts, tab in (([1], [40], None, table), ([-1], [40], None, table), ([0], [65], None, table),
                                     ([0], [40], None, torch.full_like(table, cache.num_pages)), ([0], [40], [0, 2], table),
                                     ([0], [40], [1, 0], table), ([0], [40], [-1, 1], table)):
        plan.update(_i32(slots), _i32(lens), None if starts is None else _i32(starts))
        plan.attend(0, q, tab, 0.1)
        with pytest.raises(RuntimeError, match="error status"):
            plan.check()
    check_attention(cache, table, 2, [0], [40], plan=plan)
    plan.update(_i32([0, 0, 0]), _i32([1, 2, 3]), _i32([0, 3]))   # more rows of a sequence than the plan takes
    with pytest.raises(RuntimeError, match="error status"):
        plan.check()
    plan.update(_i32([0] * 4), _i32([9] * 4), _i32([0, 2, 4]))
    plan.check()


# --------------------------------------------------------------------------------- together
def test_generation_loop_in_a_graph_over_a_page_pool():
    """Prompt rows written and attended as a chunk, sequences forked, then single tokens written and attended by one
    captured graph, replayed."""
    hkv, hq, dim = 2, 8, 128
    cache = QuantCache(1, 64, hkv, dim)
    pool = PagePool([cache.data], num_slots=4, max_pages=8)
    g = torch.Generator(device=DEV).manual_seed(0)
    rnd = lambda n, h: torch.randn(n, h, dim, generator=g, device=DEV).to(torch.bfloat16)  # noqa: E731
    prompt = 37
    pool.extend(_i32([0]), _i32([prompt]))
    slots, pos = places_of([prompt])
    k, v, q = rnd(prompt, hkv), rnd(prompt, hkv), rnd(prompt, hq)
    cache.write(0, k, v, pool.page_table, slots, pos)
    chunk = QuantAttention(cache, hq, prompt, 1, prompt)
    chunk.update(slots, pos + 1, _i32([0, prompt]))
    got = chunk.attend(0, q, pool.page_table, 0.1)
    want, tol = reference(cache, pool.page_table, q, [0] * prompt, (pos + 1).tolist(), 0.1)
    assert np.all(np.abs(got.double().cpu().numpy() - want) <= tol)
    pool.fork(_i32([0, 0]), _i32([2, 3]))
    live = _i32([0, 2, 3])
    step = QuantAttention(cache, hq, 3)
    k, v, q = rnd(3, hkv), rnd(3, hkv), rnd(3, hq)
    out = torch.empty(3, hq * dim, dtype=torch.bfloat16, device=DEV)
    at = torch.full((3,), prompt, dtype=torch.int32, device=DEV)

    def one():
        pool.extend(live, at + 1)
        cache.write(0, k, v, pool.page_table, live, at)
        step.update(live, at + 1)
        step.attend(0, q, pool.page_table, 0.1, out=out)
        at.add_(1)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        one()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one()
    for i in range(1, 30):
        k.copy_(rnd(3, hkv))
        v.copy_(rnd(3, hkv))
        q.copy_(rnd(3, hq))
        graph.replay()
        n = prompt + i + 1
        want, tol = reference(cache, pool.page_table, q, [0, 2, 3], [n] * 3, 0.1)
        assert np.all(np.abs(out.double().cpu().numpy() - want) <= tol), i
        held = cache.read(0, pool.page_table, live, at - 1, dtype=torch.float32)[0].double().cpu().numpy()
        assert np.allclose(held, quantised(k, 4)[0], rtol=2.0 ** -23, atol=0)
    for x in (pool, cache, step, chunk):
        x.check()


def test_plan_is_shared_by_layers_and_its_workspace_is_reused():
    lens, dim = [90, 33], 128
    table, pages = table_of(lens, 16)
    cache = QuantCache(3, pages, 2, dim)
    slots, pos = places_of(lens)
    for layer in range(3):
        cache.write(layer, rows_of(len(slots), 2, dim, torch.bfloat16, layer), rows_of(len(slots), 2, dim, torch.bfloat16, 9 + layer),
                    table, slots, pos)
    plan = QuantAttention(cache, 4, 2)
    q = torch.randn(2, 4, dim, device=DEV).to(torch.bfloat16)
    plan.update(_i32([0, 1]), _i32(lens))
    got = [plan.attend(layer, q, table, 0.1).clone() for layer in range(3)]
    for layer in range(3):
        one = QuantCache(1, pages, 2, dim)
        one.data[0].copy_(cache.data[layer])
        want, tol = reference(one, table, q, [0, 1], lens, 0.1)
        assert np.all(np.abs(got[layer].double().cpu().numpy() - want) <= tol)
    assert math.isfinite(float(got[0].float().sum()))


# ------------------------------------------------------------- many query slots, and the ends of the ranges
def wide_tolerance(cache, table, q, slots, lens, scale):
    """What sequences of many slots may be off by in addition: K and V go through f16 there, which is half a step
    (2^-12) of a value, or 2^-16 of the largest scale of its block (at most 2^-3 of the largest value) where it is a
    subnormal.  A score is then off by that share of the sum of |q| |k|, a weight by twice that, V by the share itself."""
    rows, hq, dim = q.shape
    kvh = cache.num_kv_heads
    tol = np.zeros((rows, hq, dim))
    qn = q.double().abs().sum(-1).cpu().numpy()
    for r in range(rows):
        if int(lens[r]) <= 0:
            continue
        pos = torch.arange(int(lens[r]), dtype=torch.int32, device=DEV)
        k, v = (t.double().abs().cpu().numpy() for t in cache.read(0, table, torch.full_like(pos, int(slots[r])), pos, dtype=torch.float32))
        for h in range(hq):
            kk, vv = k[:, h * kvh // hq].max(), v[:, h * kvh // hq]
            share = 2.0 ** -12 + 2.0 ** -19
            tol[r, h] = (2 * abs(scale) * qn[r, h] * share * kk + share) * (vv.max(0) + vv.max())
    return tol.reshape(rows, -1)


def run_rows(cache, table, q, slots, lens, starts, scale, **kw):
    most = max([b - a for a, b in zip(starts, starts[1:])] + [1])
    plan = QuantAttention(cache, q.shape[1], max_rows=len(slots), max_seqs=len(starts) - 1, max_seq_rows=most)
    plan.update(_i32(slots), _i32(lens), _i32(starts))
    got = plan.attend(0, q, table, scale, **kw)
    plan.check()
    return got


def assert_near(got, cache, table, q, slots, lens, scale, gate=None, absolute=True):
    want, tol = reference(cache, table, q, slots, lens, scale, gate)
    tol = tol + wide_tolerance(cache, table, q, slots, lens, scale) - (0 if absolute else 2.0 ** -25)
    err = np.abs(got.double().cpu().numpy() - want)
    assert np.all(err <= tol), (float(np.nanmax(err / np.maximum(tol, 1e-300))), int(np.isnan(err).sum()), np.argwhere(~(err <= tol))[:4].tolist())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,bits", [(64, 4), (128, 4), (256, 4), (64, 8), (128, 8), (256, 8)])
@pytest.mark.parametrize("per", [3, 5, 7, 33])
def test_rows_of_each_size_of_unit(dim, bits, per, dtype):
    """12, 20, 28 and 132 slots, both types, pages of 256 tokens; rows without keys and sequences of 0 and 1 keys."""
    lens = [300, 1, 0, 65]
    cache, table = filled(lens, 2, dim, bits, page=256, dtype=dtype, seed=per)
    starts = [i * per for i in range(5)]
    slots = [s for s in range(4) for _ in range(per)]
    seen = [max(0, lens[s] - (i % 3) * (s != 1)) if i != 1 else 0 for s in range(4) for i in range(per)]
    g = torch.Generator(device=DEV).manual_seed(per)
    q = torch.randn(4 * per, 8, dim, generator=g, device=DEV).to(dtype)
    scale = dim ** -0.5
    got = run_rows(cache, table, q, slots, seen, starts, scale)
    assert_near(got, cache, table, q, slots, seen, scale)
    empty = [r for r, n in enumerate(seen) if n == 0]
    assert not got[empty].any()


@pytest.mark.parametrize("per", [1, 4, 20])
@pytest.mark.parametrize("bits", [4, 8])
def test_scores_of_either_sign_and_none(bits, per):
    lens = [100, 37]
    cache, table = filled(lens, 1, 128, bits, seed=per)
    starts, slots, seen = [0, per, 2 * per], [0] * per + [1] * per, [100] * per + [37] * per
    q = torch.randn(2 * per, 8, 128, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(torch.bfloat16)
    for scale in (-0.2, 0.0, 0.2):
        assert_near(run_rows(cache, table, q, slots, seen, starts, scale), cache, table, q, slots, seen, scale)
    plan = QuantAttention(cache, 8, 2 * per)
    plan.update(_i32(slots), _i32(seen))
    for scale in (float("nan"), float("inf"), 1e300):
        with pytest.raises(ValueError, match="sm_scale"):
            plan.attend(0, q, table, scale)


@pytest.mark.parametrize("per", [1, 20])
@pytest.mark.parametrize("dim,bits", [(64, 8), (128, 4), (256, 4), (256, 8)])
def test_values_of_any_size(dim, bits, per):
    """V from 2^-40 to 2^120, K that q makes up for, and V whose groups are constant."""
    lens = [150, 33]
    starts, slots, seen = [0, per, 2 * per], [0] * per + [1] * per, [150] * per + [33] * per
    g = torch.Generator(device=DEV).manual_seed(per)
    q = torch.randn(2 * per, 8, dim, generator=g, device=DEV).to(torch.bfloat16)
    scale = dim ** -0.5
    for v_scale in (2.0 ** -40, 2.0 ** 60, 2.0 ** 104, 2.0 ** 120):
        cache, table = filled(lens, 1, dim, bits, seed=3, v_scale=v_scale)
        got = run_rows(cache, table, q, slots, seen, starts, scale)
        assert_near(got, cache, table, q, slots, seen, scale, absolute=False)
    table, pages = table_of(lens, 16)
    at, pos = places_of(lens)
    for k_scale in (2.0 ** -60, 2.0 ** 90, 2.0 ** 120):
        for const in (0.0, 2.0 ** -30, -2.0 ** 20, 2.0 ** 100):
            cache = QuantCache(1, pages, 1, dim, bits=bits)
            k = rows_of(len(at), 1, dim, torch.bfloat16, 5, k_scale)
            v = torch.full((len(at), 1, dim), const, device=DEV, dtype=torch.bfloat16)
            cache.write(0, k, v, table, at, pos)
            small = (q.float() * min(max(1 / k_scale, 2.0 ** -90), 2.0 ** 90)).to(torch.bfloat16)
            rest = scale / k_scale / min(max(1 / k_scale, 2.0 ** -90), 2.0 ** 90)
            got = run_rows(cache, table, small, slots, seen, starts, rest)
            # Weights that add up to 1 times a constant: the rounding of the weights, the images and the output.
            assert np.all(np.abs(got.double().cpu().numpy() - const) <= abs(const) * (2.0 ** -9 + 2.0 ** -10))


def test_sizes_that_differ_from_group_to_group():
    """V whose groups are 2^12 apart, within a block of many slots too: the small one keeps its own precision."""
    n, dim, per = 200, 128, 20
    table, pages = table_of([n], 16)
    at, pos = places_of([n])
    k, v = rows_of(n, 1, dim, torch.bfloat16, 1), rows_of(n, 1, dim, torch.bfloat16, 2)
    v[:, :, 64:] *= 2.0 ** -8
    for bits in (4, 8):
        cache = QuantCache(1, pages, 1, dim, bits=bits)
        cache.write(0, k, v, table, at, pos)
        q = torch.randn(per, 4, dim, generator=torch.Generator(device=DEV).manual_seed(2), device=DEV).to(torch.bfloat16)
        got = run_rows(cache, table, q, [0] * per, [n] * per, [0, per], 0.09).view(per, 4, 2, 64)
        want, tol = reference(cache, table, q, [0] * per, [n] * per, 0.09)
        vmax = cache.read(0, table, at, pos, dtype=torch.float32)[1].abs().double().cpu().numpy().reshape(n, 2, 64).max((0, 2))
        want = want.reshape(per, 4, 2, 64)
        # A weight is off by 2^-12 and K's rounding, V by 2^-12 of itself and 2^-16 of the block's largest scale (2/15 of
        # its largest value at most), the output by half a step.
        dk = 0.09 * float(q.float().abs().sum(-1).max()) * float(k.float().abs().max()) * (2.0 ** -12 + 2.0 ** -19)
        for gi in range(2):
            limit = 2 * (2 * dk + 2.0 ** -11 + 2.0 ** -17) * vmax[gi] + 2.0 ** -16 * 2 / 15 * vmax.max() + 2.0 ** -8 * np.abs(want[:, :, gi])
            assert np.all(np.abs(got[:, :, gi].double().cpu().numpy() - want[:, :, gi]) <= limit)


@pytest.mark.parametrize("dim,bits", [(64, 8), (128, 4), (256, 4), (256, 8)])
def test_poison_in_many_rows(dim, bits):
    """As for few rows: a poisoned K spoils the rows that see it, a poisoned V their dims of its group."""
    n, per = 90, 45
    table, pages = table_of([n], 16)
    at, pos = places_of([n])
    k, v = rows_of(n, 1, dim, torch.bfloat16, 1), rows_of(n, 1, dim, torch.bfloat16, 2)
    q = torch.randn(per, 4, dim, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV).to(torch.bfloat16)
    q[7, 2, 5] = float("inf")
    q[8, 1, 9] = 2.0 ** 101
    seen = [n - per + 1 + i for i in range(per)]
    for which, group in (("k", 0), ("v", 0), ("v", dim // 64 - 1)):
        a, b = k.clone(), v.clone()
        (a if which == "k" else b)[70, 0, group * 64 + 9] = float("nan")   # seen by rows of more than 70 keys
        cache = QuantCache(1, pages, 1, dim, bits=bits)
        cache.write(0, a, b, table, at, pos)
        got = run_rows(cache, table, q, [0] * per, seen, [0, per], 0.1).view(per, 4, dim)
        bad = torch.zeros(per, 4, dim, dtype=torch.bool, device=DEV)
        sees = torch.tensor([x > 70 for x in seen], device=DEV)
        if which == "k":
            bad[sees] = True
        else:
            bad[sees, :, group * 64:group * 64 + 64] = True
        bad[7, 2] = bad[8, 1] = True
        assert torch.equal(got.isnan(), bad)
        clean = [r for r in range(per) if seen[r] <= 70 and r not in (7, 8)]
        assert_near(got.view(per, -1)[clean], cache, table, q[clean], [0] * len(clean), [seen[r] for r in clean], 0.1)


def test_strided_queries_and_mxfp8_of_many_rows():
    from zstep_b200.ops import mx

    per, hq, dim, n = 140, 4, 128, 260
    cache, table = filled([n], 2, dim, 4, seed=12)
    wide = torch.randn(per, 2 * hq + 1, dim, device=DEV).to(torch.bfloat16)
    q, gate = wide[:, 0:2 * hq:2], wide[:, 1:2 * hq:2]
    seen = [n - per + 1 + i for i in range(per)]
    out = torch.empty(per, hq * dim, dtype=torch.bfloat16, device=DEV)
    out_q = torch.empty(256, hq * dim, dtype=torch.uint8, device=DEV)
    out_sf = torch.zeros(mx.atoms_bytes(per, hq * dim), dtype=torch.uint8, device=DEV)
    run_rows(cache, table, q, [0] * per, seen, [0, per], 0.09, gate=gate, out=out, out_q=out_q, out_sf=out_sf)
    assert_near(out, cache, table, q, [0] * per, seen, 0.09, gate)
    got = mx.dequantize(out_q[:per], mx.codes_from_atoms(out_sf, per, hq * dim))
    block = out.float().abs().view(per, -1, 32).amax(-1, keepdim=True).expand(-1, -1, 32).reshape(per, -1)
    assert bool(((got - out.float()).abs() <= out.float().abs() * (2.0 ** -4 + 2.0 ** -8) + block * 2.0 ** -10).all())


def test_one_row_of_many_heads_and_results_that_repeat():
    """80 heads of a kv head; the same call twice, and on another stream, gives the same bits."""
    lens = [500, 3, 64, 65]
    cache, table = filled(lens, 1, 128, 4, seed=2)
    q = torch.randn(4, 80, 128, generator=torch.Generator(device=DEV).manual_seed(4), device=DEV).to(torch.bfloat16)
    plan = QuantAttention(cache, 80, 4)
    plan.update(_i32([0, 1, 2, 3]), _i32(lens))
    got = plan.attend(0, q, table, 0.09)
    assert_near(got, cache, table, q, [0, 1, 2, 3], lens, 0.09)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x = rows_of(4, 1, 128, torch.bfloat16, 6)
        cache.write(0, x, x, table, _i32([0, 1, 2, 3]), _i32([499, 2, 63, 64]))
        plan.update(_i32([0, 1, 2, 3]), _i32(lens))
        other = plan.attend(0, q, table, 0.09)
        assert_near(other, cache, table, q, [0, 1, 2, 3], lens, 0.09)
        assert torch.equal(plan.attend(0, q, table, 0.09), other)
    torch.cuda.current_stream().wait_stream(side)


def test_graphs_that_share_a_plan():
    """Each captured step plans and attends: replayed in any order they do not disturb one another.  A captured attend
    alone, whose plan was made for other rows since, reports that and gives zeros."""
    lens = [150, 80]
    cache, table = filled(lens, 1, 64, 4, seed=2)
    plan = QuantAttention(cache, 4, 24, 2, 12)
    g = torch.Generator(device=DEV).manual_seed(4)
    steps = []
    for per in (1, 12, 3):
        q = torch.randn(2 * per, 4, 64, generator=g, device=DEV).to(torch.bfloat16)
        s, n, at = _i32([0] * per + [1] * per), _i32([150] * per + [80] * per), _i32([0, per, 2 * per])
        out = torch.empty(2 * per, 256, dtype=torch.bfloat16, device=DEV)
        plan.update(s, n, at)
        plan.attend(0, q, table, 0.125, out=out)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            plan.update(s, n, at)
            plan.attend(0, q, table, 0.125, out=out)
        steps.append((graph, q, s, n, at, out))
    for i in (2, 0, 1, 1, 0):
        graph, q, s, n, _, out = steps[i]
        out.zero_()
        graph.replay()
        assert_near(out, cache, table, q, s.tolist(), n.tolist(), 0.125)
    plan.check()
    _, q, s, n, at, out = steps[2]
    plan.update(s, n, at)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan.attend(0, q, table, 0.125, out=out)
    graph.replay()
    assert_near(out, cache, table, q, s.tolist(), n.tolist(), 0.125)
    plan.check()
    steps[1][0].replay()
    graph.replay()
    assert not out.any()
    with pytest.raises(RuntimeError, match="error status"):
        plan.check()


def test_lengths_beyond_any_cache_are_reported():
    cache, table = filled([40], 1, 64, 4)
    q = torch.randn(1, 2, 64, device=DEV).to(torch.bfloat16)
    plan = QuantAttention(cache, 2, 4)
    plan.update(_i32([0]), _i32([2 ** 31 - 1]))
    assert not plan.attend(0, q, table, 0.1).any()
    with pytest.raises(RuntimeError, match="error status"):
        plan.check()
    plan.update(_i32([0]), _i32([-5]))
    assert not plan.attend(0, q, table, 0.1).any()
    plan.check()


def test_places_beyond_32_bits():
    """Pages whose bytes lie more than 2^32 into a layer."""
    dim, heads, page = 256, 2, 256
    cache = QuantCache(1, 20000, heads, dim, bits=8, page_size=page)
    assert cache.page_bytes * 15500 > 2 ** 32
    n = 300
    table = _i32([[19999, 15500], [3, 19998]])
    slots, pos = places_of([n, n])
    k, v = rows_of(2 * n, heads, dim, torch.bfloat16, 1), rows_of(2 * n, heads, dim, torch.bfloat16, 2)
    cache.write(0, k, v, table, slots, pos)
    for x, y in zip((k, v), cache.read(0, table, slots, pos, dtype=torch.float32)):
        want = quantised(x, 8)[0]
        assert np.all(np.abs(y.double().cpu().numpy() - want) <= 2.0 ** -24 * np.abs(want))
    check_attention(cache, table, 8, [0, 1], [n, n])
    q = torch.randn(20, 8, dim, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(torch.bfloat16)
    got = run_rows(cache, table, q, [0] * 10 + [1] * 10, [n] * 20, [0, 10, 20], 0.06)
    assert_near(got, cache, table, q, [0] * 10 + [1] * 10, [n] * 20, 0.06)


@pytest.mark.parametrize("bits", [4, 8])
def test_outputs_near_zero_of_long_sequences(bits):
    """V around zero: what is left of a long sum of numbers that are not negative has the precision of an f16 output.

    320 rows of one sequence give a warp some 90 stages.  The 32-bit sums may take a quarter of the rounding's norm:
    16 additions of 2^-23 each between two sums near zero, times the 2^7 by which 20 000 keys' numbers exceed what is
    left, are 2^-12, a third of them in the root mean square, spread over ten such stretches of either sign."""
    n, dim, rows = 20000, 64, 320
    table, pages = table_of([n], 16)
    at, pos = places_of([n])
    g = torch.Generator(device=DEV).manual_seed(7)
    cache = QuantCache(1, pages, 1, dim, bits=bits)
    cache.write(0, torch.randn(n, 1, dim, generator=g, device=DEV).half(), torch.randn(n, 1, dim, generator=g, device=DEV).half(), table, at, pos)
    q = torch.randn(rows, 8, dim, generator=g, device=DEV).half()
    plan = QuantAttention(cache, 8, rows)
    plan.update(_i32([0] * rows), _i32([n] * rows))
    got = plan.attend(0, q, table, 0.125).view(rows, 8, dim).double()
    plan.check()
    k, v = (x[:, 0].double() for x in cache.read(0, table, at, pos, dtype=torch.float32))
    want = torch.softmax(q.double() @ k.T * 0.125, -1) @ v
    assert float((got - want).norm()) <= 1.25 * float((want.half().double() - want).norm())
