"""Token probabilities and draft verification against 64-bit and whole-number references."""

import math
from fractions import Fraction

import pytest
import torch

from zstep_b200.ops.spec_sampling import DraftVerifier, token_probs

gpu = pytest.mark.gpu


# ------------------------------------------------------------------------------ probabilities
def want_probs(x, temp, k=0, p=1.0):
    """64 bits; also the tokens whose place in the kept set 32-bit sums may decide either way."""
    x = torch.where(torch.isnan(x), -math.inf, x.double()).clamp(max=3.4028234663852886e38)
    out = torch.zeros_like(x)
    unsure = torch.zeros_like(x, dtype=torch.bool)
    if x.max() == -math.inf:
        return out, unsure
    if temp <= 0:
        out[int((x == x.max()).nonzero()[0])] = 1
        return out, unsure
    keep = torch.ones_like(x, dtype=torch.bool)
    if 0 < k < x.numel():
        keep = x >= torch.sort(x, descending=True).values[k - 1]
    e = torch.where(keep, torch.exp((x - x.max()) / temp), 0.0)
    if p < 1:
        # kept: tokens whose larger ones hold less than p of the mass; the mass before a token is
        # known to 1e-5 of the whole.
        vals, idx = torch.sort(x.masked_fill(~keep, -math.inf), descending=True)
        before = torch.cumsum(e[idx], 0) - e[idx]
        first = torch.searchsorted(-vals, -vals, right=False)   # the first of equal values
        before = before[first] / e.sum()
        unsure[idx[(before - p).abs() < 1e-5]] = True
        keep[idx[before >= p]] = False
        keep[idx[0]] = True
        keep |= x == x.max()
        e = torch.where(keep, e, 0.0)
    return e / e.sum(), unsure


def check_probs(x, temp, k=None, p=None, out=None):
    rows = x.shape[0]
    f = lambda v, t: None if v is None else torch.tensor(v, dtype=t, device="cuda")  # noqa: E731
    got = token_probs(x.cuda() if out is None else x, f(temp, torch.float32), f(k, torch.int32), f(p, torch.float32), out=out)
    torch.cuda.synchronize()
    got = got.cpu().double()
    for r in range(rows):
        y, unsure = want_probs(x[r].cpu(), temp[r], k[r] if k else 0, p[r] if p else 1.0)
        # exp's argument a = (x - max) / T is rounded three times: |a| 2^-22 of the value; the sum
        # and quotient add 1e-6.  Probabilities below 1e-30 may be flushed.  A token at the
        # nucleus' edge may be on either side, which scales the others by less than 2e-5 + itself.
        arg = (torch.log(y.clamp(min=1e-300)) - torch.log(y.max().clamp(min=1e-300))).abs()
        edge = (2e-5 + float(y[unsure].sum()) if unsure.any() else 0.0)
        tol = y * (arg * 2.0 ** -22 + 2e-6 + edge) + 1e-30
        bad = ((got[r] - y).abs() > tol) & ~unsure
        assert not bad.any(), (r, int(bad.sum()), got[r][bad][:3], y[bad][:3])
    return got


@gpu
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 4097, 62081, 248320])
def test_probs_temperature_and_top_k(vocab):
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(6, vocab, generator=g) * 4
    check_probs(x, [1.0, 0.3, 2.5, 0.0, -1.0, 0.7], [0, 5, vocab, 3, 0, 1])


@gpu
@pytest.mark.parametrize("vocab", [16384, 16385, 65537, 262144, 262145, 300001])
def test_probs_sizes_around_the_clusters(vocab):
    """Vocabularies that fill a CTA, a cluster, or neither; k on either side of the candidate lists."""
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(6, vocab, generator=g) * 4
    check_probs(x, [1.0, 0.8, 0.0, 1.2, 1.0, 0.6], [0, 256, 0, 257, 3000, 40], [1.0, 1.0, 1.0, 1.0, 0.9, 0.7])


@gpu
def test_probs_candidates_in_one_place():
    """The largest logits side by side (all in one CTA's part), equal in hundreds, or rarer than k."""
    x = torch.full((6, 100000), -5.0)
    x[0] = torch.arange(100000).float() / 3000       # ascending: the last CTA holds the top
    x[1, 70000:70400] = 2.0                          # 400 tie for the first place
    x[2, 40000:43000] = 1.0                          # 3000 do
    x[3] = -math.inf
    x[3, [5, 90000, 50000]] = torch.tensor([1.0, 2.0, 3.0])   # fewer than k tokens
    x[4, ::2] = math.nan
    x[5, 10:200] = torch.arange(190) / 10.0
    got = check_probs(x, [1.0, 1.0, 1.0, 1.0, 1.0, 1.0], [200, 50, 50, 50, 50, 256], [1.0, 1.0, 0.5, 1.0, 1.0, 0.95])
    assert int((got[1] > 0).sum()) == 400 and int((got[2] > 0).sum()) == 3000 and int((got[3] > 0).sum()) == 3


@gpu
def test_probs_ties_and_masks():
    x = torch.zeros(9, 777)
    x[0, 300:] = -math.inf
    x[1] = -math.inf                       # nothing left
    x[2] = torch.nan
    x[3, 5], x[3, 9] = math.nan, 3.0
    x[4, [7, 70, 700]] = math.inf          # share the mass
    x[5] = torch.arange(777) // 7          # groups of 7 equal logits: ties with the k-th stay
    x[6, [400, 50]] = 2.0                  # greedy tie: the lowest id
    x[7] = -3.4e38                         # the lowest numbers are not masks
    x[7, 3] = -math.inf
    x[8, :] = 1.0
    got = check_probs(x, [1.0, 1.0, 1.0, 0.5, 1.0, 1.0, 0.0, 1.0, 1e-42], [0, 3, 0, 0, 2, 10, 1, 0, 0])
    assert not got[1].any() and not got[2].any()
    assert int((got[5] > 0).sum()) == 14 and int(got[6].argmax()) == 50


@gpu
@pytest.mark.parametrize("vocab", [50, 5000, 248320])
def test_probs_top_p(vocab):
    g = torch.Generator().manual_seed(vocab)
    x = torch.randn(7, vocab, generator=g) * 3
    check_probs(x, [1.0, 0.5, 1.5, 1.0, 1.0, 0.0, 0.8], [0, 0, 20, 3, 0, 0, 0], [0.9, 0.5, 0.99, 0.7, 0.0, 0.5, 1e-9])


@gpu
@pytest.mark.parametrize("vocab", [700, 30000, 248320])
def test_probs_wide_nuclei_and_large_k(vocab):
    # From peaked rows to flat ones whose nucleus reaches across zero and far below the top's image.
    x = torch.randn(8, vocab, generator=torch.Generator().manual_seed(vocab)) * 4
    x[6] = x[6].abs() * 1e-3
    x[7] -= 200.0
    x[:, 5::11] = -math.inf
    check_probs(x, [1.0, 8.0, 50.0, 1.0, 8.0, 50.0, 2.0, 3.0], [0, 0, 0, 300, 600, 257, 0, 400],
                [0.95, 0.5, 0.999, 1.0, 0.9, 0.3, 0.7, 0.99])


@gpu
def test_probs_top_p_keeps_ties():
    x = torch.zeros(2, 100)
    x[0, :10] = 5.0
    x[1, 3] = 9.0
    got = check_probs(x, [1.0, 1.0], None, [0.05, 0.05])
    assert int((got[0] > 0).sum()) == 10 and got[1, 3] == 1.0


@gpu
@pytest.mark.parametrize("vocab", [90, 248320, 262150])
def test_probs_infinite_temperature_leaves_the_unmasked_alike(vocab):
    x = torch.randn(2, vocab, generator=torch.Generator().manual_seed(2))
    x[:, ::3] = -math.inf
    x[:, 1::7] = math.nan
    kept = x > -math.inf
    for k, p in ((0, 1.0), (0, 0.999999)):
        got = token_probs(x.cuda(), torch.tensor([math.inf, math.inf], device="cuda"),
                          top_k=torch.tensor([k, k], dtype=torch.int32, device="cuda"),
                          top_p=torch.tensor([p, p], device="cuda")).cpu()
        assert not got[~kept].any()
        if p == 1.0:
            # a sum of n ones is within n 2^-24 of it, the quotient within 2^-23
            torch.testing.assert_close(got[kept].double(), (1.0 / kept.sum(1, keepdim=True).double()).expand(-1, vocab)[kept],
                                       rtol=vocab * 2.0 ** -24 + 2.0 ** -22, atol=0)


@gpu
@pytest.mark.parametrize("vocab", [16384, 248320, 262144])
def test_probs_one_value_everywhere_fills_one_bin(vocab):
    x = torch.full((2, vocab), 1.5)
    got = token_probs(x.cuda(), torch.tensor([1.0, 0.5], device="cuda"), top_k=torch.tensor([0, 400], dtype=torch.int32, device="cuda"),
                      top_p=torch.tensor([0.5, 0.9], device="cuda")).cpu().double()
    torch.testing.assert_close(got, torch.full_like(got, 1.0 / vocab), rtol=vocab * 2.0 ** -24 + 2.0 ** -22, atol=0)


@gpu
def test_probs_strided_rows_and_repeats():
    g = torch.Generator(device="cuda").manual_seed(3)
    x = torch.randn(5, 1003, generator=g, device="cuda")[:, 1:999]   # rows that start off 16-byte boundaries
    out = torch.full((5, 1010), 7.0, device="cuda")
    check_probs(x, [1.0] * 5, [0, 4, 0, 50, 0], [0.9, 1.0, 1.0, 0.8, 1.0], out=out[:, 3:1001])
    assert (out[:, :3] == 7).all() and (out[:, 1001:] == 7).all()
    t = torch.ones(5, device="cuda")
    assert torch.equal(token_probs(x, t, top_p=t * 0.8), token_probs(x, t, top_p=t * 0.8))


@gpu
@pytest.mark.parametrize("vocab,k", [(248320, 257), (248320, 300), (62081, 257), (16384, 17), (8192, 50), (2000, 33)])
def test_probs_of_many_rows_repeat_beyond_the_candidate_path(vocab, k):
    """k above 256, or above the warps of a row's CTAs: no candidates, the radix select comes right behind the
    row's maximum.  Every row is the same one and has to give the same bits, launch after launch."""
    x = torch.randn(1, vocab, generator=torch.Generator().manual_seed(k)) * 4
    check_probs(x, [0.9], [k], [0.95])
    rows = 256
    wide = x.cuda().expand(rows, vocab).contiguous()
    t, p = torch.full((rows,), 0.9, device="cuda"), torch.full((rows,), 0.95, device="cuda")
    ks = torch.full((rows,), k, dtype=torch.int32, device="cuda")
    first, out = token_probs(wide, t, ks, p)[0].clone(), torch.empty_like(wide)
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(40):
        wrong += (token_probs(wide, t, ks, p, out=out) != first).sum()
    assert int(wrong) == 0


@gpu
@pytest.mark.parametrize("vocab", [1000, 62081])
def test_probs_of_one_row_under_several_settings(vocab):
    """Rows that are one row in memory (a stride of 0), and rows that overlap."""
    x = torch.randn(vocab + 9, generator=torch.Generator().manual_seed(vocab)).cuda() * 4
    temp, k, p = [0.0, 0.5, 1.0, 2.0], [0, 0, 7, 300], [1.0, 0.9, 1.0, 1.0]
    for rows in (x[:vocab].expand(4, vocab), x.as_strided((4, vocab), (3, 1))):
        check_probs(rows, temp, k, p, out=torch.empty(4, vocab, device="cuda"))


@gpu
def test_probs_refusals():
    x, t = torch.zeros(3, 10, device="cuda"), torch.ones(3, device="cuda")
    for args in ((x.half(), t), (x.t(), t), (x, t[:2]), (x, t, t), (x, t, None, t.int()), (x[0], t), (x.cpu(), t)):
        with pytest.raises(RuntimeError):
            token_probs(*args)
    with pytest.raises(RuntimeError):
        token_probs(x, t, out=torch.zeros(3, 11, device="cuda"))
    assert token_probs(x[:0], t[:0]).shape == (0, 10)


# ------------------------------------------------------------------------------- verification
def fix(p):
    if p != p:
        return 0
    return int(Fraction(min(max(p, 0.0), 1.0)) * 2 ** 38)


def want_record(target, drafts, uniform, q, count):
    """The definition in Python's whole numbers, one sequence."""
    k = len(drafts)
    m = min(max(count, 0), k)
    u = [int(Fraction(min(max(float(x), 0.0), 0.99999994)) * 2 ** 24) for x in uniform]
    j = 0
    while j < m:
        d = drafts[j]
        if not 0 <= d < target.shape[1]:
            break
        qd = 2 ** 38 if q is None else fix(float(q[j, d]))
        if not u[j] * qd < fix(float(target[j, d])) * 2 ** 24:
            break
        j += 1
    p = [fix(x) for x in target[j].tolist()]
    w = p
    if j < m:
        if q is None:
            w = [0 if i == drafts[j] else x for i, x in enumerate(p)]
        else:
            w = [max(0, x - fix(y)) for x, y in zip(p, q[j].tolist())]
        if not any(w):
            w = p
    goal, run, token = u[k] * sum(w) >> 24, 0, 0
    for i, x in enumerate(w):
        run += x
        if run > goal:
            token = i
            break
    return [j + 1] + drafts[:j] + [token] + [-1] * (k - j)


def check_verify(target, drafts, uniform, q=None, counts=None, verifier=None):
    n, k1, vocab = target.shape
    c = lambda t: None if t is None else t.cuda()  # noqa: E731
    v = verifier or DraftVerifier(n, k1 - 1, vocab)
    got = v.verify(c(target), c(drafts), c(uniform), c(q), c(counts)).tolist()
    cnt = counts.tolist() if counts is not None else [k1 - 1] * n
    for s in range(n):
        assert got[s] == want_record(target[s].cpu(), drafts[s].tolist(), uniform[s].tolist(), None if q is None else q[s].cpu(), cnt[s]), s
    return v, got


def random_case(n, k, vocab, seed, with_q=True, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    base = torch.randn(n, k + 1, vocab, generator=g) * spread
    p = torch.softmax(base, -1)
    q = torch.softmax(base[:, :k] + torch.randn(n, k, vocab, generator=g) * 0.7, -1)
    d = torch.multinomial(q.reshape(-1, vocab), 1, generator=g).view(n, k).int() if with_q else q.argmax(-1).int()
    return p, d, torch.rand(n, k + 1, generator=g), q if with_q else None


@gpu
@pytest.mark.parametrize("n,k,vocab,with_q", [(1, 1, 1, True), (1, 1, 2, False), (5, 3, 33, True), (3, 7, 1000, True),
                                              (40, 2, 129, False), (2, 3, 62081, True), (1, 64, 300, True), (3, 1, 248320, True)])
def test_verify_matches_whole_numbers(n, k, vocab, with_q):
    p, d, u, q = random_case(n, k, vocab, n * 31 + vocab, with_q)
    g = torch.Generator().manual_seed(1)
    check_verify(p, d, u, q, torch.randint(0, k + 1, (n,), generator=g).int())
    v, _ = check_verify(p, d, u, q)
    v.check()


@gpu
def test_verify_every_outcome():
    """Numbers at their ends, drafts out of range, tokens the target excludes or the draft never had."""
    p, d, u, q = random_case(12, 3, 50, 5)
    u[0] = 0.0                                # 0 accepts whatever the target allows
    u[1] = 1.0                                # counts as 1 - 2^-24
    u[2] = 0.99999994
    d[3, 0], d[4, 1], d[5, 2] = -1, 50, 2 ** 30
    p[6, 0, d[6, 0]] = 0.0                    # excluded by the target, whatever u
    u[6, 0] = 0.0
    q[7, 0, d[7, 0]] = 0.0                    # never drafted, but the target allows it
    p[8, 1] = q[8, 1]                         # equal distributions: accepted
    p[9, :, :] = 0.0
    p[9, :, 49] = 1.0                         # the last token
    q[10, 0] = p[10, 0]
    q[10, 0, d[10, 0]] = 1.0                  # rejected with a residual that excludes only the draft
    u[10, 0] = 0.99
    p[11, 0], q[11, 0, :] = math.nan, 0.5
    counts = torch.tensor([3, 3, 3, 3, 3, 3, 3, 3, 3, 0, 3, -4], dtype=torch.int32)
    check_verify(p, d, u, q, counts)
    check_verify(p, d, u, None, counts + 9)   # counts past k are k


@gpu
def test_verify_residual_empty_draws_from_the_target():
    """p <= q at every token (masses differ): the residual is empty."""
    p = torch.full((1, 2, 8), 0.05)
    q = torch.full((1, 1, 8), 0.5)
    _, got = check_verify(p, torch.tensor([[3]], dtype=torch.int32), torch.tensor([[0.9, 0.51]]), q)
    assert got == [[1, 4, -1]]


@gpu
def test_verify_reports_rows_without_mass():
    p, d, u, q = random_case(3, 2, 40, 8)
    p[1] = 0.0
    v, got = check_verify(p, d, u, q)
    assert got[1] == [1, 0, -1, -1]
    with pytest.raises(RuntimeError, match="mass"):
        v.check()
    v.check()


@gpu
def test_verify_flat_distribution_hits_every_part():
    """Equal probabilities: the token is floor(u * vocab), wherever its part of the row is."""
    vocab, n = 248320, 64
    p = torch.full((1, 2, vocab), 1 / vocab, device="cuda").expand(n, 2, vocab)   # strides of 0
    u = torch.zeros(n, 2)
    u[:, 1] = (torch.arange(n) + 0.5) / n
    v = DraftVerifier(n, 1, vocab)
    rec = v.verify(p, torch.zeros(n, 1, dtype=torch.int32, device="cuda"), u.cuda(), counts=torch.zeros(n, dtype=torch.int32, device="cuda"))
    w = fix(float(p[0, 0, 0]))
    goal = [int(Fraction(float(x)) * 2 ** 24) * (w * vocab) >> 24 for x in u[:, 1]]
    assert rec[:, 1].tolist() == [g // w for g in goal]


@gpu
def test_verify_keeps_the_target_distribution():
    """Drafts from q, verified against p: the first token is distributed as p (chi-square, 15 degrees
    of freedom: above 45 in 1 of 10^4 seeds)."""
    vocab, n = 16, 40000
    g = torch.Generator(device="cuda").manual_seed(11)
    p1 = torch.softmax(torch.randn(vocab, generator=g, device="cuda") * 1.2, 0)
    q1 = torch.softmax(torch.randn(vocab, generator=g, device="cuda") * 1.2, 0)
    d = torch.multinomial(q1.expand(n, vocab), 1, generator=g).int()
    rec = DraftVerifier(n, 1, vocab).verify(p1.expand(n, 2, vocab), d, torch.rand(n, 2, generator=g, device="cuda"), q1.expand(n, 1, vocab))
    seen = torch.bincount(rec[:, 1].long(), minlength=vocab).double()
    chi = float(((seen - p1.double() * n) ** 2 / (p1.double() * n)).sum())
    assert chi < 45, chi


@gpu
def test_verify_strides_streams_and_graphs():
    p, d, u, q = random_case(4, 3, 501, 21)
    wide_p, wide_q = torch.zeros(4, 4, 640, device="cuda"), torch.zeros(4, 5, 640, device="cuda")
    wide_p[:, :, 7:508], wide_q[:, 1:4, 3:504] = p.cuda(), q.cuda()
    v, got = check_verify(p, d, u, q)
    dc, uc = d.cuda(), u.cuda()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        rec = v.verify(wide_p[:, :, 7:508], dc, uc, wide_q[:, 1:4, 3:504]).clone()
    s.synchronize()
    assert rec.tolist() == got
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = v.verify(wide_p[:, :, 7:508], dc, uc, wide_q[:, 1:4, 3:504])
    for _ in range(3):
        out.zero_()
        gr.replay()
        assert out.tolist() == got
    uc.copy_(1.0 - uc)
    gr.replay()
    assert out.tolist() == [want_record(p[i], d[i].tolist(), uc[i].tolist(), q[i], 3) for i in range(4)]


@gpu
def test_verify_refusals():
    p, d, u, q = (t.cuda() for t in random_case(2, 3, 40, 2))
    v = DraftVerifier(2, 3, 40)
    for args in ((p[:, :3], d, u, q), (p.double(), d, u, q), (p, d.long(), u, q), (p, d[:, :2], u, q), (p, d, u[:, :3], q),
                 (p, d, u, q[:, :2]), (p, d, u, q[..., :39]), (p[..., :39], d, u, q), (torch.cat([p, p]), d, u, q), (p, d.cpu(), u, q),
                 (p, d, u, q, torch.zeros(3, dtype=torch.int32, device="cuda")), (p.transpose(1, 2), d, u, q)):
        with pytest.raises((ValueError, RuntimeError)):
            v.verify(*args)


@pytest.mark.parametrize("n,k,vocab", [(0, 1, 5), (1, 0, 5), (1, 65, 5), (1, 1, 0), (1, 1, (1 << 24) + 1)])
def test_verifier_sizes_that_are_refused(n, k, vocab):
    with pytest.raises(ValueError):
        DraftVerifier(n, k, vocab, device="cpu")
