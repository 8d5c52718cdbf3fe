"""Cases of the operators that serve many continuations of shared prompts: what one pass of
each computes, from which inputs, and in plain torch operations.

* ``attention``: one decode or verify step's gated grouped-query attention over a paged cache
  whose sequences share leading pages (the shared pages are read once for all their rows).
* ``fork``: new sequences that share their prompt's whole pages, copy its last partial page
  and are grown by the rows of the next step.
* ``reclaim``: dropped sequences give their pages back, others are cut to their accepted
  length, and the live pages move to the front of the pool.
* ``probs``: logits to probabilities under per-row temperature and top-k.
* ``verify``: drafted tokens accepted or replaced against the target's probabilities, from
  given uniform numbers, in fixed-point arithmetic (so the tokens have one right value).

With ``own`` false, ``run`` is the plain form; with ``own`` true it calls zstep_b200.
"""

import random

import numpy as np
import torch

own = False

PAGE = 16     # tokens of a cache page
DIM = 256     # head dimension of the paged attention
FIX = 2.0 ** 38   # fixed-point scale of a probability
UBITS = 24        # bits of a uniform number


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # Four samples of one prompt of about a thousand tokens: a lone request, latency counts.
        dict(name="attention_4_samples", op="attention", q_heads=16, kv_heads=2, groups=1, fan=4, rows=1, prefix=64,
             suffix=40, shape=1),
        # 128 requests over 8 distinct 2048-token prefixes with 256-token suffixes and what
        # they have generated so far: a decode step.
        dict(name="attention_8_prefixes", op="attention", q_heads=16, kv_heads=2, groups=8, fan=16, rows=1, prefix=128,
             suffix=384, shape=2),
        # The same requests in a verify step: the last token and three drafts of each.
        dict(name="attention_8_prefixes_verify", op="attention", q_heads=16, kv_heads=2, groups=8, fan=16, rows=4,
             prefix=128, suffix=384, shape=3),
        # Many questions about one long document, on one rank of two.
        dict(name="attention_long_document", op="attention", q_heads=8, kv_heads=1, groups=1, fan=96, rows=1,
             prefix=2047, suffix=601, shape=4),
        # Four samples of one prompt, with every attention layer's K and V.
        dict(name="fork_4_samples", op="fork", layers=10, kv_heads=2, pages=512, prompts=1, samples=4, tokens=1000,
             share=1.0, append=4, shape=5),
        # Eight samples of each of 32 prompts on one rank of two; the last quarter of a prompt
        # is copied, not shared (the samples edit it).
        dict(name="fork_32_prompts", op="fork", layers=10, kv_heads=1, pages=4096, prompts=32, samples=8, tokens=640,
             share=0.75, append=4, shape=6),
        # A few sequences of a small pool end.
        dict(name="reclaim_small", op="reclaim", layers=10, kv_heads=2, pages=256, seqs=12, tokens=300, drop=0.3, cut=3,
             shape=7),
        # Half of a full pool's sequences end and the pool is packed.
        dict(name="reclaim_half", op="reclaim", layers=10, kv_heads=1, pages=4096, seqs=96, tokens=1200, drop=0.5,
             cut=40, shape=8),
        # A sampled verify step of two requests with three drafts each.
        dict(name="probs_8_rows", op="probs", rows=8, vocab=248320, top_k=0, shape=9),
        # A decode step's 256 rows, half of them with top-k.
        dict(name="probs_256_rows", op="probs", rows=256, vocab=248320, top_k=50, shape=10),
        # Two requests with three drafts each.
        dict(name="verify_2_requests", op="verify", seqs=2, drafts=3, vocab=248320, draft_probs=True, shape=11),
        # 128 requests with three drafts each.
        dict(name="verify_128_requests", op="verify", seqs=128, drafts=3, vocab=248320, draft_probs=True, shape=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    """One more case of the listed ones' ranges; no dearer than the largest of its operator."""
    op = rng.choice(["attention", "attention", "attention", "fork", "reclaim", "probs", "verify", "verify"])
    most = {k: max(work(c)[k] for c in listed() if c["op"] == op) for k in ("bytes", "flops")}
    while True:
        shape = rng.randrange(100, 1 << 30)
        if op == "attention":
            hq, hkv = rng.choice([(16, 2), (16, 2), (8, 1), (4, 1), (2, 1)])
            case = dict(op=op, q_heads=hq, kv_heads=hkv, groups=_log(rng, 1, 32), fan=_log(rng, 1, 96),
                        rows=rng.choice([1, 1, 2, 4]), prefix=_log(rng, 4, 2047), suffix=_log(rng, 5, 700), shape=shape)
        elif op == "fork":
            case = dict(op=op, layers=rng.randint(1, 10), kv_heads=rng.choice([1, 2]), pages=_log(rng, 300, 4096),
                        prompts=_log(rng, 1, 32), samples=rng.randint(1, 8), tokens=_log(rng, 17, 1000),
                        share=rng.choice([1.0, 1.0, 0.75, 0.5]), append=rng.randint(1, 20), shape=shape)
            if _fork_pages(case) > case["pages"] - 1:
                continue
        elif op == "reclaim":
            case = dict(op=op, layers=rng.randint(1, 10), kv_heads=rng.choice([1, 2]), pages=_log(rng, 200, 4096),
                        seqs=_log(rng, 3, 96), tokens=_log(rng, 20, 1200), drop=rng.choice([0.2, 0.35, 0.5]),
                        cut=rng.randint(1, 40), shape=shape)
            if _reclaim_pages(case) > case["pages"] - 1:
                continue
        elif op == "probs":
            case = dict(op=op, rows=_log(rng, 1, 256), vocab=rng.choice([248320, 129280, 124160, 62081]),
                        top_k=rng.choice([0, 1, 7, 50, 1000]), shape=shape)
        else:
            case = dict(op=op, seqs=_log(rng, 1, 128), drafts=rng.randint(1, 7),
                        vocab=rng.choice([248320, 129280, 124160, 62081]), draft_probs=rng.random() < 0.7, shape=shape)
        w = work(case)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and (op != "verify" or case["seqs"] * (case["drafts"] + 1) <= 512):
            return case


# ------------------------------------------------------------------------------- case sizes
def _pages(tokens):
    return -(-tokens // PAGE)


def _attention_shape(c):
    """Per group its prefix pages; per sequence its group and its length in tokens."""
    r = random.Random(c["shape"])
    prefix = [c["prefix"] - (r.randrange(c["prefix"] // 8 + 1) if g else 0) for g in range(c["groups"])]
    seqs = []
    for g in range(c["groups"]):
        fan = c["fan"] if g == 0 else max(1, c["fan"] - r.randrange(c["fan"] // 4 + 1))
        low = c["rows"]
        seqs += [(g, prefix[g] * PAGE + r.randint(low, max(low, c["suffix"]))) for _ in range(fan)]
    r.shuffle(seqs)
    return prefix, seqs


def _fork_shape(c):
    r = random.Random(c["shape"])
    lens = [r.randint(max(1, c["tokens"] // 2), c["tokens"]) for _ in range(c["prompts"])]
    share = [int(n * c["share"]) for n in lens]
    return lens, share


def _fork_pages(c):
    """Pages in use after the pass."""
    lens, share = _fork_shape(c)
    return sum(_pages(n) + c["samples"] * (_pages(n + c["append"]) - s // PAGE) for n, s in zip(lens, share))


def _reclaim_shape(c):
    """Lengths; for every third sequence the pages that it shares with the one before; which
    sequences end; to what length the others are cut."""
    r = random.Random(c["shape"])
    lens = [r.randint(1, c["tokens"]) for _ in range(c["seqs"])]
    shared = [min(lens[i], lens[i - 1]) // PAGE // 2 if i % 3 == 2 else 0 for i in range(c["seqs"])]
    drop = sorted(r.sample(range(c["seqs"]), max(1, int(c["seqs"] * c["drop"]))))
    cut = {i: max(1, lens[i] - r.randrange(c["cut"] + 1)) for i in range(c["seqs"]) if i not in drop}
    return lens, shared, drop, cut


def _reclaim_pages(c):
    lens, shared, _, _ = _reclaim_shape(c)
    return sum(_pages(n) for n in lens) - sum(shared)


def work(c):
    if c["op"] == "attention":
        prefix, seqs = _attention_shape(c)
        kv = sum(prefix) * PAGE + sum(n - prefix[g] * PAGE for g, n in seqs)
        rows = len(seqs) * c["rows"]
        keys = sum(n - j for _, n in seqs for j in range(c["rows"]))
        return {"bytes": kv * c["kv_heads"] * DIM * 4 + 3 * rows * c["q_heads"] * DIM * 2 + 8 * rows + 4 * sum(prefix),
                "flops": 4 * DIM * c["q_heads"] * keys}
    page = 2 * c.get("layers", 0) * c.get("kv_heads", 0) * PAGE * DIM * 2   # bytes of one page, every layer's K and V
    if c["op"] == "fork":
        lens, share = _fork_shape(c)
        copied = sum(c["samples"] * (_pages(n) - s // PAGE) for n, s in zip(lens, share))
        entries = sum(c["samples"] * _pages(n + c["append"]) for n in lens)
        return {"bytes": 2 * copied * page + 16 * entries + c["pages"] // 8, "flops": entries}
    if c["op"] == "reclaim":
        plan = _reclaim_plan(c)
        return {"bytes": 2 * plan["moves"] * page + 8 * plan["entries"] + c["pages"] // 4, "flops": plan["entries"]}
    if c["op"] == "probs":
        return {"bytes": 8 * c["rows"] * c["vocab"], "flops": 4 * c["rows"] * c["vocab"]}
    # About seven drafts in ten are accepted; a sequence whose drafts all are needs no draft probabilities.
    rejected = (1 - 0.7 ** c["drafts"]) if c["draft_probs"] else 0.0
    return {"bytes": int(c["seqs"] * c["vocab"] * 4 * (1 + rejected)), "flops": 4 * c["seqs"] * c["vocab"]}


def _reclaim_plan(c):
    """The pool's tables before the pass (page ids spread at random) and how many pages the pass moves."""
    lens, shared, drop, cut = _reclaim_shape(c)
    r = random.Random(c["shape"] + 1)
    ids = list(range(1, c["pages"]))
    r.shuffle(ids)
    table, at = [], 0
    for i, n in enumerate(lens):
        k = _pages(n) - shared[i]
        table.append((table[i - 1][:shared[i]] if shared[i] else []) + ids[at:at + k])
        at += k
    live = {0}
    for i, n in cut.items():
        live.update(table[i][:_pages(n)])
    return dict(table=table, moves=sum(p >= len(live) for p in live), entries=sum(len(t) for t in table))


# ----------------------------------------------------------------------------------- inputs
def _padded(lists, width, dev):
    a = np.zeros((len(lists), max(1, width)), dtype=np.int32)
    for i, x in enumerate(lists):
        a[i, :len(x)] = x
    return torch.from_numpy(a).to(dev)


def _ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    host = random.Random(seed)
    return {"attention": _prepare_attention, "fork": _prepare_fork, "reclaim": _prepare_reclaim,
            "probs": _prepare_probs, "verify": _prepare_verify}[case["op"]](case, dev, gen, host)


def _normal(gen, dev, *shape, scale=1.0):
    return (torch.randn(*shape, generator=gen, device=dev) * scale).to(torch.bfloat16)


def _prepare_attention(c, dev, gen, host):
    prefix, seqs = _attention_shape(c)
    R, hq, hkv = c["rows"], c["q_heads"], c["kv_heads"]
    rows = len(seqs) * R
    own_pages = [_pages(n) - prefix[g] for g, n in seqs]
    ids = list(range(1, 1 + sum(prefix) + sum(own_pages)))   # page 0 is the padding page
    host.shuffle(ids)
    take = iter(ids)
    shared = [[next(take) for _ in range(p)] for p in prefix]
    tail = [[next(take) for _ in range(p)] for p in own_pages]
    table = [shared[g] + t for (g, _), t in zip(seqs, tail)]
    st = dict(op="attention", hq=hq, hkv=hkv, scale=DIM ** -0.5,
              q=_normal(gen, dev, rows, hq, DIM), gate=_normal(gen, dev, rows, hq, DIM),
              k_cache=_normal(gen, dev, len(ids) + 1, hkv, PAGE, DIM), v_cache=_normal(gen, dev, len(ids) + 1, hkv, PAGE, DIM),
              page_table=_padded(table, max(len(t) for t in table), dev),
              slots=_ints([s for s in range(len(seqs)) for _ in range(R)], dev),
              seq_lens=_ints([n - R + 1 + j for _, n in seqs for j in range(R)], dev))
    members = [[s * R + j for s, (q, _) in enumerate(seqs) if q == g for j in range(R)] for g in range(len(prefix))]
    if own:
        from zstep_b200.ops.shared_prefix import SharedPrefixPlan

        st["plan"] = SharedPrefixPlan.from_prefixes(st["slots"].tolist(), list(zip(members, prefix)), hq, hkv, device=dev)
        st["out"] = torch.empty(rows, hq * DIM, dtype=torch.bfloat16, device=dev)
    else:
        wide = max(len(m) for m in members)
        where = {r: (g, i) for g, m in enumerate(members) for i, r in enumerate(m)}
        at = torch.tensor([where[r] for r in range(rows)], device=dev)
        st.update(R=R, prefix_pages=_padded(shared, max(prefix), dev).long(), prefix_len=_ints([p * PAGE for p in prefix], dev),
                  tail_pages=_padded(tail, max(own_pages), dev).long(), row_group=at[:, 0], row_place=at[:, 1],
                  group_rows=_padded(members, wide, dev).long(), perm=_block_order(dev))
    return st


def _block_order(dev):
    """Where element (token r, dim d) of a (page, head) block is stored: halves of 8 tokens, chunks of
    64 dims, and in a chunk the 16-byte pieces of token r at piece ^ (r % 8)."""
    r = torch.arange(PAGE, device=dev).view(-1, 1)
    d = torch.arange(DIM, device=dev).view(1, -1)
    return ((r // 8) * 2048 + (d // 64) * 512 + (r % 8) * 64 + (((d % 64) // 8) ^ (r % 8)) * 8 + d % 8).reshape(-1)


def _pool_inputs(c, dev, gen, table, lens, slots):
    width = max(len(t) for t in table) + _pages(c.get("append", 0)) + 1
    table = _padded(table + [[]] * (slots - len(table)), width, dev)
    seq_len = _ints(lens + [0] * (slots - len(lens)), dev)
    ref = torch.zeros(c["pages"], dtype=torch.int32, device=dev)
    used = torch.arange(width, device=dev)[None, :] < ((seq_len + PAGE - 1) // PAGE)[:, None]
    ref.index_add_(0, table[used].long(), torch.ones_like(table[used]))
    ref[0] += 1   # page 0 is the padding page
    shape = (c["layers"], c["pages"], c["kv_heads"], PAGE, DIM)
    st = dict(op=c["op"], caches=[_normal(gen, dev, *shape), _normal(gen, dev, *shape)])
    if own:
        from zstep_b200.ops.pages import PagePool

        st["pool"] = PagePool(st["caches"], slots, width, page_size=PAGE)
        st["pool"].adopt(seq_len, table)
        st["start"] = st["pool"].state.clone()
    else:
        st["start"] = (ref, seq_len, table)
        st["live"] = tuple(torch.empty_like(t) for t in st["start"])
    return st


def _prepare_fork(c, dev, gen, host):
    lens, share = _fork_shape(c)
    ids = list(range(1, c["pages"]))
    host.shuffle(ids)
    take = iter(ids)
    table = [[next(take) for _ in range(_pages(n))] for n in lens]
    n = c["prompts"] * c["samples"]
    st = _pool_inputs(c, dev, gen, table, lens, c["prompts"] + n)
    parent = [i for i in range(c["prompts"]) for _ in range(c["samples"])]
    child = list(range(c["prompts"], c["prompts"] + n))
    host.shuffle(child)
    st.update(parents=_ints(parent, dev), children=_ints(child, dev), share=_ints([share[p] for p in parent], dev),
              grown=_ints([lens[p] + c["append"] for p in parent], dev))
    return st


def _prepare_reclaim(c, dev, gen, host):
    lens, _, drop, cut = _reclaim_shape(c)
    st = _pool_inputs(c, dev, gen, _reclaim_plan(c)["table"], lens, c["seqs"])
    host.shuffle(drop)
    st.update(drop=_ints(drop, dev), cut=_ints(list(cut), dev), cut_len=_ints(list(cut.values()), dev))
    return st


def _prepare_probs(c, dev, gen, host):
    rows = c["rows"]
    logits = torch.randn(rows, c["vocab"], generator=gen, device=dev) * 4.0
    temp = [0.0 if host.random() < 0.1 else round(host.uniform(0.5, 1.3), 3) for _ in range(rows)]
    top_k = [c["top_k"] if host.random() < 0.5 else 0 for _ in range(rows)]
    st = dict(op="probs", logits=logits, temperature=torch.tensor(temp, device=dev), top_k=_ints(top_k, dev))
    if own:
        st["out"] = torch.empty_like(logits)
    return st


def _prepare_verify(c, dev, gen, host):
    n, k, vocab = c["seqs"], c["drafts"], c["vocab"]
    base = torch.randn(n, k + 1, vocab, generator=gen, device=dev) * 4.0
    target = torch.softmax(base, dim=-1)
    q = base[:, :k].add_(torch.randn(n, k, vocab, generator=gen, device=dev), alpha=0.6)
    q = torch.softmax(q, dim=-1)
    # Drafts are the draft distribution's own samples, or its likeliest tokens when it gives no probabilities.
    noise = torch.empty(n, k, vocab, device=dev).exponential_(generator=gen)
    drafts = (q / noise if c["draft_probs"] else q).argmax(-1).int()
    count = [k if host.random() < 0.8 else host.randint(0, k) for _ in range(n)]
    st = dict(op="verify", target=target.contiguous(), drafts=drafts, counts=_ints(count, dev),
              draft_probs=q.contiguous() if c["draft_probs"] else None,
              uniform=torch.rand(n, k + 1, generator=gen, device=dev))
    if own:
        from zstep_b200.ops.spec_sampling import DraftVerifier

        st["verifier"] = DraftVerifier(n, k, vocab, device=dev)
    return st


# --------------------------------------------------------------------------------- one pass
def run(st):
    if own:
        return _OWN[st["op"]](st)
    return _PLAIN[st["op"]](st)


def _own_attention(st):
    plan = st["plan"]
    plan.update(st["seq_lens"])
    return plan.attend(st["q"], st["gate"], st["k_cache"], st["v_cache"], st["page_table"], st["seq_lens"], st["scale"],
                       out=st["out"])


def _own_fork(st):
    pool = st["pool"]
    pool.state.copy_(st["start"])
    pool.fork(st["parents"], st["children"], st["share"])
    pool.extend(st["children"], st["grown"])
    return pool.refcount, pool.seq_len, pool.page_table, *st["caches"]


def _own_reclaim(st):
    pool = st["pool"]
    pool.state.copy_(st["start"])
    pool.free(st["drop"])
    pool.truncate(st["cut"], st["cut_len"])
    pool.compact()
    return pool.refcount, pool.seq_len, pool.page_table, *st["caches"]


def _own_probs(st):
    from zstep_b200.ops.spec_sampling import token_probs

    return token_probs(st["logits"], st["temperature"], top_k=st["top_k"], out=st["out"])


def _own_verify(st):
    return st["verifier"].verify(st["target"], st["drafts"], st["uniform"], draft_probs=st["draft_probs"], counts=st["counts"])


_OWN = dict(attention=_own_attention, fork=_own_fork, reclaim=_own_reclaim, probs=_own_probs, verify=_own_verify)


# ------------------------------------------------------------------------------ plain forms
def _tokens(cache, pages, perm):
    """[b, p] page ids -> [b, p * 16, heads, 256] in 32 bits."""
    x = cache[pages].flatten(-2)[..., perm].float()
    b, p, h, _ = x.shape
    return x.view(b, p, h, PAGE, DIM).transpose(2, 3).reshape(b, p * PAGE, h, DIM)


def _plain_attention(st):
    rows, hq, hkv, R = st["q"].shape[0], st["hq"], st["hkv"], st["R"]
    q = st["q"].float().view(rows, hkv, hq // hkv, DIM)
    k1, v1 = (_tokens(st[n], st["prefix_pages"], st["perm"]) for n in ("k_cache", "v_cache"))
    k2, v2 = (_tokens(st[n], st["tail_pages"], st["perm"]) for n in ("k_cache", "v_cache"))
    lens, first = st["seq_lens"], st["prefix_len"][st["row_group"]]
    s1 = torch.einsum("gmhnd,gthd->gmhnt", q[st["group_rows"]], k1)[st["row_group"], st["row_place"]] * st["scale"]
    s2 = torch.einsum("srhnd,sthd->srhnt", q.view(-1, R, hkv, hq // hkv, DIM), k2).flatten(0, 1) * st["scale"]
    t1, t2 = s1.shape[-1], s2.shape[-1]
    seen1 = torch.arange(t1, device=q.device)[None, :] < torch.minimum(lens, first)[:, None]
    seen2 = torch.arange(t2, device=q.device)[None, :] < (lens - first)[:, None]
    s = torch.cat([s1.masked_fill_(~seen1[:, None, None, :], float("-inf")),
                   s2.masked_fill_(~seen2[:, None, None, :], float("-inf"))], -1)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o1 = torch.einsum("gmhnt,gthd->gmhnd", p[st["group_rows"]][..., :t1], v1)[st["row_group"], st["row_place"]]
    o2 = torch.einsum("srhnt,sthd->srhnd", p[..., t1:].reshape(-1, R, hkv, hq // hkv, t2), v2).flatten(0, 1)
    o = (o1 + o2).reshape(rows, hq, DIM) * torch.sigmoid(st["gate"].float())
    return o.reshape(rows, hq * DIM).to(torch.bfloat16)


def _restore(st):
    for a, b in zip(st["live"], st["start"]):
        a.copy_(b)
    return st["live"]


def _take_free(ref, need):
    """need [n, w] marks the table entries that want a page: they get the lowest free ids in order."""
    free = torch.sort((ref > 0).int(), stable=True).indices.int()
    rank = torch.cumsum(need.flatten().long(), 0) - 1
    return torch.where(need.flatten(), free[rank.clamp(min=0)], 0).view_as(need).int()


def _plain_fork(st):
    ref, seq_len, table = _restore(st)
    par, chi, grown = st["parents"].long(), st["children"].long(), st["grown"]
    at = torch.arange(table.shape[1], device=table.device)[None, :]
    n = seq_len[par]
    whole = (torch.minimum(n, st["share"]) // PAGE)[:, None]
    used = ((n + PAGE - 1) // PAGE)[:, None]
    need = (at >= whole) & (at < used)
    fresh = _take_free(ref, need)
    new = torch.where(at < whole, table[par], fresh)
    table[chi] = new
    seq_len[chi] = n
    ref.index_add_(0, new[at < used].long(), torch.ones_like(new[at < used]))
    src, dst = table[par][need].long(), fresh[need].long()
    st["caches"][0][:, dst] = st["caches"][0][:, src]
    st["caches"][1][:, dst] = st["caches"][1][:, src]
    need = (at >= used) & (at < ((grown + PAGE - 1) // PAGE)[:, None])   # the grown rows' pages
    fresh = _take_free(ref, need)
    table[chi] = torch.where(need, fresh, new)
    seq_len[chi] = grown
    ref.index_add_(0, fresh[need].long(), torch.ones_like(fresh[need]))
    return ref, seq_len, table, *st["caches"]


def _plain_reclaim(st):
    ref, seq_len, table = _restore(st)
    at = torch.arange(table.shape[1], device=table.device)[None, :]
    slots = torch.cat([st["drop"], st["cut"]]).long()
    left = torch.cat([torch.zeros_like(st["drop"]), st["cut_len"]])
    gone = (at >= ((left + PAGE - 1) // PAGE)[:, None]) & (at < ((seq_len[slots] + PAGE - 1) // PAGE)[:, None])
    was = table[slots]
    ref.index_add_(0, was[gone].long(), -torch.ones_like(was[gone]))
    table[slots] = torch.where(gone, 0, was)
    seq_len[slots] = left
    live = ref > 0
    count = live.sum()
    ids = torch.arange(ref.numel(), device=ref.device)
    src = torch.nonzero(live & (ids >= count)).flatten()
    dst = torch.nonzero(~live & (ids < count)).flatten()
    st["caches"][0][:, dst] = st["caches"][0][:, src]
    st["caches"][1][:, dst] = st["caches"][1][:, src]
    to = ids.int()
    to[src] = dst.int()
    table.copy_(to[table.long()])
    ref[dst] = ref[src]
    ref[src] = 0
    return ref, seq_len, table, *st["caches"]


def _plain_probs(st):
    x, temp, top_k = st["logits"], st["temperature"][:, None], st["top_k"][:, None].long()
    kth = torch.sort(x, dim=-1, descending=True).values.gather(1, (top_k - 1).clamp(min=0))
    keep = (x >= kth) | (top_k <= 0)
    top = x.amax(-1, keepdim=True)
    p = torch.where(keep, torch.exp((x - top) / torch.where(temp > 0, temp, 1.0)), 0.0)
    p = p / p.sum(-1, keepdim=True)
    best = x == top
    best = best & (torch.cumsum(best.int(), -1) == 1)
    return torch.where(temp > 0, p, best.float())


def _fixed(p):
    return (torch.nan_to_num(p.float(), nan=0.0).clamp(0.0, 1.0) * FIX).long()


def _plain_verify(st):
    p, d, q = st["target"], st["drafts"].long(), st["draft_probs"]
    n, k = d.shape
    u = (st["uniform"] * 2.0 ** UBITS).long()
    pd = _fixed(p[:, :k].gather(2, d[..., None])[..., 0])
    qd = torch.full_like(pd, int(FIX)) if q is None else _fixed(q.gather(2, d[..., None])[..., 0])
    at = torch.arange(k, device=d.device)[None, :]
    ok = (u[:, :k] * qd < (pd << UBITS)) & (at < st["counts"][:, None])
    taken = torch.cumprod(ok.long(), 1).sum(1)
    seq = torch.arange(n, device=d.device)
    last = taken.clamp(max=k - 1)
    w = _fixed(p[seq, taken])
    if q is None:
        less = torch.zeros_like(w).scatter_(1, d[seq, last][:, None], int(FIX))
    else:
        less = _fixed(q[seq, last])
    rest = (w - less).clamp(min=0)
    rest = torch.where((taken < st["counts"])[:, None] & (rest.sum(1, keepdim=True) > 0), rest, w)
    run_ = torch.cumsum(rest, 1)
    total, un = run_[:, -1], u[:, k]
    goal = un * (total >> UBITS) + ((un * (total & ((1 << UBITS) - 1))) >> UBITS)
    token = (run_ <= goal[:, None]).sum(1)
    out = torch.cat([d, torch.zeros_like(d[:, :1])], 1)
    at = torch.arange(k + 1, device=d.device)[None, :]
    out = torch.where(at < taken[:, None], out, torch.where(at == taken[:, None], token[:, None], -1))
    return torch.cat([taken[:, None] + 1, out], 1).int()


_PLAIN = dict(attention=_plain_attention, fork=_plain_fork, reclaim=_plain_reclaim, probs=_plain_probs, verify=_plain_verify)


# --------------------------------------------------------------------------- 64-bit results
def exact(case, seed):
    st = prepare(case, seed)
    return {"attention": _exact_attention, "fork": _exact_fork, "reclaim": _exact_reclaim, "probs": _exact_probs,
            "verify": _exact_verify}[case["op"]](case, st)


def _exact_attention(c, st):
    """Row by row over the row's own pages, with no notion of a shared prefix."""
    hq, hkv = c["q_heads"], c["kv_heads"]
    table, slots, lens = st["page_table"].long(), st["slots"].tolist(), st["seq_lens"].tolist()
    t = np.arange(PAGE * DIM)
    r, d = t // DIM, t % DIM
    flat = torch.from_numpy((r >> 3 << 11) + (d >> 6 << 9) + ((r & 7) << 6) + (((d >> 3 & 7) ^ (r & 7)) << 3) + (d & 7)).to(table.device)
    out = torch.empty(len(lens), hq, DIM, dtype=torch.float64, device=table.device)
    held = (-1, None, None)
    for i, (s, n) in enumerate(zip(slots, lens)):
        if held[0] != s:
            most = max(m for q, m in zip(slots, lens) if q == s)
            pages = table[s, :_pages(most)]
            k, v = (st[x][pages].reshape(len(pages), hkv, -1)[:, :, flat].view(-1, hkv, PAGE, DIM).double().permute(1, 0, 2, 3)
                    .reshape(hkv, -1, DIM) for x in ("k_cache", "v_cache"))
            held = (s, k, v)
        _, k, v = held
        a = torch.bmm(st["q"][i].double().view(hkv, -1, DIM), k[:, :n].transpose(1, 2)) * DIM ** -0.5
        a = torch.exp(a - torch.logsumexp(a, -1, keepdim=True))
        out[i] = torch.bmm(a, v[:, :n]).reshape(hq, DIM)
    return (out / (1 + torch.exp(-st["gate"].double()))).reshape(len(lens), hq * DIM)


def _tables(st):
    """The pool's integers before the pass, as lists."""
    if own:
        pool = st["pool"]
        pool.state.copy_(st["start"])
        return pool.refcount.tolist(), pool.seq_len.tolist(), pool.page_table.tolist()
    return tuple(t.tolist() for t in st["start"])


def _finish(st, ref, lens, table, moves):
    dev = st["caches"][0].device
    for src, dst in moves:
        for x in st["caches"]:
            x[:, dst] = x[:, src]
    return (*(torch.tensor(v, dtype=torch.int32, device=dev) for v in (ref, lens, table)), *(x.double() for x in st["caches"]))


def _exact_fork(c, st):
    ref, lens, table = _tables(st)
    moves = []

    def fresh():
        p = ref.index(0)
        ref[p] = 1
        return p

    for p, ch, share in zip(st["parents"].tolist(), st["children"].tolist(), st["share"].tolist()):
        lens[ch] = lens[p]
        for j in range(_pages(lens[p])):
            src = table[p][j]
            if (j + 1) * PAGE <= min(share, lens[p]):
                table[ch][j] = src
                ref[src] += 1
            else:
                table[ch][j] = fresh()
                moves.append((src, table[ch][j]))
    for ch, n in zip(st["children"].tolist(), st["grown"].tolist()):
        for j in range(_pages(lens[ch]), _pages(n)):
            table[ch][j] = fresh()
        lens[ch] = n
    return _finish(st, ref, lens, table, moves)


def _exact_reclaim(c, st):
    ref, lens, table = _tables(st)
    ends = [(s, 0) for s in st["drop"].tolist()] + list(zip(st["cut"].tolist(), st["cut_len"].tolist()))
    for s, n in ends:
        for j in range(_pages(n), _pages(lens[s])):
            ref[table[s][j]] -= 1
            table[s][j] = 0
        lens[s] = n
    live = [p for p in range(len(ref)) if ref[p] > 0]
    holes = [p for p in range(len(live)) if ref[p] == 0]
    moves = list(zip([p for p in live if p >= len(live)], holes))
    to = dict(moves)
    table = [[to.get(p, p) for p in row] for row in table]
    for a, b in moves:
        ref[b], ref[a] = ref[a], 0
    return _finish(st, ref, lens, table, moves)


def _exact_probs(c, st):
    out = torch.zeros(st["logits"].shape, dtype=torch.float64, device=st["logits"].device)
    for i, (x, temp, k) in enumerate(zip(st["logits"], st["temperature"].tolist(), st["top_k"].tolist())):
        if temp <= 0:
            out[i, int(torch.nonzero(x == x.max())[0])] = 1.0
            continue
        z = x.double() / float(np.float32(temp))
        if k:
            z = z.masked_fill(x < torch.topk(x, k).values[-1], float("-inf"))
        out[i] = torch.exp(z - torch.logsumexp(z, 0))
    return out


def _exact_verify(c, st):
    """Whole numbers held in float64 (all below 2^53), the products in Python's integers."""
    fix = lambda x: torch.floor(x.double().clamp(0, 1) * FIX)  # noqa: E731
    out = []
    for i, m in enumerate(st["counts"].tolist()):
        d, u = st["drafts"][i].tolist(), [int(v * 2 ** UBITS) for v in st["uniform"][i].double().tolist()]
        j = 0
        while j < m:
            q = 2 ** 38 if st["draft_probs"] is None else int(fix(st["draft_probs"][i, j, d[j]]).item())
            if not u[j] * q < int(fix(st["target"][i, j, d[j]]).item()) * 2 ** UBITS:
                break
            j += 1
        w = p = fix(st["target"][i, j])
        if j < m:
            if st["draft_probs"] is None:
                w = p.clone()
                w[d[j]] = 0
            else:
                w = (p - fix(st["draft_probs"][i, j])).clamp(min=0)
            w = w if w.sum().item() else p
        acc = torch.cumsum(w, 0)
        goal = u[-1] * int(acc[-1].item()) >> UBITS
        token = int(torch.searchsorted(acc, torch.tensor([float(goal)], dtype=torch.float64, device=acc.device), right=True).item())
        out.append([j + 1] + d[:j] + [token] + [-1] * (len(d) - j))
    return torch.tensor(out, dtype=torch.int32, device=st["target"].device)
