"""Cases of the operators of a K/V cache held in 4 or 8 bits: what one pass of each computes,
from which inputs, and in plain torch operations.

* ``store``: rows of K and V are quantised into their places of a paged cache, and what the
  cache then holds there is read back.
* ``load``: the values that the cache holds at given places.
* ``attend``: one step's grouped-query attention over the cache, every row up to its own length:
  single tokens, the rows of a verify step, chunks of prompts.

A group of 64 dims of one token and head is held as whole numbers n in 0..N (N = 15 or 255) with
a scale s and an offset z in bf16: z is the group's minimum rounded down, s is (maximum - z) / N
rounded up, n is (x - z) / s rounded to the nearest (ties to even), and the value held is s n + z.

With ``own`` false, ``run`` is the plain form; with ``own`` true it calls zstep_b200.
"""

import random

import numpy as np
import torch

own = False

PAGE = 16     # tokens of a cache page
GROUP = 64    # dims that share a scale and an offset


# ------------------------------------------------------------------------------------ cases
def listed():
    return [
        # A lone request of about a thousand tokens: latency counts.
        dict(name="attend_1_request", op="attend", q_heads=16, kv_heads=2, dim=256, bits=4, half=False, seqs=1, rows=1,
             tokens=1040, gate=True, shape=1),
        # A decode step of 256 requests, 1024 prompt tokens and up to 256 generated ones.
        dict(name="attend_256_requests", op="attend", q_heads=16, kv_heads=2, dim=256, bits=4, half=False, seqs=256, rows=1,
             tokens=1280, gate=True, shape=2),
        # The verify step of 128 requests with shared 2048-token prompts: the last token and three drafts.
        dict(name="attend_128_verify", op="attend", q_heads=16, kv_heads=2, dim=256, bits=4, half=False, seqs=128, rows=4,
             tokens=2300, gate=True, shape=3),
        # A few long documents, fp16, heads of 128.
        dict(name="attend_long_documents", op="attend", q_heads=32, kv_heads=4, dim=128, bits=4, half=True, seqs=7, rows=1,
             tokens=65535, gate=False, shape=4),
        # 8 bits, a kv head for each query head.
        dict(name="attend_8_bits", op="attend", q_heads=8, kv_heads=8, dim=128, bits=8, half=False, seqs=61, rows=1,
             tokens=4001, gate=False, shape=5),
        # Small heads, six query heads for each kv head.
        dict(name="attend_small_heads", op="attend", q_heads=24, kv_heads=4, dim=64, bits=4, half=False, seqs=33, rows=1,
             tokens=2048, gate=False, shape=6),
        # Chunks of prompts behind what is in the cache already: a prefill step.
        dict(name="attend_chunks", op="attend", q_heads=16, kv_heads=2, dim=256, bits=4, half=False, seqs=3, rows=700,
             tokens=4500, gate=True, shape=7),
        # The new tokens of a small decode step.
        dict(name="store_24_rows", op="store", kv_heads=2, dim=256, bits=4, half=False, seqs=24, rows=1, tokens=1100, shape=8),
        # A prefill step of 8192 tokens.
        dict(name="store_8192_rows", op="store", kv_heads=2, dim=256, bits=4, half=False, seqs=8, rows=1024, tokens=2000,
             shape=9),
        # fp16, 8 bits, chunks of odd lengths.
        dict(name="store_8_bits", op="store", kv_heads=8, dim=128, bits=8, half=True, seqs=7, rows=611, tokens=1500, shape=10),
        # A short sequence is read back.
        dict(name="load_500_tokens", op="load", kv_heads=2, dim=256, bits=4, half=False, seqs=1, rows=500, tokens=500, shape=11),
        # Long sequences are read back whole.
        dict(name="load_100000_tokens", op="load", kv_heads=4, dim=128, bits=4, half=False, seqs=3, rows=33400, tokens=33400,
             shape=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    """One more case of the listed ones' ranges; no dearer than the largest of its operator."""
    op = rng.choice(["attend", "attend", "attend", "store", "load"])
    most = {k: max(work(c)[k] for c in listed() if c["op"] == op) for k in ("bytes", "flops")}
    while True:
        shape = rng.randrange(100, 1 << 30)
        dim, bits, half = rng.choice([64, 128, 256, 256]), rng.choice([4, 4, 4, 8]), rng.random() < 0.3
        kv = rng.choice([1, 2, 2, 4, 8])
        case = dict(op=op, kv_heads=kv, dim=dim, bits=bits, half=half, seqs=_log(rng, 1, 256), rows=1,
                    tokens=_log(rng, 20, 65535), shape=shape)
        if op == "attend":
            case.update(q_heads=kv * rng.choice([1, 2, 4, 6, 8, 8, 16]), gate=rng.random() < 0.5,
                        rows=rng.choice([1, 1, 1, 2, 4, 7, _log(rng, 16, 700)]))
        elif op == "store":
            case["rows"] = rng.choice([1, 2, 4, _log(rng, 8, 2048), _log(rng, 8, 2048)])
        else:
            case["rows"] = case["tokens"]
        if case["rows"] > case["tokens"]:
            continue
        w = work(case)
        held = case["seqs"] * case["tokens"] * kv * dim
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and held <= 250_000_000 \
                and case["seqs"] * case["rows"] <= 120_000:
            return case


# ------------------------------------------------------------------------------- case sizes
def _pages(tokens):
    return -(-tokens // PAGE)


def _shape(c):
    """Per sequence its length in tokens and how many of its last tokens are this pass's rows."""
    r = random.Random(c["shape"])
    out = []
    for i in range(c["seqs"]):
        n = c["tokens"] if i == 0 else r.randint(max(c["rows"], c["tokens"] // 2), c["tokens"])
        rows = c["rows"] if c["rows"] <= 8 or i == 0 else r.randint(c["rows"] // 2, c["rows"])
        out.append((n, n if c["op"] == "load" else rows))
    return out


def _token_bytes(c):
    """Bytes of one token's K and V in the cache."""
    return 2 * c["kv_heads"] * (c["dim"] * c["bits"] // 8 + c["dim"] // GROUP * 4)


def work(c):
    seqs = _shape(c)
    rows, keys = sum(r for _, r in seqs), sum(n for n, _ in seqs)
    plain = 4 * rows * c["kv_heads"] * c["dim"]   # the rows' K and V in 16 bits
    if c["op"] == "attend":
        seen = sum(r * n - r * (r - 1) // 2 for n, r in seqs)
        return {"bytes": keys * _token_bytes(c) + (3 if c["gate"] else 2) * rows * c["q_heads"] * c["dim"] * 2 + 8 * rows
                + 4 * sum(_pages(n) for n, _ in seqs), "flops": 4 * c["dim"] * c["q_heads"] * seen}
    if c["op"] == "store":
        return {"bytes": 2 * plain + rows * (_token_bytes(c) + 8), "flops": 4 * rows * c["kv_heads"] * c["dim"]}
    return {"bytes": plain + rows * (_token_bytes(c) + 8), "flops": 4 * rows * c["kv_heads"] * c["dim"]}


# ----------------------------------------------------------------------------------- inputs
def _ints(x, dev):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def _kv(gen, dev, tokens, heads, dim, dtype):
    """Keys and values as a model makes them: channels with an offset and a size of their own, a few large."""
    k = torch.randn(tokens, heads, dim, generator=gen, device=dev)
    size = torch.exp(0.4 * torch.randn(heads, dim, generator=gen, device=dev))
    k = k.mul_(size).add_(torch.randn(heads, dim, generator=gen, device=dev) * size).to(dtype)
    v = torch.randn(tokens, heads, dim, generator=gen, device=dev).mul_(0.7).to(dtype)
    return k, v


def _inputs(c, seed):
    """Everything that a pass is given, before it is put into either side's form."""
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    host = random.Random(seed)
    dtype = torch.float16 if c["half"] else torch.bfloat16
    seqs = _shape(c)
    pages = [_pages(n) for n, _ in seqs]
    ids = list(range(1, 1 + sum(pages)))   # page 0 is the padding page
    host.shuffle(ids)
    table = np.zeros((len(seqs), max(pages)), dtype=np.int32)
    at = 0
    for i, p in enumerate(pages):
        table[i, :p] = ids[at:at + p]
        at += p
    d = dict(c=c, seqs=seqs, dtype=dtype, num_pages=len(ids) + 1, page_table=torch.from_numpy(table).to(dev))
    row_seq = np.repeat(np.arange(len(seqs)), [r for _, r in seqs])
    position = np.concatenate([np.arange(n - r, n) for n, r in seqs])
    d["slots"] = torch.from_numpy(row_seq.astype(np.int32)).to(dev)
    d["positions"] = torch.from_numpy(position.astype(np.int32)).to(dev)
    rows = len(row_seq)
    if c["op"] == "store":
        d["k"], d["v"] = _kv(gen, dev, rows, c["kv_heads"], c["dim"], dtype)
        return d
    # What the cache holds: every page full, as if other sequences had used it before.
    d["k"], d["v"] = _kv(gen, dev, d["num_pages"] * PAGE, c["kv_heads"], c["dim"], dtype)
    if c["op"] == "attend":
        d["q"] = torch.randn(rows, c["q_heads"], c["dim"], generator=gen, device=dev).to(dtype)
        d["gate"] = torch.randn(rows, c["q_heads"], c["dim"], generator=gen, device=dev).to(dtype) if c["gate"] else None
        d["lens"] = d["positions"] + 1
        d["start"] = _ints([0] + list(np.cumsum([r for _, r in seqs])), dev)
    return d


def prepare(case, seed):
    d = _inputs(case, seed)
    dev = d["slots"].device
    c = case
    filled = c["op"] != "store"
    if own:
        from zstep_b200.ops.quant_cache import QuantAttention, QuantCache

        d["cache"] = QuantCache(1, d["num_pages"], c["kv_heads"], c["dim"], bits=c["bits"], page_size=PAGE, device=dev)
        if filled:
            every = torch.arange(d["num_pages"], dtype=torch.int32, device=dev)
            places = torch.arange(d["num_pages"] * PAGE, dtype=torch.int32, device=dev)
            d["cache"].write(0, d["k"], d["v"], every[None], torch.zeros_like(places), places)
        if c["op"] == "attend":
            rows = max(r for _, r in d["seqs"])
            d["plan"] = QuantAttention(d["cache"], c["q_heads"], max_rows=len(d["q"]), max_seqs=len(d["seqs"]), max_seq_rows=rows)
            d["out"] = torch.empty(len(d["q"]), c["q_heads"] * c["dim"], dtype=d["dtype"], device=dev)
    else:
        held = []
        for x in (d["k"], d["v"]):
            shape = (d["num_pages"], PAGE, c["kv_heads"])
            if filled:
                n, s, z = _plain_quantise(x, c["bits"])
                held.append([n.view(*shape, -1), s.view(*shape, -1), z.view(*shape, -1)])
            else:
                held.append([torch.zeros(*shape, c["dim"] * c["bits"] // 8, dtype=torch.uint8, device=dev),
                             *(torch.zeros(*shape, c["dim"] // GROUP, dtype=torch.bfloat16, device=dev) for _ in range(2))])
        d["held"] = held
        d["lens_list"] = [n for n, _ in d["seqs"]]
        d["rows_list"] = [r for _, r in d["seqs"]]
    if filled:
        del d["k"], d["v"]
    return d


# --------------------------------------------------------------------------------- one pass
def run(st):
    if own:
        return _OWN[st["c"]["op"]](st)
    return _PLAIN[st["c"]["op"]](st)


def _own_store(st):
    st["cache"].write(0, st["k"], st["v"], st["page_table"], st["slots"], st["positions"])
    return st["cache"].read(0, st["page_table"], st["slots"], st["positions"], dtype=st["dtype"])


def _own_load(st):
    return st["cache"].read(0, st["page_table"], st["slots"], st["positions"], dtype=st["dtype"])


def _own_attend(st):
    plan = st["plan"]
    plan.update(st["slots"], st["lens"], st["start"])
    return plan.attend(0, st["q"], st["page_table"], st["c"]["dim"] ** -0.5, gate=st["gate"], out=st["out"])


_OWN = dict(store=_own_store, load=_own_load, attend=_own_attend)


# ------------------------------------------------------------------------------ plain forms
def _up(x):
    """Non-negative 32-bit numbers rounded up to bf16."""
    return ((x.view(torch.int32) + 0xFFFF) & ~0xFFFF).view(torch.float32)


def _down(x):
    """32-bit numbers rounded down to bf16."""
    cut = (x.view(torch.int32) & ~0xFFFF).view(torch.float32)
    return torch.where(x < 0, -_up(x.abs()), cut)


def _plain_quantise(x, bits):
    """Rows [n, heads, dim] as packed numbers (element 2i in the low four bits), scales and offsets.  In
    pieces, so that the 32-bit intermediates stay small."""
    n, h, d = x.shape
    top = (1 << bits) - 1
    parts = torch.tensor(float(top), device=x.device)   # a tensor: dividing by a number may multiply by its inverse
    packed = torch.empty(n, h, d * bits // 8, dtype=torch.uint8, device=x.device)
    s = torch.empty(n, h, d // GROUP, dtype=torch.bfloat16, device=x.device)
    z = torch.empty_like(s)
    piece = max(1, (1 << 25) // (h * d))
    for i in range(0, n, piece):
        f = x[i:i + piece].float().view(-1, h, d // GROUP, GROUP)
        low = _down(f.amin(-1, keepdim=True))
        step = _up((f.amax(-1, keepdim=True) - low) / parts)
        q = torch.round((f - low) / torch.where(step > 0, step, 1.0)).clamp(0, top).to(torch.uint8).view(-1, h, d)
        packed[i:i + piece] = q if bits == 8 else q[..., 0::2] | (q[..., 1::2] << 4)
        s[i:i + piece], z[i:i + piece] = step[..., 0], low[..., 0]
    return packed, s, z


def _plain_values(held, bits):
    """What packed numbers, scales and offsets stand for, in 32 bits."""
    n, s, z = held
    if bits == 4:
        n = torch.stack([n & 15, n >> 4], -1).flatten(-2)
    f = n.float().unflatten(-1, (-1, GROUP))
    return f.mul_(s.float()[..., None]).add_(z.float()[..., None]).flatten(-2)


def _places(st):
    p = st["positions"].long()
    return st["page_table"][st["slots"].long(), p // PAGE].long(), p % PAGE


def _plain_load(st):
    at = _places(st)
    return tuple(_plain_values([t[at] for t in held], st["c"]["bits"]).to(st["dtype"]) for held in st["held"])


def _plain_store(st):
    at = _places(st)
    for x, held in zip((st["k"], st["v"]), st["held"]):
        for t, new in zip(held, _plain_quantise(x, st["c"]["bits"])):
            t[at] = new
    return _plain_load(st)


def _plain_attend(st):
    c = st["c"]
    S, R, kvh, dim = c["seqs"], max(st["rows_list"]), c["kv_heads"], c["dim"]
    lens, rows = torch.tensor(st["lens_list"]), torch.tensor(st["rows_list"])
    pad = torch.arange(R)[None, :] < rows[:, None]
    dev = st["q"].device
    where = torch.nonzero(pad.flatten()).flatten().to(dev)   # place of every row in the padded batch
    q = torch.zeros(S * R, kvh, c["q_heads"] // kvh, dim, device=dev)
    q[where] = st["q"].float().view(-1, kvh, c["q_heads"] // kvh, dim)
    seen = torch.zeros(S * R, dtype=torch.int32, device=dev)
    seen[where] = st["lens"]
    seen = seen.view(S, R)
    pages = st["page_table"][:, :_pages(int(lens.max()))].long()
    out = torch.empty(S * R, kvh, c["q_heads"] // kvh, dim, device=dev)
    step = max(1, (1 << 30) // (R * c["q_heads"] * pages.shape[1] * PAGE))
    for i in range(0, S, step):
        part = slice(i, i + step)
        k, v = (_plain_values([t[pages[part]].flatten(1, 2) for t in held], c["bits"]) for held in st["held"])
        s = torch.einsum("srhnd,sthd->srhnt", q.view(S, R, kvh, -1, dim)[part], k) * dim ** -0.5
        hidden = torch.arange(k.shape[1], device=dev)[None, None, :] >= seen[part, :, None]
        s.masked_fill_(hidden[:, :, None, None, :], float("-inf"))
        s = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-3e38))
        total = s.sum(-1, keepdim=True)
        o = torch.einsum("srhnt,sthd->srhnd", s, v) / torch.where(total > 0, total, 1.0)
        out.view(S, R, kvh, -1, dim)[part] = o
    o = out[where].reshape(-1, c["q_heads"] * dim)
    if st["gate"] is not None:
        o = o * torch.sigmoid(st["gate"].float()).view_as(o)
    return o.to(st["dtype"])


_PLAIN = dict(store=_plain_store, load=_plain_load, attend=_plain_attend)


# --------------------------------------------------------------------------- 64-bit results
def exact(case, seed):
    d = _inputs(case, seed)
    p = d["positions"].long()
    page, place = d["page_table"][d["slots"].long(), p // PAGE].long(), p % PAGE
    if case["op"] == "store":
        return tuple(_exact_held(d[n], case["bits"]) for n in ("k", "v"))
    if case["op"] == "load":
        return tuple(_exact_held(d[n][page * PAGE + place], case["bits"]) for n in ("k", "v"))
    return _exact_attend(case, d)


def _bf16_beside(x, up):
    """The nearest bf16 not below (up) or not above 64-bit numbers."""
    m, e = torch.frexp(x)   # |m| in [0.5, 1): eight bits of it are kept
    m = torch.ldexp(m, torch.full_like(e, 8))
    return torch.ldexp(torch.ceil(m) if up else torch.floor(m), e - 8)


def _exact_held(x, bits):
    f = x.double().unflatten(-1, (-1, GROUP))
    low = _bf16_beside(f.min(-1, keepdim=True).values, False)
    step = _bf16_beside((f.max(-1, keepdim=True).values - low) / (2 ** bits - 1), True)
    n = torch.where(step > 0, torch.round((f - low) / step), 0.0)
    return (n.clamp(max=2 ** bits - 1) * step + low).flatten(-2)


def _exact_attend(c, d):
    """Sequence by sequence and head by head, over the sequence's own tokens."""
    dim, n = c["dim"], c["q_heads"] // c["kv_heads"]
    out = torch.empty(len(d["q"]), c["q_heads"], dim, dtype=torch.float64, device=d["q"].device)
    first = 0
    for s, (length, rows) in enumerate(d["seqs"]):
        pages = d["page_table"][s, :_pages(length)].long()
        seen = torch.arange(length - rows + 1, length + 1, device=out.device)
        for h in range(c["kv_heads"]):
            k, v = (_exact_held(d[x].view(-1, PAGE, c["kv_heads"], dim)[pages, :, h].reshape(-1, dim)[:length], c["bits"])
                    for x in ("k", "v"))
            for a in range(0, rows, 128):
                q = d["q"][first + a:first + min(rows, a + 128), h * n:(h + 1) * n].double()
                x = torch.matmul(q.reshape(-1, dim), k.T).view(len(q), n, length) / dim ** 0.5
                gone = torch.arange(length, device=x.device)[None, :] >= seen[a:a + 128, None]
                x = torch.where(gone[:, None, :], float("-inf"), x)
                w = torch.exp(x - torch.logsumexp(x, -1, keepdim=True))
                out[first + a:first + a + len(q), h * n:(h + 1) * n] = torch.matmul(w.view(-1, length), v).view(len(q), n, dim)
        first += rows
    if d["gate"] is not None:
        out = out / (1 + torch.exp(-d["gate"].double()))
    return out.reshape(len(out), -1)
