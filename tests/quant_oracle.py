"""The quantised K/V cache and the attention over it in 64 bits, and how far an output is from it: a plain
implementation of the definition, apart from the kernels and from the other tests' references."""

import torch

GROUP = 64
# An output's distance from the 64-bit result, as a multiple of what rounding that result to the output's type costs
# alone.  The other roundings are independent of it and random: bf16 outputs (0.0017 of the norm) come with weights, and
# with many query slots K and V, in f16 (0.0002 of the norm each, K's times a score's spread of about 2), which makes
# (1 + 0.0002^2 (1 + 1 + 4) / 0.0017^2)^(1/2) = 1.04; f16 outputs (0.00021) with 32-bit sums that are cut behind their 24th
# bit (0.0001 over some thousands of keys): 1.11.
LIMIT = 1.25


def beside(x, up):
    """The nearest bf16 not below (up) or not above."""
    m, e = torch.frexp(x)
    m = torch.ldexp(m, torch.full_like(e, 8))
    return torch.ldexp(torch.ceil(m) if up else torch.floor(m), e - 8)


def held(x, bits):
    """What a cache holds of rows [..., dim]."""
    f = x.double().unflatten(-1, (-1, GROUP))
    z = beside(f.amin(-1, keepdim=True), False)
    s = beside((f.amax(-1, keepdim=True) - z) / (2 ** bits - 1), True)
    n = torch.where(s > 0, torch.round((f - z) / torch.where(s > 0, s, 1.0)), 0.0).clamp(max=2 ** bits - 1)
    return (n * s + z).flatten(-2)


def attention(q, k, v, lens, scale, gate=None):
    """Rows ``q`` [rows, q heads, dim], row r over the first lens[r] of ``k`` and ``v`` [keys, kv heads, dim] (64-bit).
    [rows, q heads, dim]; a row without keys is 0."""
    rows, hq, dim = q.shape
    group = hq // k.shape[1]
    out = torch.zeros(rows, hq, dim, dtype=torch.float64, device=q.device)
    hidden = torch.arange(len(k), device=q.device)[None, :] >= torch.as_tensor(lens, device=q.device)[:, None]
    some = ~hidden.all(1)
    for h in range(hq):
        x = (q[:, h].double() @ k[:, h // group].T) * scale
        w = torch.softmax(x.masked_fill(hidden, float("-inf")), -1)
        w = torch.where(hidden, 0.0, w)   # also where nothing is seen
        out[:, h] = torch.where(some[:, None], w @ v[:, h // group], 0.0)
    if gate is not None:
        out = out * torch.sigmoid(gate.double())
    return out


def distance(got, want):
    """|got - want| over |want rounded to got's type - want|; 0 where got is want."""
    want = want.reshape(got.shape)
    off, alone = (got.double() - want).norm(), (want.to(got.dtype).double() - want).norm()
    return float(off / alone) if off != 0 else 0.0
