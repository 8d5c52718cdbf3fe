"""The limit that the precision tests hold the quantised attention to tells mistakes from roundings."""

import pytest
import torch

from tests.quant_oracle import LIMIT, attention, distance, held


def inputs(dim=64, keys=300, rows=12, heads=4, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(3)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    size = torch.exp(0.5 * rnd(2, dim))
    k = held((size * (rnd(keys, 2, dim) + rnd(2, dim))).to(dtype), 4)
    v = held((0.7 * rnd(keys, 2, dim)).to(dtype), 4)
    return rnd(rows, heads, dim).to(dtype), k, v, [keys - i % 3 for i in range(rows)]


def test_the_definition():
    """One group by hand: 0..15 with 4 bits are the numbers themselves, and two keys of equal scores their mean."""
    x = torch.arange(64).remainder(16).float().to(torch.bfloat16)
    assert torch.equal(held(x, 4), x.double())
    y = held(torch.tensor([-1.0, 1.0]).repeat(32), 8)   # z = -1, s = 2 / 255 rounded up to 8 bits
    assert y[0] == -1 and y[1] == -1 + 254 * (129 * 2.0 ** -14)   # 2 / s = 254.02
    q = torch.zeros(2, 1, 64)
    v = torch.stack([torch.full((1, 64), 1.0), torch.full((1, 64), 4.0)]).double()
    got = attention(q, torch.ones(2, 1, 64).double(), v, [2, 0], 1.0)
    assert torch.all(got[0] == 2.5) and torch.all(got[1] == 0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_roundings_pass(dtype):
    """f16 weights, and for bf16 outputs f16 keys and values too."""
    q, k, v, lens = inputs(dtype=dtype)
    want = attention(q, k, v, lens, 0.125)
    assert distance(want.to(dtype), want) == 1.0
    if dtype == torch.bfloat16:
        assert distance(attention(q, k.half().double(), v.half().double(), lens, 0.125).to(dtype), want) < LIMIT
    else:
        assert distance(attention(q, k.float().double(), v.float().double(), lens, 0.125).to(dtype), want) < 1.01


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("mistake", ["a key less", "a key more", "scores 2 % off", "equal weights", "zeros", "a tile less", "another head",
                                     "a group of V 1 % off", "two keys exchanged"])
def test_mistakes_do_not(mistake, dtype):
    q, k, v, lens = inputs(dtype=dtype)
    want = attention(q, k, v, lens, 0.125)
    if mistake == "a key less":
        got = attention(q, k, v, [n - 1 for n in lens], 0.125)
    elif mistake == "a key more":
        got = attention(q, torch.cat([k, k[:1]]), torch.cat([v, -v[:1]]), [n + 1 for n in lens], 0.125)
    elif mistake == "scores 2 % off":
        got = attention(q, k, v, lens, 0.1275)
    elif mistake == "equal weights":
        got = attention(q, k, v, lens, 0.0)
    elif mistake == "zeros":
        got = torch.zeros_like(want)
    elif mistake == "a tile less":
        got = attention(q, k[16:], v[16:], [n - 16 for n in lens], 0.125)
    elif mistake == "another head":
        got = attention(q, k.flip(1), v, lens, 0.125)
    elif mistake == "a group of V 1 % off":
        got = want * 1.01
    else:
        w = v.clone()
        w[[5, 9]] = v[[9, 5]]
        got = attention(q, k, w, lens, 0.125)
    assert distance(got.to(dtype), want) > 2 * LIMIT
