"""The decays' gradient of linear_attn_fn at its own size: heads that remember a thousand positions and heads that forget at
once, cut into segments and whole, packed, between decays of nothing."""

from __future__ import annotations

import pytest
import torch

from _attn_dg import FORGETS, close_dg, parts
from test_attn_gpu import BF16, DEV, FP16, FP32, TYPES, make, own

pytestmark = pytest.mark.gpu
RATES = (0.001, 0.03, 0.3, 1.0, 4.0, 10.0, 20.0)


def rated(B, L, H, K, dk, dv, dtype, states=False, seqs=None, seed=0, rates=RATES):
    """Heads whose log decays are around one of the rates each, in turns."""
    p = make(B, L, H, K, dk, dv, dtype, states, True, seqs, seed)
    gen = torch.Generator().manual_seed(seed + 1)
    r = torch.tensor(rates).repeat(-(-H // len(rates)))[:H]
    p["g"] = (-r * (0.5 + torch.rand(B, L, H, generator=gen))).to(dtype).to(DEV)
    return p


def check(p, ends=None, name=""):
    if ends is None:
        return close_dg(own(p)["dg"], p, name)
    got = own(p, torch.tensor(ends, dtype=torch.int32, device=DEV))["dg"]
    for i, (a, b) in enumerate(zip(ends, ends[1:])):
        if b > a:
            close_dg(got[:, a:b], parts(p, a, b, i), f"{name}sequence {i}")


@TYPES
@pytest.mark.parametrize("size", [(1, 5, 7, 7, 16, 16), (1, 130, 7, 1, 64, 64), (1, 203, 7, 7, 128, 128), (2, 97, 14, 7, 40, 72),
                                  (1, 150, 7, 7, 72, 40), (1, 64, 7, 7, 61, 33), (1, 161, 7, 7, 128, 48)], ids=str)
@pytest.mark.parametrize("states", [False, True])
def test_short(size, states, dtype):
    check(rated(*size, dtype, states))


@TYPES
@pytest.mark.parametrize("L", [450, 1029])
def test_cut(L, dtype):
    """Few heads: segments side by side."""
    check(rated(1, L, 7, 7, 16, 24, dtype, True))


@TYPES
@pytest.mark.parametrize("L", [511, 1300])
def test_whole(L, dtype):
    """Enough heads that sequences are not cut: in fp32 the states of every 512 positions are left on the way."""
    check(rated(1, L, 49, 49, 8, 8, dtype, True))


@pytest.mark.parametrize("dtype", [BF16, FP16], ids=["bf16", "fp16"])
def test_whole_and_long(dtype):
    """Past the 2048 positions of a piece, with one position to spare and with whole pieces."""
    check(rated(1, 2 * 2048 + 1, 49, 49, 4, 4, dtype, True))
    check(rated(1, 2 * 2048, 49, 49, 4, 4, dtype))


@TYPES
@pytest.mark.parametrize("size", [(61, 33), (72, 128), (30, 7)], ids=str)
def test_whole_of_odd_sizes(size, dtype):
    """States that are left on the way have rows of no whole vectors."""
    p = rated(1, 1100 if dtype == FP32 else 2100, 43, 43, *size, dtype, True)
    got = own(p)["dg"]
    for h in (0, 15, 30, 39, 42):
        close_dg(got[:, :, h:h + 1], {n: None if t is None else t[:, h:h + 1] if n in ("init", "dfinal") else t[:, :, h:h + 1]
                                      for n, t in p.items()}, f"head {h}")


@TYPES
def test_batches(dtype):
    """Rows of a batch, whole: states on the way have places of their own."""
    check(rated(7, 1100, 7, 7, 8, 8, dtype, True))


@TYPES
@pytest.mark.parametrize("states", [False, True])
def test_packed(states, dtype):
    ends = [0, 3, 3, 700, 701, 765, 1200, 1207]
    check(rated(1, ends[-1], 7, 7, 16, 16, dtype, states, len(ends) - 1), ends)


@TYPES
def test_packed_and_whole(dtype):
    """768 heads and more: packed sequences are not cut, and pieces begin at each one's first position."""
    ends = [0, 2, 650, 650, 1300, 2500]
    p = rated(1, ends[-1], 768, 2, 2, 2, dtype, True, len(ends) - 1, rates=RATES[:6])
    got = own(p, torch.tensor(ends, dtype=torch.int32, device=DEV))["dg"]
    some = [0, 1, 2, 3, 4, 5, 384, 767]  # (of the first and the second key head)
    for i, (a, b) in enumerate(zip(ends, ends[1:])):
        if b > a:
            for h in some:
                one = {n: None if t is None else (t[:, :, h // 384:h // 384 + 1] if n in ("q", "k") else
                                                  t[:, h:h + 1] if n in ("init", "dfinal") else t[:, :, h:h + 1])
                       for n, t in parts(p, a, b, i).items()}
                close_dg(got[:, a:b, h:h + 1], one, f"sequence {i} head {h}")


@TYPES
def test_any_decays(dtype):
    """Positions that forget far more than the ones around them."""
    p = rated(1, 500, 7, 7, 16, 16, dtype, True)
    gen = torch.Generator().manual_seed(5)
    p["g"] = (p["g"].float() - 12.0 * (torch.rand(1, 500, 7, generator=gen) < 0.1).float().to(DEV)).to(dtype)
    check(p)


@TYPES
@pytest.mark.parametrize("g", [-88.0, -200.0, -1e4, float("-inf")], ids=str)
@pytest.mark.parametrize("L", [150, 900])
def test_decays_of_nothing(L, g, dtype):
    """Nothing is left of what is behind them, whatever it is, and their own gradient is 0."""
    p = rated(1, L, 7, 7, 16, 16, dtype, True)
    at = [0, 7, 63, 64, 100, L // 2]
    p["g"][:, at] = g
    check(p)
    got = own(p)["dg"]
    assert not got[:, at].any()
    for n, by in (("dout", 1000.0), ("q", -3.0)):
        hit = {**p, n: p[n].clone()}
        hit[n][:, L // 2:] *= by
        assert torch.equal(own(hit)["dg"][:, :L // 2], got[:, :L // 2]), n
    hit = {**p, "dfinal": -7.0 * p["dfinal"]}
    assert torch.equal(own(hit)["dg"][:, :L // 2], got[:, :L // 2])
    assert FORGETS > -87.0


@pytest.mark.parametrize("heads", [7, 49])
def test_errors_are_those_of_32_bits(heads):
    """Root mean square errors of a head, 1300 positions: a thousandth of a thousandth, whatever the head's rate (a term
    has 16 * 2**-24 of its size, 1e-6; what passes over chunks of 32 adds up over 512 / 32 of them, sqrt(32) times that at
    most were every rounding the largest)."""
    from _attn_dg import definition
    p = rated(1, 1300, heads, heads, 16, 16, FP32, rates=(0.001, 0.03, 0.3, 1.0, 4.0, 10.0, 15.0))
    e, z = definition(p)
    err = (own(p)["dg"].double().cpu() - e).square().mean((0, 1)).sqrt() / z.square().mean((0, 1)).sqrt()
    assert (err < 16 * 2.0**-24 * (1 + 32**0.5)).all(), err
