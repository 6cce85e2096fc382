"""The bound that the decays' gradient is held to tells a right one from wrong ones."""

from __future__ import annotations

import pytest
import torch

from _attn import attn64
from _attn_dg import bound, definition

RATES = torch.tensor([0.001, 0.03, 0.3, 1.0, 4.0, 10.0])
TYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32], ids=["bf16", "fp16", "fp32"])


def make(L, d, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    H = len(RATES)
    p = {"q": r(1, L, H, d), "k": r(1, L, H, d), "v": r(1, L, H, d), "g": -RATES * (0.5 + torch.rand(1, L, H, generator=gen)),
         "dout": r(1, L, H, d)}
    p = {n: t.to(dtype) for n, t in p.items()}
    return {**p, "init": r(1, H, d, d), "dfinal": r(1, H, d, d)}


def fails(got, p, where=slice(None)):
    """Share of positions beyond the bound, by head."""
    e, z = definition(p)
    lim = bound(e, z, p["g"], p["q"].dtype)
    return ((got - e).abs() > lim)[:, where].double().mean((0, 1))


def gradients(p, **kw):
    p = {**p, **kw}
    return attn64(p["q"], p["k"], p["v"], p["g"], p["q"].shape[-1] ** -0.5, p["init"], p["dout"], p["dfinal"])


@TYPES
@pytest.mark.parametrize("L", [700, 2500])
def test_zeros_fail(L, dtype):
    p = make(L, 8, dtype)
    share = fails(torch.zeros(1, L, len(RATES)), p)
    assert (share[:4] > 0.9).all()
    # decays of exp(-2) to exp(-6): the bound has 6 * 2**-15 * (1 + sqrt(2 * 22)) = 1.4e-3 of the largest later size, and
    # where a position's own is exp(-4) of that (0.018), one gradient in ten or so is smaller still
    assert share[4] > 0.8


@TYPES
def test_a_missing_final_state_fails(dtype):
    p = make(300, 8, dtype)
    got = gradients(p, dfinal=None)["dg"]
    share = fails(got, p, slice(250, 300))
    assert (share[:2] > 0.8).all()
    # of the third, exp(-0.3 n) of the term is left n positions before the end: above bf16's 2**-8 for 18 of these 50
    assert share[2] > 0.3
    assert not fails(gradients(p)["dg"].to(dtype).double(), p).any()  # and the definition, rounded, does not


@TYPES
def test_a_missing_carry_fails(dtype):
    """Segments of 192 positions whose gradients come from no further than their end."""
    p = make(576, 8, dtype)
    got, init = [], p["init"]
    for a in range(0, 576, 192):
        one = {n: t[:, a:a + 192] for n, t in p.items() if n in ("q", "k", "v", "g", "dout")}
        r = gradients({**one, "init": init, "dfinal": p["dfinal"] if a == 384 else None})
        got.append(r["dg"])
        init = r["final"]
    share = fails(torch.cat(got, 1), p, slice(0, 384))
    assert share[0] > 0.9 and share[1] > 0.3 and (share[:4] > 0).all()


def test_a_running_sum_of_what_cancels_fails():
    """q . dq - k . dk in fp32, summed in 64 bits: where a head forgets at once, what is lost with the rest is as large."""
    p = make(700, 8, torch.float32)
    r = gradients(p)
    rows, cols = ((p[n].double() * r["d" + n]).sum(-1).float().double() for n in ("q", "k"))
    end = (p["dfinal"].double() * r["final"]).sum((-1, -2))[:, None]
    share = fails(end + (rows - cols).flip(1).cumsum(1).flip(1), p)
    assert share[5] > 0.05 and not share[:3].any()
