"""Tolerances of the decays' gradient, which is held to its own size.

dg[t] = exp(g[t]) <G[t], S[t-1]> is a sum of products, one for each pair of positions on its two sides and each pair of
elements. Inputs of the tests have independent signs, so a sum is about the root of its terms' squares, Z[t], which is the
definition once more over the squares of its operands (``size``). Errors of the terms are independent as well:

* a product's operands are off by e_T of it: bf16 planes leave out up to 2**-15 where a 16-bit result follows (``_attn``),
  and a few dozen roundings of 2**-24, independent, come to no more than 16 * 2**-24 of it;
* what passes over a whole chunk is a difference of sums at the chunks' ends, whose errors add up from chunk to chunk back
  to where they begin anew: at the end of the sequence, every 2048 positions, or where a position forgets all (a decay of
  less than 2**-24). At most n = 2048 / 32 chunks, each with an error of e_T Z of its two sums.

    |got - exact| <= u_T |exact| + 6 e_T (Z[t] + sqrt(2 n) max Z[later, as far as errors come from])

six standard deviations. A result of zeros is off by |exact|, about Z: it has to fail.
"""

from __future__ import annotations

import math

import torch

from _attn import UNIT, attn64

FORGETS = -16.64  # log(2**-24)


def parts(p, a, b, i):
    """Sequence i, positions a to b."""
    return {n: None if t is None else (t[i:i + 1] if n in ("init", "dfinal") else t[:, a:b]) for n, t in p.items()}


def definition(p, scale=None):
    """dg, and its size Z, in float64."""
    s = p["q"].shape[-1] ** -0.5 if scale is None else scale
    ops = [p["q"], p["k"], p["v"], p["g"]]
    e = attn64(*ops, s, p["init"], p["dout"], p["dfinal"])["dg"]
    sq = lambda t: None if t is None else t.detach().double() ** 2  # noqa: E731
    each = p["v"].shape[2] // p["q"].shape[2]
    q, k = (sq(t).repeat_interleave(each, 2) for t in ops[:2])
    z = attn64(q, k, sq(p["v"]), 2.0 * p["g"].detach().double(), s * s, sq(p["init"]), sq(p["dout"]), sq(p["dfinal"]))["dg"]
    return e, z.sqrt()


def bound(e, z, g, dtype):
    g = g.detach().double().cpu()
    L = e.shape[1]
    reach = z.clone()
    for t in reversed(range(L - 1)):
        later = torch.where(g[:, t + 1] < FORGETS, torch.zeros_like(z[:, t]), reach[:, t + 1])
        reach[:, t] = torch.maximum(z[:, t], later)
    eps = 16 * 2.0**-24 + (0.0 if dtype == torch.float32 else 2.0**-15)
    n = min(math.ceil(L / 32), 2048 // 32)
    spacing = 2.0**-25 if dtype == torch.float16 else 1e-30
    return UNIT[dtype] * e.abs() + 6 * eps * (z + math.sqrt(2 * n) * reach) + spacing


def close_dg(got, p, name="", scale=None):
    e, z = definition(p, scale)
    assert got.shape == e.shape and got.dtype == p["g"].dtype
    lim = bound(e, z, p["g"], got.dtype)
    err = (got.detach().double().cpu() - e).abs()
    bad = ~(err <= lim)
    if bad.any():
        at = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} beyond the bound; at {at} (g {p['g'][at].item()}): "
                             f"{got[at].item()} against {e[at].item()}, bound {lim[at].item()}; heads "
                             f"{sorted(set(bad.nonzero()[:, 2].tolist()))}, worst {(err / lim).max().item()} of it")
