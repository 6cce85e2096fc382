"""linear_attn_fn on the GPU against its definition in float64."""

from __future__ import annotations

import math

import pytest
import torch

import causal_conv1d_amd as cc
from _attn import attn64, close

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
TYPES = pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
GRADS = {"q": "dq", "k": "dk", "v": "dv", "g": "dg", "init": "dinit"}


def make(B, L, H, K, dk, dv, dtype, states=False, train=False, seqs=None, seed=0):
    gen = torch.Generator().manual_seed(seed + 7 * L + dk)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    n = B if seqs is None else seqs
    # heads that forget at once and heads that hardly do
    rate = torch.logspace(-3, 0.5, H)
    p = {"q": r(B, L, K, dk), "k": r(B, L, K, dk), "v": r(B, L, H, dv), "g": -rate * torch.rand(B, L, H, generator=gen)}
    p = {name: t.to(dtype).to(DEV) for name, t in p.items()}
    p["init"] = r(n, H, dk, dv).to(DEV) if states else None
    p["dout"] = r(B, L, H, dv).to(dtype).to(DEV) if train else None
    p["dfinal"] = r(n, H, dk, dv).to(DEV) if train and states else None
    return p


def own(p, cu=None, scale=None):
    """out, final and the gradients, by name."""
    states = p["init"] is not None
    if p["dout"] is None:
        r = cc.linear_attn_fn(p["q"], p["k"], p["v"], p["g"], scale, cu, p["init"], states)
        return {"out": r[0], "final": r[1]} if states else {"out": r}
    leaves = {n: p[n].detach().requires_grad_() for n in GRADS if p[n] is not None}
    r = cc.linear_attn_fn(leaves["q"], leaves["k"], leaves["v"], leaves["g"], scale, cu, leaves.get("init"), states)
    grads = torch.autograd.grad(r, list(leaves.values()), (p["dout"], p["dfinal"]) if states else p["dout"])
    got = {"out": r[0], "final": r[1]} if states else {"out": r}
    return {**got, **{GRADS[n]: g for n, g in zip(leaves, grads)}}


def compare(got, p, scale=None, rows=slice(None), name=""):
    s = p["q"].shape[-1] ** -0.5 if scale is None else scale
    args = [p[n] for n in ("q", "k", "v", "g")]
    e, m = (attn64(*args, s, p["init"], p["dout"], p["dfinal"], mag=x) for x in (False, True))
    for n, t in got.items():
        close(t, e[n], m[n], p["q"].shape[1], f"{name}{n}")


def check(p, scale=None):
    compare(own(p, scale=scale), p, scale)


def check_packed(p, ends, scale=None):
    """Every sequence as on its own; nothing where there is none."""
    got = own(p, torch.tensor(ends, dtype=torch.int32, device=DEV), scale)
    for i, (a, b) in enumerate(zip(ends, ends[1:])):
        one = {n: None if t is None else (t[i:i + 1] if n in ("init", "dfinal") else t[:, a:b]) for n, t in p.items()}
        part = {n: t[i:i + 1] if n in ("final", "dinit") else t[:, a:b] for n, t in got.items()}
        compare(part, one, scale, name=f"sequence {i} ")
    for n, t in got.items():
        if n not in ("final", "dinit"):
            assert (t[:, :ends[0]] == 0).all() and (t[:, ends[-1]:] == 0).all(), n
    return got


SIZES = [(1, 1, 1, 1, 1, 1), (2, 64, 2, 2, 64, 64), (1, 65, 3, 1, 128, 128), (2, 33, 4, 2, 128, 64), (1, 130, 2, 1, 64, 128),
         (1, 31, 2, 2, 17, 5), (3, 7, 6, 3, 80, 72), (1, 200, 1, 1, 96, 33), (1, 129, 2, 2, 8, 100), (1, 63, 5, 5, 127, 127)]


@TYPES
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_forward(size, dtype):
    check(make(*size, dtype))
    check(make(*size, dtype, states=True))


@TYPES
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_gradients(size, dtype):
    check(make(*size, dtype, train=True))
    check(make(*size, dtype, states=True, train=True))


@TYPES
@pytest.mark.parametrize("size", [(1, 700, 2, 1, 64, 64), (2, 1100, 1, 1, 128, 96)], ids=str)
def test_segments(size, dtype):
    """Few heads and many positions: the sequence is cut into segments that run side by side."""
    check(make(*size, dtype, states=True, train=True))


@TYPES
@pytest.mark.parametrize("ends", [[0, 1, 64, 64, 130, 131], [3, 70, 90], [0, 0, 0], [5, 5, 40], [0, 600, 601, 1100]], ids=str)
@pytest.mark.parametrize("states", [False, True])
def test_packed(ends, states, dtype):
    L = max(ends[-1] + (5 if ends[0] else 0), 2)
    check_packed(make(1, L, 4, 2, 64, 72, dtype, states, True, len(ends) - 1), ends)


@TYPES
def test_scale(dtype):
    check(make(1, 70, 2, 1, 32, 40, dtype, True, True), scale=0.7)
    check(make(1, 70, 2, 1, 32, 40, dtype, True, True), scale=-1.5)


def test_scale_zero():
    p = make(1, 70, 2, 1, 32, 40, BF16, True, True)
    got = own(p, scale=0.0)
    assert (got["out"] == 0).all() and (got["dq"] == 0).all()
    compare({n: t for n, t in got.items() if n != "dg"}, p, 0.0)
