"""Decode steps inside torch.compile: traced whole, their states written in place."""

from __future__ import annotations

import pytest
import torch

import causal_conv1d_amd as cc
from test_attn_update_gpu import call, make
from test_scan_update_gpu import make as scan_make

pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:.*torch.jit.script.*:DeprecationWarning")]
DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32


def compiled(f, args, state):
    """f eagerly and compiled, from copies of its arguments: results and states alike."""
    eager = [a.clone() for a in args]
    want = f(*eager)
    torch._dynamo.reset()
    traced = [a.clone() for a in args]
    g = torch.compile(f, backend="aot_eager", fullgraph=True)
    got = g(*traced)
    assert torch.equal(got, want) and torch.equal(traced[state], eager[state]) and not torch.equal(traced[state], args[state])
    assert torch.equal(g(*traced), f(*eager)) and torch.equal(traced[state], eager[state])  # and from there on


@pytest.mark.parametrize("T", [None, 3])
@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("pool", [False, True])
def test_linear_attn_update(pool, dtype, T):
    p = make(4, T, 4, 2, 64, 48, dtype, rows=6 if pool else None)
    idx = torch.tensor([5, -1, 0, 2], dtype=torch.int32, device=DEV) if pool else None

    def f(q, state, k, v, g):
        return cc.linear_attn_update(q, state, k, v, g, attn_state_indices=idx) * 2.0

    compiled(f, [p[n] for n in ("q", "state", "k", "v", "g")], 1)


def test_linear_attn_update_opcheck():
    p = make(3, 2, 4, 2, 32, 24, BF16, rows=5)
    idx = torch.tensor([4, -1, 0], dtype=torch.int32, device=DEV)
    torch.library.opcheck(torch.ops.causal_conv1d_amd._attn_update_inplace.default,
                          (p["q"], p["state"], p["k"], p["v"], p["g"], 0.2, idx, torch.empty_like(p["v"])))


def test_linear_attn_update_of_tensors_that_want_gradients():
    """No autograd, on either path: nothing is recorded, and nothing is refused."""
    p = make(2, None, 2, 2, 16, 16, FP32)
    want = call({**p, "state": p["state"].clone()})
    q = p["q"].detach().requires_grad_()
    out = call({**p, "q": q, "state": p["state"].clone()})
    assert not out.requires_grad and torch.equal(out, want)
    big = torch.stack((p["state"], p["state"]))  # a view, which is written through
    out = call({**p, "q": q, "state": big[1]})
    assert torch.equal(out, want) and torch.equal(big[0], p["state"]) and not torch.equal(big[1], p["state"])


@pytest.mark.parametrize("T", [None, 3])
@pytest.mark.parametrize("softplus", [False, True])
def test_ssm_scan_update(softplus, T):
    p = scan_make(4, 24, 16, 2, T, BF16, rows=6)
    idx = torch.tensor([5, -1, 0, 2], dtype=torch.int32, device=DEV)

    def f(u, state, delta, A, B, C, z):
        return cc.ssm_scan_update(u, state, delta, A, B, C, D=p["D"], z=z, delta_bias=p["bias"], delta_softplus=softplus,
                                  ssm_state_indices=idx) * 2.0

    compiled(f, [p[n] for n in ("u", "state", "delta", "A", "B", "C", "z")], 1)


@pytest.mark.parametrize("T", [None, 3])
@pytest.mark.parametrize("ring", [False, True])
def test_causal_conv1d_update(ring, T):
    x = torch.randn(2, 24, *(() if T is None else (T,)), device=DEV)
    w, bias, state = torch.randn(24, 4, device=DEV), torch.randn(24, device=DEV), torch.randn(2, 24, 5, device=DEV)
    heads = torch.tensor([0, 2], dtype=torch.int32, device=DEV) if ring else None

    def f(x, state, w):
        return cc.causal_conv1d_update(x, state, w, bias, activation="silu", cache_seqlens=heads) * 2.0

    compiled(f, [x, state, w], 1)


def test_opchecks():
    ops = torch.ops.causal_conv1d_amd
    x, w, state = torch.randn(2, 24, 2, device=DEV), torch.randn(24, 4, device=DEV), torch.randn(2, 24, 5, device=DEV)
    torch.library.opcheck(ops._update_inplace.default, (x, w, None, state, None, None, torch.empty_like(x), True))
    p = scan_make(3, 8, 16, 1, 2, BF16, rows=5)
    idx = torch.tensor([4, -1, 0], dtype=torch.int32, device=DEV)
    torch.library.opcheck(ops._scan_update_inplace.default,
                          (p["u"], p["state"], p["delta"], p["A"], p["B"], p["C"], p["D"], p["z"], p["bias"], True, idx,
                           torch.empty_like(p["u"])))
