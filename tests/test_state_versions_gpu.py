"""Decode steps write their states in place, and autograd is told: the backward of a prompt that went on from the same
buffer raises instead of reading what is there by then."""

from __future__ import annotations

import pytest
import torch

import causal_conv1d_amd as cc
from test_attn_gpu import make as attn_make
from test_attn_update_gpu import call as attn_call
from test_attn_update_gpu import make as attn_update_make
from test_scan_gpu import make as scan_make
from test_scan_update_gpu import call as scan_call
from test_scan_update_gpu import make as scan_update_make
from test_ssm_host_path_gpu import both  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _refuses(forward, step, state):
    """Backward before the step works, after it raises; the step moves the version by one or more, not more often than
    its calls."""
    out, leaf = forward(state)
    torch.autograd.grad(out.float().sum(), leaf, retain_graph=True)
    before = state._version
    step(state)
    assert state._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out.float().sum(), leaf)
    out, leaf = forward(state)  # from the buffer as it is now
    torch.autograd.grad(out.float().sum(), leaf)
    return {"v": torch.tensor(state._version - before)}


@pytest.mark.parametrize("pool", [False, True])
def test_linear_attn_update(both, pool):  # noqa: F811
    p = attn_make(2, 40, 4, 2, 64, 64, torch.bfloat16, states=True)
    u = attn_update_make(2, None, 4, 2, 64, 64, torch.bfloat16)
    idx = torch.tensor([1, 0], dtype=torch.int32, device=DEV) if pool else None

    def forward(state):
        q = p["q"].detach().requires_grad_()
        return cc.linear_attn_fn(q, p["k"], p["v"], p["g"], initial_states=state), q

    def f():
        return _refuses(forward, lambda state: attn_call({**u, "state": state}, idx), u["state"].clone())

    a, b = both(f, "linear_attn", "linear_attn_update", "linear_attn")
    assert int(a["v"]) == int(b["v"]) == 1


def test_linear_attn_update_in_inference_mode():
    u = attn_update_make(2, None, 4, 2, 64, 64, torch.bfloat16)
    want = attn_call({**u, "state": u["state"].clone()})
    with torch.inference_mode():
        state = u["state"].clone()  # has no version
        assert torch.equal(attn_call({**u, "state": state}), want)
    assert attn_call({**u, "state": state}).shape == want.shape


@pytest.mark.parametrize("pool", [False, True])
def test_ssm_scan_update(both, pool):  # noqa: F811
    p = scan_make(2, 24, 40, 16, 1, torch.bfloat16)
    u = scan_update_make(2, 24, 16, 1, None, torch.bfloat16)
    idx = torch.tensor([1, 0], dtype=torch.int32, device=DEV) if pool else None

    def forward(state):
        x = p["u"].detach().requires_grad_()
        return cc.ssm_scan_fn(x, p["delta"], p["A"], p["B"], p["C"], initial_states=state), x

    def f():
        return _refuses(forward, lambda state: scan_call({**u, "state": state}, idx), u["state"].clone())

    a, b = both(f, "ssm_scan", "ssm_scan_update", "ssm_scan")
    assert int(a["v"]) == int(b["v"]) == 1


@pytest.mark.parametrize("ring", [False, True])
def test_causal_conv1d_update(both, ring):  # noqa: F811
    w, x, step = (torch.randn(*s, device=DEV) for s in ((24, 4), (2, 24, 40), (2, 24)))
    heads = torch.tensor([0, 2], dtype=torch.int32, device=DEV) if ring else None

    def forward(state):
        leaf = w.clone().requires_grad_()
        return cc.causal_conv1d_fn(x, leaf, initial_states=state), leaf

    def f():
        return _refuses(forward, lambda state: cc.causal_conv1d_update(step, state, w, cache_seqlens=heads),
                        torch.randn(2, 24, 3, device=DEV))

    a, b = both(f, "fn", "update", "fn")
    assert int(a["v"]) == int(b["v"]) == 1
