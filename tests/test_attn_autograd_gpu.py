"""What autograd may do around linear attention and the norm with rotation: hooks on saved tensors see and replace them;
forward mode, vmap and the functional transforms are refused, on either host path, rather than answered without them."""

from __future__ import annotations

import pytest
import torch

import causal_conv1d_amd as cc
from test_attn_gpu import BF16, FP32, make, own
from test_rotary_gpu import make as rotary_make
from test_rotary_gpu import own as rotary_own

# (torch itself imports scripted code for forward mode, and warns of it)
pytestmark = [pytest.mark.gpu, pytest.mark.filterwarnings("ignore:.*torch.jit.script.*:DeprecationWarning")]


def _offloaded(f):
    seen = []

    def pack(t):
        seen.append(t.shape)
        return t.cpu(), t.device

    with torch.autograd.graph.saved_tensors_hooks(pack, lambda p: p[0].to(p[1])):
        return f(), seen


@pytest.mark.parametrize("states", [False, True])
def test_saved_tensors_of_attention_leave_and_come_back(states):
    p = make(1, 130, 4, 2, 64, 48, BF16, states, True)
    want = own(p)
    got, seen = _offloaded(lambda: own(p))
    assert len(seen) == 5 if states else len(seen) == 4
    assert all(torch.equal(got[n], want[n]) for n in want)


def test_saved_tensors_of_the_rotation_leave_and_come_back():
    p = rotary_make((2, 9), 4, 2, 80, 36, BF16, train=True)
    want = rotary_own(p)
    got, seen = _offloaded(lambda: rotary_own(p))
    assert seen and all(torch.equal(got[n], want[n]) for n in want)


def _attn(p):
    return lambda q: cc.linear_attn_fn(q, p["k"], p["v"], p["g"])


def test_forward_mode_is_refused():
    p = make(1, 20, 2, 2, 16, 16, FP32)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.jvp(_attn(p), (p["q"],), (torch.ones_like(p["q"]),))
    with torch.autograd.forward_ad.dual_level():
        q = torch.autograd.forward_ad.make_dual(p["q"], torch.ones_like(p["q"]))
        with pytest.raises((RuntimeError, NotImplementedError)):
            _attn(p)(q)
        with pytest.raises((RuntimeError, NotImplementedError)):
            cc.head_norm_rotary_fn(q, p["k"], torch.ones(16, device="cuda"))


def test_transforms_are_refused():
    p = make(3, 20, 2, 2, 16, 16, FP32)
    one = make(1, 20, 2, 2, 16, 16, FP32)
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.vmap(lambda q: cc.linear_attn_fn(q[None], one["k"], one["v"], one["g"]))(p["q"])
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.grad(lambda q: _attn(one)(q).sum())(one["q"])
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.vmap(lambda q: cc.head_norm_rotary_fn(q[None], one["k"], torch.ones(16, device="cuda"))[0])(p["q"])
    with pytest.raises((RuntimeError, NotImplementedError)):
        torch.func.vmap(lambda q: cc.linear_attn_update(q[None, 0], torch.zeros(1, 2, 16, 16, device="cuda"), one["k"][:, 0],
                                                        one["v"][:, 0], one["g"][:, 0]))(p["q"])
    # and ordinary calls go on
    assert torch.isfinite(_attn(one)(one["q"])).all()


def test_second_derivatives_are_refused():
    p = make(1, 20, 2, 2, 16, 16, FP32, train=True)
    q = p["q"].detach().requires_grad_()
    first = torch.autograd.grad(_attn(p)(q), q, p["dout"], create_graph=True)[0]
    with pytest.raises(RuntimeError):
        torch.autograd.grad(first.sum(), q)
