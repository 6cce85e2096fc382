"""The native host path of linear attention, its decode step and the norm with rotation gives what the Python code and the
torch.library ops give: bits, strides, dtypes and errors; calls that are not its own go to them."""

from __future__ import annotations

import pytest
import torch

import causal_conv1d_amd as cc
from test_attn_gpu import make, own
from test_attn_update_gpu import call as update_call
from test_attn_update_gpu import make as update_make
from test_rotary_gpu import make as rotary_make
from test_rotary_gpu import own as rotary_own
from test_ssm_host_path_gpu import _same, both  # noqa: F401  (a fixture)

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("layout", ["rows", "heads first", "odd"])
@pytest.mark.parametrize("extra", ["plain", "states", "cu", "scale"])
def test_attn(both, layout, extra, train):  # noqa: F811
    p = make(1, 130, 4, 2, 64, 48, BF16, extra in ("states", "cu"), train, seqs=3 if extra == "cu" else None)
    for n in ("q", "k", "v", "g"):
        if layout == "heads first":
            p[n] = p[n].transpose(1, 2).contiguous().transpose(1, 2)
        if layout == "odd":
            p[n] = torch.stack((p[n], p[n]), -1).flatten(-2)[..., ::2]
    cu = torch.tensor([0, 30, 30, 130], dtype=torch.int32, device=DEV) if extra == "cu" else None
    _same(*both(lambda: own(p, cu, 0.3 if extra == "scale" else None), "linear_attn"))


def test_only_states_wanted(both):  # noqa: F811
    p = make(1, 130, 4, 2, 64, 48, BF16, True, True)
    leaves = [p[n].detach().requires_grad_() for n in ("q", "k", "v", "g")]

    def f():
        out, fin = cc.linear_attn_fn(*leaves, return_final_states=True)
        a = torch.autograd.grad(fin, leaves, p["dfinal"], retain_graph=True)
        b = torch.autograd.grad(out.sum(), leaves[1:2])
        return dict(enumerate((out.detach(), fin.detach(), *a, *b)))

    _same(*both(f, "linear_attn"))


@pytest.mark.parametrize("T", [None, 3])
@pytest.mark.parametrize("pool", [False, True])
def test_update(both, T, pool):  # noqa: F811
    p = update_make(4, T, 4, 2, 64, 48, BF16, rows=6 if pool else None)
    idx = torch.tensor([5, -1, 0, 2], dtype=torch.int32, device=DEV) if pool else None

    def f():
        q = {**p, "state": p["state"].clone()}
        return {"out": update_call(q, idx), "state": q["state"]}

    _same(*both(f, "linear_attn_update"))


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("lead", [(2, 9), (5,)], ids=str)
def test_rotary(both, lead, interleaved, train):  # noqa: F811
    p = rotary_make(lead, 4, 2, 80, 36, BF16, train=train)
    _same(*both(lambda: rotary_own(p, interleaved=interleaved), "head_norm_rotary"))


def test_a_backward_under_create_graph_goes_through_the_op():
    p = make(1, 60, 2, 1, 32, 32, FP32, train=True)
    q = p["q"].detach().requires_grad_()
    out = cc.linear_attn_fn(q, p["k"], p["v"], p["g"])
    a = torch.autograd.grad(out, q, p["dout"], retain_graph=True)[0]
    b = torch.autograd.grad(out, q, p["dout"], create_graph=True)[0]
    assert torch.equal(a, b)


def test_no_grad_records_nothing():
    p = make(1, 20, 2, 1, 32, 32, BF16)
    q = p["q"].detach().requires_grad_()
    with torch.no_grad():
        assert not cc.linear_attn_fn(q, p["k"], p["v"], p["g"]).requires_grad
    with torch.inference_mode():
        out = cc.linear_attn_fn(q, p["k"], p["v"], p["g"])
    assert torch.equal(out, cc.linear_attn_fn(p["q"], p["k"], p["v"], p["g"]))
