"""The native host path of the scan, its decode step and the norm gives what the Python code and the
torch.library ops give: bits, strides, dtypes and errors; calls that are not its own go to them."""

from __future__ import annotations

import pytest
import torch

import causal_conv1d_amd as cc
from causal_conv1d_amd import _host
from test_norm_gpu import make as norm_make
from test_norm_gpu import own as norm_own
from test_scan_gpu import make as scan_make
from test_scan_gpu import own as scan_own
from test_scan_update_gpu import call as update_call
from test_scan_update_gpu import make as update_make

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP32 = torch.bfloat16, torch.float32


class _Off:
    def __getattr__(self, name):
        return lambda *a: NotImplemented


@pytest.fixture
def both(monkeypatch):
    """f() natively (and seen to be), then through Python."""
    def run(f, *names):
        ext, seen = _host.native(), []

        class Spy:
            def __getattr__(self, name):
                def g(*a):
                    r = getattr(ext, name)(*a)
                    seen.append((name, r is not NotImplemented))
                    return r
                return g

        monkeypatch.setattr(_host, "native", lambda: Spy())
        a = f()
        assert [s for s in seen if s[0] in names] == [(n, True) for n in names], seen
        monkeypatch.setattr(_host, "native", lambda: _Off())
        b = f()
        monkeypatch.undo()
        return a, b
    return run


def _same(a, b):
    assert a.keys() == b.keys()
    for k in a:
        assert torch.equal(a[k], b[k]) and a[k].stride() == b[k].stride() and a[k].dtype == b[k].dtype, k


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("layout", ["rows", "last", "odd"])
@pytest.mark.parametrize("extra", ["plain", "states", "ids", "cu"])
def test_scan(both, layout, extra, train):
    p = scan_make(2 if extra != "cu" else 1, 12, 130, 16, 2, BF16, layout, seqs=3 if extra == "cu" else None)
    kw = {}
    if extra == "ids":
        kw["seq_idx"] = (torch.arange(130, dtype=torch.int32, device=DEV) // 50).repeat(2, 1)
    if extra == "cu":
        kw["cu_seqlens"] = torch.tensor([0, 30, 30, 130], dtype=torch.int32, device=DEV)
    if extra in ("states", "cu"):
        kw["init"] = True
    _same(*both(lambda: scan_own(p, True, train=train, **dict(kw)), "ssm_scan"))


def test_scan_without_groups_axis_and_only_states_wanted(both):
    p = scan_make(2, 12, 130, 16, 1, BF16)
    u, B = p["u"].detach().requires_grad_(), p["B"][:, 0].detach().requires_grad_()

    def f():
        out, fin = cc.ssm_scan_fn(u, p["delta"], p["A"], B, p["C"][:, 0], delta_softplus=True, return_final_states=True)
        g = torch.autograd.grad(fin, (u, B), p["dfinal"], retain_graph=True)
        h = torch.autograd.grad(out.sum(), (u, B))
        return dict(enumerate((out.detach(), fin.detach(), *g, *h)))

    _same(*both(f, "ssm_scan"))


@pytest.mark.parametrize("T", [None, 3])
@pytest.mark.parametrize("pool", [False, True])
def test_update(both, T, pool):
    p = update_make(4, 36, 16, 2, T, BF16, rows=6 if pool else None)
    idx = torch.tensor([5, -1, 0, 2], dtype=torch.int32, device=DEV) if pool else None

    def f():
        q = {**p, "state": p["state"].clone()}
        return {"out": update_call(q, idx), "state": q["state"]}

    _same(*both(f, "ssm_scan_update"))


@pytest.mark.parametrize("train", [False, True])
@pytest.mark.parametrize("residual", ["none", "same", "fp32"])
@pytest.mark.parametrize("dim", [64, 300, 9000])
def test_norm(both, dim, residual, train):
    p = norm_make(7, dim, BF16, residual)
    _same(*both(lambda: norm_own(p, train=train), "add_norm"))


def test_norm_of_more_axes(both):
    p = norm_make(6, 64, BF16, "fp32")
    x, r = p["x"].view(2, 3, 64).requires_grad_(), p["residual"].view(2, 3, 64).requires_grad_()

    def f():
        y, s = cc.add_norm_fn(x, p["weight"], p["bias"], residual=r, return_residual=True)
        return dict(enumerate((y.detach(), s.detach(), *torch.autograd.grad(y.float().sum() + s.sum(), (x, r)))))

    _same(*both(f, "add_norm"))


def test_errors_are_the_python_ones():
    p = scan_make(1, 12, 30, 16, 1, BF16)
    with pytest.raises(ValueError, match="delta shape"):
        cc.ssm_scan_fn(p["u"], p["delta"][..., 1:], p["A"], p["B"], p["C"])
    with pytest.raises(NotImplementedError, match="A.dtype"):
        cc.ssm_scan_fn(p["u"], p["delta"], p["A"].bfloat16(), p["B"], p["C"])
    with pytest.raises(NotImplementedError, match="must match u.device"):
        cc.ssm_scan_fn(p["u"], p["delta"], p["A"].cpu(), p["B"], p["C"])
    with pytest.raises(ValueError, match="mutually exclusive"):
        cc.ssm_scan_fn(p["u"], p["delta"], p["A"], p["B"], p["C"], return_final_states=True,
                       seq_idx=torch.zeros(1, 30, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="ssm_state shape"):
        cc.ssm_scan_update(p["u"][..., 0], torch.zeros(2, 12, 16, device=DEV), p["delta"][..., 0], p["A"], p["B"][..., 0],
                           p["C"][..., 0])
    with pytest.raises(ValueError, match="weight shape"):
        cc.add_norm_fn(torch.zeros(3, 8, device=DEV), torch.ones(7, device=DEV))


def test_a_backward_under_create_graph_goes_through_the_op():
    p = scan_make(1, 12, 60, 16, 1, FP32)
    u = p["u"].detach().requires_grad_()
    out = cc.ssm_scan_fn(u, p["delta"], p["A"], p["B"], p["C"], delta_softplus=True)
    a = torch.autograd.grad(out, u, p["dout"], retain_graph=True)[0]
    b = torch.autograd.grad(out, u, p["dout"], create_graph=True)[0]
    assert torch.equal(a, b)
    q = norm_make(5, 64, BF16, "same")
    x = q["x"].detach().requires_grad_()
    y, s = cc.add_norm_fn(x, q["weight"], residual=q["residual"], return_residual=True)
    a = torch.autograd.grad((y, s), x, (q["dy"], q["dsum"]), retain_graph=True)[0]
    b = torch.autograd.grad((y, s), x, (q["dy"], q["dsum"]), create_graph=True)[0]
    assert torch.equal(a, b)


def test_checkpointed_layer():
    from torch.utils.checkpoint import checkpoint

    p = scan_make(1, 12, 300, 16, 1, BF16)
    u = p["u"].detach().requires_grad_()
    f = lambda v: cc.ssm_scan_fn(v, p["delta"], p["A"], p["B"], p["C"], delta_softplus=True)  # noqa: E731
    want = torch.autograd.grad(f(u), u, p["dout"])[0]
    assert torch.equal(torch.autograd.grad(checkpoint(f, u, use_reentrant=False), u, p["dout"])[0], want)
