"""head_norm_rotary_fn: numbers of heads against wavefronts, offsets past 32 bits, graphs with gradients, torch.compile."""

from __future__ import annotations

import pytest
import torch

import causal_conv1d_amd as cc
from test_rotary_gpu import BF16, DEV, FP16, FP32, check, make, own

pytestmark = pytest.mark.gpu
TYPES = pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])


@TYPES
@pytest.mark.parametrize("dim,rotated", [(8, 8), (128, 128), (128, 60), (256, 128), (250, 250)], ids=str)
@pytest.mark.parametrize("heads", [(1, 1), (5, 4), (17, 1), (2, 33)], ids=str)
def test_heads(heads, dim, rotated, dtype):
    """Fewer heads than a stop of a wavefront takes, some more, queries and keys unlike."""
    check(make((2, 3), *heads, dim, rotated, dtype, train=True))


@TYPES
@pytest.mark.parametrize("which", ["heads first", "odd elements", "rows that begin anywhere"])
def test_layouts(which, dtype):
    p = make((2, 70), 4, 2, 64, 64, dtype, train=True)
    for n in ("q", "k", "dq", "dk"):
        t = p[n]
        if which == "heads first":
            p[n] = t.transpose(1, 2).contiguous().transpose(1, 2)
        elif which == "odd elements":
            p[n] = torch.stack((t, t), -1).flatten(-2)[..., ::2]
        else:
            p[n] = torch.cat((t, t[..., :1]), -1)[..., :-1]
    check(p)


@pytest.mark.parametrize("rotated", [64, 36])
def test_values_past_32_bits(rotated):
    """More than 2**31 elements of q: the last tokens are their own."""
    L, H, D, tail = 140000, 128, 128, 40
    small = make((1, tail), H, 1, D, rotated, BF16)
    q = torch.zeros(1, L, H, D, dtype=BF16, device=DEV)
    k = torch.zeros(1, L, 1, D, dtype=BF16, device=DEV)
    pos = torch.zeros(1, L, dtype=torch.int64, device=DEV)
    q[:, -tail:], k[:, -tail:], pos[:, -tail:] = small["q"], small["k"], torch.arange(tail, device=DEV)
    a, b = cc.head_norm_rotary_fn(q, k, small["wq"], small["wk"], small["freq"], pos)
    want = own(small)
    assert torch.equal(a[:, -tail:], want["q"]) and torch.equal(b[:, -tail:], want["k"])
    assert not a[:, :-tail].any()


@pytest.mark.parametrize("axis", [0, 1])
def test_strides_past_32_bits(axis):
    """Batch rows or tokens 1.1e9 elements apart."""
    p = make((3, 1) if axis == 0 else (1, 3), 4, 2, 64, 64, BF16, train=True)
    for n in ("q", "dq"):
        far = torch.empty(3, 1100000000, dtype=BF16, device=DEV)
        view = far[:, :256].view(3, 1, 4, 64) if axis == 0 else far[:, :256].view(1, 3, 4, 64)
        view.copy_(p[n])
        p[n] = view
    check(p)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_graphs(dtype):
    """Forward and backward in two graphs of their own, replayed in turns with eager work in between."""
    names = ("q", "k", "wq", "wk")
    ps = [make((2, 300), 4, 2, 64, 48, dtype, train=True, seed=s) for s in (3, 4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        own(ps[0])
    side.synchronize()
    graphs, outs, leaves = [], [], []
    for p in ps:
        leaf = [p[n].detach().requires_grad_() for n in names]

        def step(leaf=leaf, p=p):
            r = cc.head_norm_rotary_fn(*leaf, p["freq"])
            return (*r, *torch.autograd.grad(r, leaf, (p["dq"], p["dk"])))

        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(step())
        graphs.append(graph)
        leaves.append(leaf)
    for seed in (0, 7, 8):
        new = [make((2, 300), 4, 2, 64, 48, dtype, train=True, seed=seed + i) for i in (0, 20)]
        for p, n, leaf in zip(ps, new, leaves):
            for name, t in zip(names, leaf):
                t.data.copy_(n[name])
            p["dq"].copy_(n["dq"])
            p["dk"].copy_(n["dk"])
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for n, out in zip(new, outs):
            want = own(n)
            for got, name in zip(out, ("q", "k", "dq", "dk", "dwq", "dwk")):
                assert torch.equal(got, want[name]), (seed, name)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_opcheck(dtype):
    ops = torch.ops.causal_conv1d_amd
    p = make((2, 5), 4, 2, 64, 48, dtype, train=True)
    args = (p["q"], p["k"], p["wq"], p["wk"], p["freq"], None, 1e-6, False, 1.0)
    torch.library.opcheck(ops._rotary_fwd_inplace.default, (*args, torch.empty_like(p["q"]), torch.empty_like(p["k"])))
    torch.library.opcheck(ops._rotary_bwd_inplace.default,
                          (*args, p["dq"], p["dk"], *(torch.empty_like(p[n]) for n in ("q", "k", "wq", "wk"))))


def test_compile_fullgraph():
    p = make((2, 30), 4, 2, 64, 64, BF16, train=True)
    leaves = [p[n].detach().requires_grad_() for n in ("q", "k", "wq", "wk")]

    def f(q, k, wq, wk):
        a, b = cc.head_norm_rotary_fn(q, k, wq, wk, p["freq"])
        return a * 2.0, b

    want = f(*leaves)
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for a, b in zip(*(torch.autograd.grad(r, leaves, (p["dq"], p["dk"])) for r in (want, got))):
        assert torch.equal(a, b)


def test_only_one_output_wanted():
    p = make((2, 9), 4, 2, 64, 64, FP32, train=True)
    leaves = [p[n].detach().requires_grad_() for n in ("q", "k", "wq", "wk")]
    q, k = cc.head_norm_rotary_fn(*leaves, p["freq"])
    got = torch.autograd.grad(k, leaves, p["dk"], allow_unused=True)
    want = own(p)
    assert torch.equal(got[1], want["dk"]) and torch.equal(got[3], want["dwk"])
    assert all(g is None or not g.any() for g in (got[0], got[2]))
