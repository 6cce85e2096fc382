"""linear_attn_fn where it can go wrong: decays that keep nothing or grow, values that are not finite, layouts, lengths of
zero, offsets past 32 bits, streams, graphs, torch.compile, and bit equality from run to run."""

from __future__ import annotations

import math

import pytest
import torch

import causal_conv1d_amd as cc
from _attn import attn64, close
from test_attn_gpu import BF16, DEV, FP16, FP32, GRADS, TYPES, check, check_packed, compare, make, own

pytestmark = pytest.mark.gpu
NAN, INF = float("nan"), float("inf")


def same(a, b):
    assert a.keys() == b.keys()
    for n in a:
        assert torch.equal(a[n], b[n]), n


@TYPES
@pytest.mark.parametrize("g", [-INF, -1e4, -300.0, 0.0, 0.02], ids=str)
def test_decays(g, dtype):
    """All positions alike, and in places among ordinary ones."""
    p = make(1, 150, 2, 1, 64, 64, dtype, states=True, train=True)
    p["g"][0, [0, 5, 63, 64, 100, 149]] = g
    check(p)
    p["g"][:] = g
    check(p)


@pytest.mark.parametrize("L", [64, 150])
def test_nothing_before_a_decay_of_zero_matters(L):
    p = make(1, L, 2, 2, 64, 64, FP32, states=True)
    p["g"][0, 40] = -INF
    want = own(p)
    p["init"].add_(3.0)
    got = own(p)
    assert torch.equal(got["out"][:, 40:], want["out"][:, 40:]) and torch.equal(got["final"], want["final"])


@TYPES
@pytest.mark.parametrize("bad", [NAN, INF, -INF], ids=str)
@pytest.mark.parametrize("t", [0, 5, 70, 149])
@pytest.mark.parametrize("quick", [True, False])
def test_what_is_not_finite_stays_in_its_rows(t, bad, quick, dtype):
    """A query in its own row; a key or value, or a decay that is NaN, in its own and later rows of its head (a value in
    its own column of them)."""
    p = make(2, 150, 4, 2, 64, 72 if quick else 71, dtype, states=True)
    want = own(p)["out"]
    for name in ("q", "k", "v", "g"):
        if name == "g" and bad != bad:
            hit = {**p, "g": p["g"].clone()}
            hit["g"][1, t, 2] = bad
            heads, cols = [2], slice(None)
        elif name == "g":
            continue
        else:
            hit = {**p, name: p[name].clone()}
            hit[name][1, t, 1, 3] = bad
            heads, cols = ([1], 3) if name == "v" else ([2, 3], slice(None))
        got = own(hit)["out"]
        rest = torch.ones_like(got, dtype=torch.bool)
        for h in heads:
            rest[1, t:t + 1 if name == "q" else None, h, cols] = False
        assert torch.equal(got[rest], want[rest]), name
        assert not got[1, t, heads][..., cols].isfinite().any(), name


@TYPES
def test_gradients_of_what_is_not_finite(dtype):
    """An output gradient reaches its own and earlier rows alone."""
    p = make(1, 150, 2, 2, 64, 64, dtype, train=True)
    want = own(p)
    p["dout"][0, 70, 1, 3] = NAN
    got = own(p)
    for n in ("dq", "dk", "dv", "dg"):
        assert torch.equal(got[n][:, 71:], want[n][:, 71:]) and torch.equal(got[n][:, :, 0], want[n][:, :, 0]), n


@TYPES
def test_packed_sequences_do_not_meet(dtype):
    p = make(1, 400, 2, 1, 64, 64, dtype, states=True, train=True, seqs=3)
    cu = torch.tensor([0, 170, 171, 400], dtype=torch.int32, device=DEV)
    want = own(p, cu)
    hit = {n: None if t is None else t.clone() for n, t in p.items()}
    for n in ("q", "k", "v", "dout"):
        hit[n][0, 170] = NAN
    hit["init"][1] = INF
    got = own(hit, cu)
    for n in want:
        if n in ("final", "dinit"):
            assert torch.equal(got[n][[0, 2]], want[n][[0, 2]]), n
        else:
            assert torch.equal(got[n][:, :170], want[n][:, :170]) and torch.equal(got[n][:, 171:], want[n][:, 171:]), n


def layouts(p, which):
    """The same values, laid out otherwise."""
    def lay(t):
        if which == "heads first":
            return t.transpose(1, 2).contiguous().transpose(1, 2)
        if which == "odd elements":
            return torch.stack((t, t), -1).flatten(-2)[..., ::2]
        if which == "one row to spare":  # rows that begin at any element
            return torch.cat((t, t[..., :1]), -1)[..., :-1]
        if which == "positions first":
            return t.transpose(0, 1).contiguous().transpose(0, 1)
    return {n: lay(t) if n in ("q", "k", "v", "g", "dout") and t is not None else t for n, t in p.items()}


@TYPES
@pytest.mark.parametrize("which", ["heads first", "odd elements", "one row to spare", "positions first"])
def test_layouts(which, dtype):
    p = make(2, 131, 4, 2, 64, 128, dtype, states=True, train=True)
    p["init"], p["dfinal"] = (t.transpose(2, 3).contiguous().transpose(2, 3) for t in (p["init"], p["dfinal"]))
    check(layouts(p, which))


@TYPES
def test_slices_of_one_projection(dtype):
    """q, k and v as they lie next to each other; every fourth position; a decay that all heads share."""
    p = make(2, 200, 4, 4, 64, 64, dtype, train=True)
    one = torch.stack((p["q"], p["k"], p["v"]), 2).flatten(2).clone().unflatten(-1, (3, 4, 64))
    p.update(q=one[:, :, 0], k=one[:, :, 1], v=one[:, :, 2], g=p["g"][:, :, :1].expand(-1, -1, 4))
    check(p)
    check({n: None if t is None or n in ("init", "dfinal") else t[:, ::4] for n, t in p.items()})


def test_a_broadcast_decay_gets_the_sum_of_its_gradients():
    p = make(2, 100, 4, 2, 64, 64, FP32, train=True)
    rate = torch.tensor(-0.05, device=DEV, requires_grad=True)
    out = cc.linear_attn_fn(p["q"], p["k"], p["v"], rate.expand(2, 100, 4))
    got = torch.autograd.grad(out, rate, p["dout"])[0]
    p["g"] = torch.full((2, 100, 4), -0.05, device=DEV)
    e, m = (attn64(*(p[n] for n in ("q", "k", "v", "g")), 64**-0.5, None, p["dout"], mag=x)["dg"] for x in (False, True))
    close(got, e.sum(), m.sum(), 100 * 8, "dg")


def test_expanded_gradient_and_only_states_wanted():
    p = make(1, 90, 2, 1, 64, 64, FP32, states=True, train=True)
    p["dout"] = torch.full((), 0.5, device=DEV).expand(1, 90, 2, 64)
    check(p)
    leaves = {n: p[n].detach().requires_grad_() for n in GRADS}
    args = [leaves[n] for n in ("q", "k", "v", "g")]
    _, fin = cc.linear_attn_fn(*args, initial_states=leaves["init"], return_final_states=True)
    grads = torch.autograd.grad(fin, list(leaves.values()), p["dfinal"])
    p["dout"] = torch.zeros_like(p["v"])
    compare({GRADS[n]: g for n, g in zip(leaves, grads)}, p)
    only = torch.autograd.grad(cc.linear_attn_fn(*args)[0, -1].sum(), (leaves["k"],))[0]
    assert torch.isfinite(only).all()


@TYPES
@pytest.mark.parametrize("B,L", [(2, 0), (0, 5), (0, 0)])
def test_no_positions(B, L, dtype):
    p = make(B, L, 4, 2, 64, 48, dtype, states=True, train=True)
    got = own(p)
    assert got["out"].shape == (B, L, 4, 48) and got["dq"].shape == (B, L, 2, 64)
    assert torch.equal(got["final"], p["init"]) and torch.equal(got["dinit"], p["dfinal"])
    p["init"] = None
    r = cc.linear_attn_fn(p["q"], p["k"], p["v"], p["g"], return_final_states=True)
    assert r[1].shape == (B, 4, 64, 48) and not r[1].any()


def test_packed_sequences_without_positions():
    p = make(1, 0, 2, 2, 64, 64, BF16, states=True, train=True, seqs=2)
    got = own(p, torch.zeros(3, dtype=torch.int32, device=DEV))
    assert torch.equal(got["final"], p["init"]) and torch.equal(got["dinit"], p["dfinal"])


def test_many_short_sequences():
    ends = list(range(0, 601, 3))
    p = make(1, 600, 2, 2, 32, 32, BF16, states=True, train=True, seqs=200)
    got = own(p, torch.tensor(ends, dtype=torch.int32, device=DEV))
    one = {n: None if t is None else (t if n in ("init", "dfinal") else t.view(200, 3, *t.shape[2:])) for n, t in p.items()}
    compare({n: t if n in ("final", "dinit") else t.view(200, 3, *t.shape[2:]) for n, t in got.items()}, one)


@TYPES
def test_long_sequences(dtype):
    """Sequences whose decays' gradients are summed by pieces; a gradient that is not finite stays before its position."""
    p = make(2, 8200, 2, 1, 16, 16, dtype, states=True, train=True)
    check(p)
    want = own(p)
    p["dout"][0, 5000, 1, 3] = NAN
    got = own(p)
    assert torch.equal(got["dg"][:, 5001:], want["dg"][:, 5001:]) and torch.equal(got["dg"][:, :, 0], want["dg"][:, :, 0])
    assert not got["dg"][0, :5000, 1].isfinite().any()
    check_packed(make(1, 9000, 2, 2, 16, 16, dtype, True, True, seqs=4), [3, 5000, 5001, 5001, 8999])


def test_values_past_32_bits():
    """More than 2**31 elements of values and outputs: the last positions are their own."""
    L, H, D, tail = 140000, 128, 128, 96
    small = make(1, tail, H, 1, 64, D, BF16)
    v = torch.zeros(1, L, H, D, dtype=BF16, device=DEV)  # 2.3e9
    q, k = (torch.zeros(1, L, 1, 64, dtype=BF16, device=DEV) for _ in range(2))
    g = torch.zeros(1, L, H, dtype=BF16, device=DEV)
    for t, n in ((q, "q"), (k, "k"), (v, "v"), (g, "g")):
        t[:, -tail:] = small[n]
    out = cc.linear_attn_fn(q, k, v, g)
    assert not out[:, :-tail].any()
    compare({"out": out[:, -tail:, :, :]}, small)


@pytest.mark.parametrize("axis", [0, 1])
def test_strides_past_32_bits(axis):
    """Batch rows 1.1e9 elements apart, or positions 4e7 (no 32-bit offset reaches over a chunk)."""
    p = make(3 if axis == 0 else 1, 70, 2, 2, 64, 64, BF16, train=True)
    for n in ("q", "v", "dout"):
        far = torch.empty((3, 1100000000) if axis == 0 else (70, 40000000), dtype=BF16, device=DEV)
        view = far[:, :70 * 128].view(3, 70, 2, 64) if axis == 0 else far[:, :128].view(1, 70, 2, 64)
        view.copy_(p[n])
        p[n] = view
    check(p)


@TYPES
def test_the_same_bits_again(dtype):
    for kw in ({}, {"cu": torch.tensor([0, 7, 500, 900], dtype=torch.int32, device=DEV)}):
        p = make(1, 900, 4, 2, 128, 64, dtype, states=True, train=True, seqs=3 if kw else None)
        first = own(p, **kw)
        for _ in range(3):
            same(first, own(p, **kw))


def test_two_streams_at_once():
    ps = [make(1, 1500, 4, 2, 128, 128, BF16, states=True, train=True, seed=s) for s in (0, 1)]
    want = [own(p) for p in ps]
    sides = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for p, s in zip(ps, sides):
        with torch.cuda.stream(s):
            got.append(own(p))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        same(a, b)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_graphs(dtype):
    """Forward and backward in two graphs of their own, replayed in turns with eager work in between."""
    names = ("q", "k", "v", "g", "init")
    ps = [make(1, 700, 4, 2, 64, 64, dtype, states=True, train=True, seed=s) for s in (3, 4)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        own(ps[0])
    side.synchronize()
    graphs, outs, leaves = [], [], []
    for p in ps:
        leaf = [p[n].detach().requires_grad_() for n in names]

        def step(leaf=leaf, p=p):
            r = cc.linear_attn_fn(*leaf[:4], initial_states=leaf[4], return_final_states=True)
            return (*r, *torch.autograd.grad(r, leaf, (p["dout"], p["dfinal"])))

        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs.append(step())
        graphs.append(graph)
        leaves.append(leaf)
    for seed in (0, 7, 8):
        new = [make(1, 700, 4, 2, 64, 64, dtype, states=True, train=True, seed=seed + i) for i in (0, 20)]
        for p, n, leaf in zip(ps, new, leaves):
            for name, t in zip(names, leaf):
                t.data.copy_(n[name])
            p["dout"].copy_(n["dout"])
            p["dfinal"].copy_(n["dfinal"])
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for n, out in zip(new, outs):
            want = own(n)
            for got, name in zip(out, ("out", "final", *(GRADS[n] for n in names))):
                assert torch.equal(got, want[name]), (seed, name)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_opcheck(dtype):
    ops = torch.ops.causal_conv1d_amd
    p = make(1, 70, 4, 2, 64, 48, dtype, states=True, train=True, seqs=2)
    cu = torch.tensor([0, 30, 70], dtype=torch.int32, device=DEV)
    args = (p["q"], p["k"], p["v"], p["g"], cu, p["init"], 0.125)
    torch.library.opcheck(ops._attn_fwd_inplace.default, (*args, torch.empty_like(p["v"]), torch.empty_like(p["init"])))
    torch.library.opcheck(ops._attn_bwd_inplace.default,
                          (*args, p["dout"], p["dfinal"], *(torch.empty_like(p[n]) for n in ("q", "k", "v", "g", "init"))))


def test_compile_fullgraph():
    p = make(1, 130, 4, 2, 64, 64, BF16, states=True, train=True)
    leaves = [p[n].detach().requires_grad_() for n in ("q", "k", "v", "g", "init")]

    def f(q, k, v, g, init):
        out, fin = cc.linear_attn_fn(q, k, v, g, initial_states=init, return_final_states=True)
        return out * 2.0, fin

    want = f(*leaves)
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(*leaves)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for a, b in zip(*(torch.autograd.grad(r, leaves, (p["dout"], p["dfinal"])) for r in (want, got))):
        assert torch.equal(a, b)


def test_half_precision_extremes():
    """fp16's largest values: sums are formed in 32 bits, and only what leaves is rounded to 16 (to infinity beyond)."""
    p = make(1, 40, 1, 1, 64, 64, FP16)
    p["q"].fill_(0.0)
    p["q"][..., 0] = 1.0
    p["k"].fill_(0.0)
    p["k"][..., 0] = 65504.0
    p["v"].fill_(1.0)
    p["g"].fill_(0.0)
    out = cc.linear_attn_fn(p["q"], p["k"], p["v"], p["g"], scale=1.0)
    assert (out[0, 0] == 65504.0).all() and (out[0, 1:] == INF).all()
    out = cc.linear_attn_fn(p["q"], p["k"], p["v"], p["g"], scale=1 / 64)
    e = 65504.0 / 64 * torch.arange(1, 41, dtype=torch.float64)[None, :, None, None].expand(1, 40, 1, 64)
    close(out, e, e, 40)


def test_refused_on_the_gpu_as_in_python():
    p = make(1, 8, 2, 1, 16, 16, BF16)
    with pytest.raises(ValueError, match="k shape"):
        cc.linear_attn_fn(p["q"], p["k"][:, :7], p["v"], p["g"])
    with pytest.raises(NotImplementedError, match="g.dtype"):
        cc.linear_attn_fn(p["q"], p["k"], p["v"], p["g"].float())
    with pytest.raises(NotImplementedError, match="head size"):
        cc.linear_attn_fn(*(torch.zeros(1, 8, 1, 129, dtype=BF16, device=DEV) for _ in range(3)), p["g"][..., :1])
    with pytest.raises(ValueError, match="multiple"):
        cc.linear_attn_fn(p["q"].expand(1, 8, 3, 16), p["k"].expand(1, 8, 3, 16), p["v"], p["g"])
    with pytest.raises(ValueError, match="batch == 1"):
        cc.linear_attn_fn(*(p[n].expand(2, *p[n].shape[1:]) for n in ("q", "k", "v", "g")),
                          cu_seqlens=torch.zeros(2, dtype=torch.int32, device=DEV))
    with pytest.raises(ValueError, match="initial_states shape"):
        cc.linear_attn_fn(p["q"], p["k"], p["v"], p["g"], initial_states=torch.zeros(1, 2, 16, 15, device=DEV))
    assert math.isfinite(cc.linear_attn_fn(p["q"], p["k"], p["v"], p["g"]).float().sum().item())
