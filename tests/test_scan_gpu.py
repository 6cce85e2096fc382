"""ssm_scan_fn on the GPU against its definition in float64 (``_ssm.py``): every
option, type and layout at the sizes where tiles, lanes, groups and states begin
and end, the gradients of every argument, packed sequences, states, padding that
holds anything, streams, graphs, torch.compile, and bit equality from run to run."""

from __future__ import annotations

import pytest
import torch

import causal_conv1d_amd as cc
from _ssm import close, scan64

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
GRADS = {"u": "du", "delta": "ddelta", "A": "dA", "B": "dB", "C": "dC", "D": "dD", "z": "dz", "bias": "dbias",
         "init": "dinit"}


def lay(t, layout):
    """t's values as a GPU tensor whose last axis lies as said."""
    t = t.to(DEV)
    if layout == "last":  # time strided, the axis before it contiguous
        return t.transpose(-1, -2).contiguous().transpose(-1, -2)
    if layout == "odd":  # no unit stride anywhere, an offset start
        big = torch.zeros(*t.shape[:-1], 2 * t.shape[-1] + 3, dtype=t.dtype, device=DEV)
        v = big[..., 3::2][..., :t.shape[-1]]
        return v.copy_(t)
    if layout == "slice":  # unit time stride, rows that start anywhere
        big = torch.zeros(*t.shape[:-1], t.shape[-1] + 5, dtype=t.dtype, device=DEV)
        v = big[..., 3:3 + t.shape[-1]]
        return v.copy_(t)
    return t.contiguous()


def make(B, D, L, N, G, dtype, layout="rows", gate=True, bias=True, skip=True, seed=0, seqs=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    p = {"u": r(B, D, L).to(dtype), "delta": (0.5 * r(B, D, L) - 1.0).to(dtype), "A": -2.0 * torch.rand(D, N, generator=g),
         "B": r(B, G, N, L).to(dtype), "C": r(B, G, N, L).to(dtype), "D": r(D) if skip else None,
         "z": r(B, D, L).to(dtype) if gate else None, "bias": 0.5 * r(D) if bias else None,
         "init": r(seqs or B, D, N), "dout": r(B, D, L).to(dtype), "dfinal": r(seqs or B, D, N)}
    wide = ("u", "delta", "B", "C", "z", "dout")
    return {k: None if v is None else (lay(v, layout) if k in wide else v.to(DEV)) for k, v in p.items()}


def own(p, softplus, train=True, **kw):
    """Results and gradients of ssm_scan_fn by the names of scan64."""
    leaves = {k: p[k].detach().requires_grad_(train) for k in GRADS if p.get(k) is not None and (k != "init" or "init" in kw)}
    init = leaves.get("init")
    states = kw.pop("init", None) is not None
    r = cc.ssm_scan_fn(leaves["u"], leaves["delta"], leaves["A"], leaves["B"], leaves["C"], D=leaves.get("D"),
                       z=leaves.get("z"), delta_bias=leaves.get("bias"), delta_softplus=softplus, initial_states=init,
                       return_final_states=states, **kw)
    got = {"out": r[0], "final": r[1]} if states else {"out": r}
    assert got["out"].dtype == p["u"].dtype and got["out"].shape == p["u"].shape
    if train:
        grads = torch.autograd.grad(r, list(leaves.values()), (p["dout"], p["dfinal"]) if states else p["dout"])
        for k, g in zip(leaves, grads):
            assert g.shape == leaves[k].shape and g.dtype == leaves[k].dtype, k
            got[GRADS[k]] = g
    return {k: v.detach() for k, v in got.items()}


def exact(p, softplus, ids=None, states=False, mag=False):
    return scan64(p["u"], p["delta"], p["A"], p["B"], p["C"], p["D"], p["z"], p["bias"], softplus, ids,
                  p["init"] if states else None, p["dout"], p["dfinal"] if states else None, mag)


def check(p, softplus=True, ids=None, states=False, **kw):
    got = own(p, softplus, seq_idx=None if ids is None else ids.to(DEV), **({"init": True} if states else {}), **kw)
    e, s = exact(p, softplus, ids, states), exact(p, softplus, ids, states, mag=True)
    L = p["u"].shape[2] * (p["u"].shape[0] + p["u"].shape[1])
    for k, v in got.items():
        close(v, e[k], s[k], L, k)


SIZES = [(1, 1, 1, 1, 1), (2, 3, 5, 4, 1), (1, 8, 64, 16, 1), (2, 4, 131, 3, 2), (1, 5, 255, 16, 1), (2, 6, 256, 16, 2),
         (1, 9, 257, 7, 3), (1, 16, 511, 16, 4), (1, 33, 512, 8, 1), (2, 4, 513, 17, 1), (1, 3, 1030, 64, 1),
         (1, 2, 300, 256, 1), (1, 130, 40, 16, 2), (3, 40, 1025, 16, 1), (1, 17, 1536, 33, 1)]


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("layout", ["rows", "last", "slice", "odd"])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes_and_layouts(size, layout, dtype):
    B, D, L, N, G = size
    check(make(B, D, L, N, G, dtype, layout, seed=L), states=(L % 2 == 1))


@pytest.mark.parametrize("layout", ["rows", "last"])
@pytest.mark.parametrize("softplus", [False, True])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("skip", [False, True])
def test_options(skip, bias, gate, softplus, layout):
    p = make(2, 20, 300, 16, 2, BF16, layout, gate, bias, skip)
    if not softplus:  # raw steps are negative here: with decaying states for them, all within fp32's range
        p["A"] = -p["A"]
        p["delta"] = p["delta"].abs().neg() if not bias else p["delta"].abs().neg() - 3.0
    check(p, softplus=softplus, states=gate)


def runs(B, L, seed=0, padding=True):
    """Ids in runs of random lengths, some of them padding (< 0), some repeated after another id."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.empty(B, L, dtype=torch.int32)
    for b in range(B):
        t, last = 0, None
        while t < L:
            n = int(torch.randint(1, max(2, L // 3), (1,), generator=g)) if torch.rand(1, generator=g) < 0.6 else 1
            v = int(torch.randint(-2 if padding else 0, 4, (1,), generator=g))
            if v != last:
                ids[b, t:t + n] = v
                t, last = t + n, v
    return ids


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("layout", ["rows", "last", "odd"])
@pytest.mark.parametrize("size", [(2, 5, 7, 16, 1), (2, 4, 100, 3, 2), (1, 18, 256, 16, 1), (2, 6, 700, 16, 1),
                                  (1, 3, 1100, 40, 1)], ids=str)
def test_packed_rows(size, layout, dtype):
    B, D, L, N, G = size
    check(make(B, D, L, N, G, dtype, layout, seed=3), ids=runs(B, L, seed=L))


def relay(p, layout, *names):
    """p with some of its tensors laid out another way."""
    return {**p, **{k: lay(p[k], layout) for k in names}}


@pytest.mark.parametrize("packed", [False, True], ids=["plain", "packed"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("pair", [("rows", "last"), ("last", "rows"), ("slice", "last"), ("last", "slice"), ("rows", "odd"),
                                  ("last", "odd")], ids="+".join)
@pytest.mark.parametrize("size", [(2, 20, 200, 16, 2), (1, 9, 1100, 24, 1), (1, 34, 60, 9, 2), (2, 40, 650, 16, 1)], ids=str)
def test_layout_pairs(size, pair, dtype, packed):
    """u, delta, z and dout one way, B and C another (as slices of a projection are beside rows from the convolution)."""
    B, D, L, N, G = size
    p = relay(make(B, D, L, N, G, dtype, pair[0], seed=L), pair[1], "B", "C")
    check(p, ids=runs(B, L, seed=D) if packed else None, states=not packed)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("bc", ["last", "rows"])
@pytest.mark.parametrize("size", [(1, 17, 300, 200, 1), (2, 9, 530, 131, 1), (1, 24, 90, 256, 2)], ids=str)
def test_channel_last_with_many_states(size, bc, dtype):
    B, D, L, N, G = size
    check(relay(make(B, D, L, N, G, dtype, "last", seed=N), bc, "B", "C"), states=True)


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("base", ["rows", "last"])
@pytest.mark.parametrize("other", ["u", "delta", "z", "dout", "C"])
@pytest.mark.parametrize("size", [(2, 20, 200, 16, 2), (1, 18, 600, 20, 1)], ids=str)
def test_one_tensor_lies_otherwise(size, other, base, dtype):
    B, D, L, N, G = size
    p = make(B, D, L, N, G, dtype, base, seed=L)
    for layout in ("last" if base == "rows" else "rows", "odd"):
        check(relay(p, layout, other), states=True)


# More channels than the card takes at once: two a wavefront, and several rounds, in the backward's blocks.
@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("layout", ["rows", "last", "odd"])
@pytest.mark.parametrize("size", [(1, 4100, 21, 16, 1), (1, 4107, 520, 5, 1), (2, 1030, 300, 9, 1), (2, 4104, 21, 17, 2),
                                  (9, 4100, 6, 3, 1)],
                         ids=str)
@pytest.mark.parametrize("packed", [False, True], ids=["plain", "packed"])
def test_many_channels(packed, size, layout, dtype):
    B, D, L, N, G = size
    check(make(B, D, L, N, G, dtype, layout, seed=5), ids=runs(B, L, seed=L) if packed else None, states=not packed)


@pytest.mark.parametrize("packed", [False, True], ids=["plain", "packed"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("pair", [("rows", "last"), ("last", "rows")], ids="+".join)
@pytest.mark.parametrize("L", [200, 520])
def test_layout_pairs_of_many_channels(L, pair, dtype, packed):
    p = relay(make(1, 4107, L, 9, 1, dtype, pair[0], seed=L), pair[1], "B", "C")
    check(p, ids=runs(1, L, seed=L) if packed else None, states=not packed)


def test_every_position_its_own_sequence_and_only_padding():
    p = make(2, 6, 300, 16, 1, FP32)
    check(p, ids=torch.arange(300, dtype=torch.int32).repeat(2, 1))
    ids = torch.full((2, 300), -1, dtype=torch.int32)
    ids[1, 100:] = 7  # row 0 holds nothing
    check(p, ids=ids)


@pytest.mark.parametrize("hole", [float("nan"), float("inf")])
@pytest.mark.parametrize("layout", ["rows", "last"])
def test_padding_may_hold_anything(layout, hole):
    ids = runs(2, 600, seed=5)
    p = make(2, 18, 600, 16, 1, BF16, layout, seed=1)
    for k in ("u", "delta", "z", "dout"):
        p[k].masked_fill_((ids < 0).to(DEV)[:, None], hole)
    for k in ("B", "C"):
        p[k].masked_fill_((ids < 0).to(DEV)[:, None, None], hole)
    check(p, ids=ids)
    for k, v in own(p, True, seq_idx=ids.to(DEV)).items():
        assert torch.isfinite(v).all(), k


@pytest.mark.parametrize("hole", [float("nan"), float("inf")])
def test_a_sequence_does_not_reach_the_next(hole):
    """A non-finite value of one packed sequence stays with it, in outputs and in gradients."""
    ids = torch.zeros(1, 700, dtype=torch.int32)
    ids[:, 130:400], ids[:, 400:] = 1, 2
    p = make(1, 18, 700, 16, 1, FP32, seed=2)
    clean = own(p, True, seq_idx=ids.to(DEV))
    p["u"][:, :, 200] = hole
    got = own(p, True, seq_idx=ids.to(DEV))
    for k in ("out", "dz", "du", "ddelta"):
        assert torch.equal(got[k][..., :130], clean[k][..., :130]) and torch.equal(got[k][..., 400:], clean[k][..., 400:]), k
    assert not torch.isfinite(got["out"][..., 200:400]).any()
    cu = torch.tensor([0, 130, 400, 700], dtype=torch.int32, device=DEV)
    p["init"] = torch.zeros(3, 18, 16, device=DEV)
    p["dfinal"] = torch.zeros_like(p["init"])
    packed = own(p, True, cu_seqlens=cu, init=True)
    for k in ("out", "du", "ddelta"):
        assert torch.equal(packed[k][..., :130], clean[k][..., :130]), k
        assert torch.isfinite(packed[k][..., 400:]).all(), k
    assert not torch.isfinite(packed["final"][1]).any() and torch.isfinite(packed["final"][[0, 2]]).all()


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("layout", ["rows", "last", "odd"])
@pytest.mark.parametrize("ends", [[0, 1], [0, 5, 5, 6, 300, 300], [0, 0, 256, 512, 1030], [0, 131, 643]], ids=str)
def test_packed_prompts(ends, layout, dtype):
    """cu_seqlens: every sequence is what it is alone, states and gradients included; empty ones keep their state."""
    D, N, G, L, n = 18, 16, 2, ends[-1], len(ends) - 1
    p = make(1, D, L, N, G, dtype, layout, seed=4, seqs=n)
    got = own(p, True, cu_seqlens=torch.tensor(ends, dtype=torch.int32, device=DEV), init=True)
    total = {k: [torch.zeros_like(v) for v in (got[k].double().cpu(),) * 2] for k in ("dA", "dD", "dbias")}
    for i, (a, b) in enumerate(zip(ends, ends[1:])):
        q = {k: v[..., a:b] if k in ("u", "delta", "z", "B", "C", "dout") else
             (v[i:i + 1] if k in ("init", "dfinal") else v) for k, v in p.items()}
        e, s = exact(q, True, states=True), exact(q, True, states=True, mag=True)
        for k in total:
            total[k][0] += e[k]
            total[k][1] += s[k]
        for k in ("out", "dz", "du", "ddelta", "dB", "dC"):
            close(got[k][..., a:b], e[k], s[k], L * D, k)
        close(got["final"][i:i + 1], e["final"], s["final"], L, "final")
        close(got["dinit"][i:i + 1], e["dinit"], s["dinit"], L, "dinit")
        if a == b:
            assert torch.equal(got["final"][i], p["init"][i]) and torch.equal(got["dinit"][i], p["dfinal"][i])
    for k, (e, s) in total.items():
        close(got[k], e, s, L * D, k)


def test_positions_outside_cu_seqlens_are_zero():
    p = make(1, 20, 900, 16, 1, BF16, seqs=2)
    for k in ("u", "delta", "z", "dout", "B", "C"):  # what lies there does not count
        p[k][..., :70], p[k][..., 650:] = float("nan"), float("inf")
    got = own(p, True, cu_seqlens=torch.tensor([70, 400, 650], dtype=torch.int32, device=DEV), init=True)
    for k in ("out", "du", "ddelta", "dz", "dB", "dC"):
        assert (got[k][..., :70] == 0).all() and (got[k][..., 650:] == 0).all(), k
    for k, v in got.items():
        assert torch.isfinite(v).all(), k


def test_no_positions():
    for B, D in ((2, 5), (0, 5), (2, 0)):
        p = make(B, D, 0 if B * D else 9, 16, 1, BF16, gate=True)
        got = own(p, True, init=True)
        assert torch.equal(got["final"], p["init"]) if B * D else got["out"].numel() == 0
        assert all((got[k] == 0).all() for k in ("dA", "dD", "dbias"))


@pytest.mark.parametrize("dtype", [BF16, FP32], ids=["bf16", "fp32"])
@pytest.mark.parametrize("prompts", [False, True])
def test_no_channels(prompts, dtype):
    """B and C of a layer without channels have gradients, of zeros."""
    p = make(1 if prompts else 2, 0, 700, 16, 2, dtype)
    for _ in range(4):  # (what their memory held before is not zeros)
        torch.full_like(p["B"], float("nan"))
    kw = {"cu_seqlens": torch.tensor([0, 300, 700], dtype=torch.int32, device=DEV)} if prompts else {}
    got = own(p, True, **kw)
    for k in ("dB", "dC"):
        assert got[k].shape == p["B"].shape and (got[k] == 0).all(), k


def test_extreme_steps():
    """Decays that underflow to 0, steps of 0 (a state that stays), large raw steps, growing states."""
    p = make(1, 16, 600, 16, 1, FP32, seed=9)
    p["delta"][:, :4] = 60.0    # exp(-60 * |A|): 0 in fp32 for most states
    p["delta"][:, 4:8] = -200.0  # softplus underflows to 0
    p["delta"][:, 8:12] = 25.0
    p["A"][12:] = 0.01           # |a| > 1
    check(p, states=True)


def live_channels(p, live):
    """p with u and dout 0 in all channels but those, and the part of it that they are: the others add nothing."""
    rest = torch.ones(p["u"].shape[1], dtype=torch.bool, device=DEV)
    rest[live] = False
    for k in ("u", "dout", "init", "dfinal"):
        p[k][:, rest] = 0
    return {k: v if v is None or k in ("B", "C") else (v[live] if k in ("A", "D", "bias") else v[:, live])
            for k, v in p.items()}


@pytest.mark.parametrize("layout", ["rows", "last"])
@pytest.mark.parametrize("size", [(1, 8192, 4300, 256), (3, 4096, 2800, 256)], ids=str)
def test_backward_in_parts_of_the_sequence(size, layout):
    """More shares of dB and dC than a launch takes: tiles in several launches."""
    B, D, L, N = size
    p = make(B, D, L, N, 1, BF16, layout, seed=8)
    live = torch.tensor([0, 7, 8, 300, 1023, 1024, 1500, D - 9, D - 1], device=DEV)
    part = live_channels(p, live)
    got = own(p, True, init=True)
    e, s = exact(part, True, states=True), exact(part, True, states=True, mag=True)
    for k, v in got.items():
        pick = v if k in ("dB", "dC") else (v[live] if k in ("dA", "dD", "dbias") else v[:, live])
        close(pick, e[k], s[k], L * (B + D), k)


@pytest.mark.parametrize("size", [(8300, 128, 64, 256), (1800, 64, 300, 256), (1040, 64, 700, 256)], ids=str)
def test_backward_in_parts_of_the_batch(size):
    """More shares of one tile than a launch takes: rows in several launches. A row is what it is alone."""
    B, D, L, N = size
    p = make(B, D, L, N, 1, BF16, seed=9)
    got = own(p, True, init=True)
    rows = torch.tensor([0, B // 3, B // 2 - 1, B // 2, B // 2 + 1, B - 1], device=DEV)
    few = {k: v if k in ("A", "D", "bias") else v[rows] for k, v in p.items()}
    e, s = exact(few, True, states=True), exact(few, True, states=True, mag=True)
    for k, v in got.items():
        if k not in ("dA", "dD", "dbias"):
            close(v[rows], e[k], s[k], L * (B + D), k)
    dA = torch.zeros_like(p["A"], dtype=torch.float64)  # the parameters' gradients: of parts that one launch takes
    mag = torch.zeros_like(dA)
    for at in torch.arange(B, device=DEV).split(500):
        one = own({k: v if k in ("A", "D", "bias") else v[at] for k, v in p.items()}, True, init=True)
        dA += one["dA"].double()
        mag += one["dA"].double().abs()
    assert ((got["dA"].double() - dA).abs() <= 4 * B * 2.0**-24 * mag + 1e-6).all()


def test_states_carry_over_chunks():
    """A prompt in pieces, the state handed on, is the prompt at once (up to fp32 rounding)."""
    p = make(2, 24, 1500, 16, 1, FP32, "rows")
    whole, final = cc.ssm_scan_fn(p["u"], p["delta"], p["A"], p["B"], p["C"], p["D"], p["z"], p["bias"], True,
                                  return_final_states=True)
    state, parts = None, []
    for a, b in ((0, 1), (1, 300), (300, 812), (812, 1500)):
        o, state = cc.ssm_scan_fn(*(p[k][..., a:b] if k in ("u", "delta", "B", "C", "z") else p[k]
                                    for k in ("u", "delta", "A", "B", "C", "D", "z", "bias")), True,
                                  initial_states=state, return_final_states=True)
        parts.append(o)
    torch.testing.assert_close(torch.cat(parts, -1), whole, rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(state, final, rtol=1e-4, atol=1e-4)


def test_broadcast_inputs():
    """Expanded tensors are read through their strides, and their gradients come back in full."""
    p = make(2, 20, 140, 16, 1, FP32)
    one = p["delta"][:, :1].expand(-1, 20, -1)  # one step for all channels
    B = p["B"][:1].expand(2, -1, -1, -1)
    A = p["A"][:, :1].expand(-1, 16)
    q = {**p, "delta": one, "B": B, "A": A}
    check(q)


def test_only_some_gradients():
    p = make(1, 20, 300, 16, 1, BF16)
    full = own(p, True)
    u = p["u"].detach().requires_grad_()
    out = cc.ssm_scan_fn(u, p["delta"], p["A"], p["B"], p["C"], p["D"], p["z"], p["bias"], True)
    assert torch.equal(out, full["out"])
    assert torch.equal(torch.autograd.grad(out, u, p["dout"])[0], full["du"])
    fin = cc.ssm_scan_fn(u, p["delta"], p["A"], p["B"], p["C"], p["D"], p["z"], p["bias"], True,
                         return_final_states=True)[1]
    torch.autograd.grad(fin.sum(), u)  # the states' gradient alone


@pytest.mark.parametrize("layout", ["rows", "last"])
def test_same_bits_every_time(layout):
    p = make(2, 200, 1100, 16, 2, BF16, layout)
    first = own(p, True, init=True)
    for _ in range(3):
        again = own(p, True, init=True)
        for k, v in first.items():
            assert torch.equal(v, again[k]), k


def test_side_stream_and_graph():
    p = make(1, 64, 700, 16, 1, BF16)
    want = own(p, True, init=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = own(p, True, init=True)
    side.synchronize()
    for k, v in want.items():
        assert torch.equal(v, got[k]), k
    leaves = [p[k].detach().requires_grad_() for k in ("u", "delta", "A", "B", "C", "D", "z", "bias", "init")]

    def step():
        out, fin = cc.ssm_scan_fn(*leaves[:5], D=leaves[5], z=leaves[6], delta_bias=leaves[7], delta_softplus=True,
                                  initial_states=leaves[8], return_final_states=True)
        return (out, fin, *torch.autograd.grad((out, fin), leaves, (p["dout"], p["dfinal"])))

    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step()
    for seed in (0, 7, 8):  # new values in the same tensors, eager work in between
        new = make(1, 64, 700, 16, 1, BF16, seed=seed)
        for k, t in zip(("u", "delta", "A", "B", "C", "D", "z", "bias", "init"), leaves):
            t.data.copy_(new[k])
        p["dout"].copy_(new["dout"])
        p["dfinal"].copy_(new["dfinal"])
        graph.replay()
        torch.cuda.synchronize()
        want = own({**new}, True, init=True)
        for got, k in zip(outs, ("out", "final", "du", "ddelta", "dA", "dB", "dC", "dD", "dz", "dbias", "dinit")):
            assert torch.equal(got, want[k]), (seed, k)


def test_compile_fullgraph():
    p = make(1, 32, 300, 16, 1, BF16)
    leaves = [p[k].detach().requires_grad_() for k in ("u", "delta", "A", "B", "C")]

    def f(u, delta, A, B, C):
        return cc.ssm_scan_fn(u, delta, A, B, C, D=p["D"], z=p["z"], delta_bias=p["bias"], delta_softplus=True) * 2.0

    want = f(*leaves)
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(*leaves)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(want, leaves, p["dout"]), torch.autograd.grad(got, leaves, p["dout"])):
        assert torch.equal(a, b)


def test_long_rows_past_32_bits():
    """More than 2**31 elements: the last batch row's values are its own."""
    D, L = 4096, 131072
    B = 5  # 2.7e9 elements of u
    u = torch.zeros(B, D, L, dtype=BF16, device=DEV)
    small = make(1, 64, 2048, 4, 1, BF16, gate=False, seed=6)
    u[-1, -64:, -2048:] = small["u"][0]
    delta = torch.full((1, 1, 1), -1.0, dtype=BF16, device=DEV).expand(B, D, L)
    Bm, Cm = (torch.zeros(1, 1, 4, L, dtype=BF16, device=DEV) for _ in range(2))
    Bm[..., -2048:], Cm[..., -2048:] = small["B"], small["C"]
    A = torch.zeros(D, 4, device=DEV)
    A[-64:] = small["A"]
    out = cc.ssm_scan_fn(u, delta, A, Bm.expand(B, -1, -1, -1), Cm.expand(B, -1, -1, -1), delta_softplus=True)
    small["delta"] = torch.full_like(small["delta"], -1.0)
    e = [scan64(small["u"], small["delta"], small["A"], small["B"], small["C"], softplus=True, mag=m)["out"] for m in (0, 1)]
    close(out[-1:, -64:, -2048:], e[0], e[1], L, "out")
    assert (out[:-1] == 0).all() and (out[-1, :-64] == 0).all()
