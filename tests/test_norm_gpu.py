"""add_norm_fn on the GPU against its definition in float64: every type pair, option and width where vectors,
wavefronts and rows begin and end, and the gradients."""

from __future__ import annotations

import pytest
import torch

import causal_conv1d_amd as cc
from _ssm import close, norm64

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def make(rows, dim, dtype, residual, bias=True, seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
    wide = {"none": None, "same": dtype, "fp32": FP32}[residual]
    return {"x": (r(rows, dim) + 0.5).to(dtype), "weight": 1.0 + 0.3 * r(dim), "bias": r(dim) if bias else None,
            "residual": None if wide is None else (2.0 * r(rows, dim)).to(wide), "dy": r(rows, dim).to(dtype),
            "dsum": None if wide is None else r(rows, dim).to(wide)}


def own(p, rms=False, train=True):
    leaves = {k: p[k].detach().requires_grad_(train) for k in ("x", "weight", "bias", "residual") if p[k] is not None}
    both = p["residual"] is not None
    r = cc.add_norm_fn(leaves["x"], leaves["weight"], leaves.get("bias"), residual=leaves.get("residual"), rms=rms,
                       return_residual=both)
    got = {"out": r[0], "sum": r[1]} if both else {"out": r}
    if train:
        grads = torch.autograd.grad(r, list(leaves.values()), (p["dy"], p["dsum"]) if both else p["dy"])
        got.update({{"x": "dx", "weight": "dw", "bias": "db", "residual": "dresidual"}[k]: g for k, g in zip(leaves, grads)})
        for k, g in zip(leaves, grads):
            assert g.dtype == leaves[k].dtype and g.shape == leaves[k].shape
    return {k: v.detach() for k, v in got.items()}


def check(p, rms=False):
    e, s = norm64(p["x"], p["weight"], p["bias"], p["residual"], 1e-5, rms, p["dy"], p["dsum"])
    e["dresidual"], s["dresidual"] = e["dx"], s["dx"]
    rows, dim = p["x"].shape
    for k, v in own(p, rms).items():
        close(v, e[k], s[k], rows + dim, k)


DIMS = [1, 2, 7, 8, 63, 64, 65, 127, 255, 256, 511, 512, 513, 768, 1024, 1025, 1533, 2048, 2560, 2561, 4096, 4100, 5120,
        8192, 8199, 16384, 20001, 32768]


@pytest.mark.parametrize("dtype,residual", [(BF16, "none"), (BF16, "same"), (BF16, "fp32"), (FP16, "fp32"), (FP32, "same")],
                         ids=["bf16", "bf16+bf16", "bf16+fp32", "fp16+fp32", "fp32+fp32"])
@pytest.mark.parametrize("dim", DIMS)
def test_widths(dim, dtype, residual):
    check(make(5, dim, dtype, residual, seed=dim), rms=dim % 2 == 1)


@pytest.mark.parametrize("rows", [0, 1, 3, 64, 65, 1000, 5003])
@pytest.mark.parametrize("dtype,residual", [(BF16, "fp32"), (FP32, "none"), (FP16, "same")], ids=["bf16", "fp32", "fp16"])
def test_rows(rows, dtype, residual):
    check(make(rows, 200, dtype, residual, bias=rows % 2 == 0), rms=rows % 2 == 1)


def test_shapes_strides_and_views():
    p = make(6, 300, BF16, "fp32")
    want = own(p, train=False)
    big = torch.zeros(6, 2, 311, dtype=BF16, device=DEV)
    x = big[:, 1, 5:305]  # rows that start off any boundary
    x.copy_(p["x"])
    got = own({**p, "x": x, "weight": torch.stack([p["weight"]] * 2, 1)[:, 0]}, train=False)
    assert torch.equal(got["out"], want["out"]) and torch.equal(got["sum"], want["sum"])
    r = cc.add_norm_fn(p["x"].view(2, 3, 300), p["weight"], p["bias"], residual=p["residual"].view(2, 3, 300),
                       return_residual=True)
    assert r[0].shape == (2, 3, 300) and torch.equal(r[0].view(6, 300), want["out"])
    cols = p["x"].t().contiguous().t()  # columns contiguous
    assert torch.equal(own({**p, "x": cols}, train=False)["out"], want["out"])
    row = p["x"][:1].expand(6, -1)
    check({**p, "x": row})
    one = cc.add_norm_fn(p["x"][0], p["weight"], p["bias"])
    assert one.shape == (300,) and torch.equal(one, cc.add_norm_fn(p["x"], p["weight"], p["bias"])[0])
    y, x2 = cc.add_norm_fn(p["x"], p["weight"], return_residual=True)  # without a residual the stream is x
    assert x2 is p["x"]


def test_gradient_layouts_and_missing_gradients():
    p = make(40, 300, BF16, "fp32")
    want = own(p)
    assert all(torch.equal(v, own({**p, "dy": p["dy"].t().contiguous().t()})[k]) for k, v in want.items())
    leaves = [p[k].detach().requires_grad_() for k in ("x", "weight", "bias", "residual")]
    y, s = cc.add_norm_fn(leaves[0], leaves[1], leaves[2], residual=leaves[3], return_residual=True)
    gy = torch.autograd.grad(y, leaves, p["dy"], retain_graph=True)   # y's gradient alone
    gs = torch.autograd.grad(s, leaves, p["dsum"], allow_unused=True)  # the stream's alone
    assert torch.equal(gs[3], p["dsum"]) and torch.equal(gs[0], p["dsum"].bfloat16())
    assert gs[1] is None or (gs[1] == 0).all()
    zero = own({**p, "dsum": torch.zeros_like(p["dsum"])})
    assert all(torch.equal(a, zero[k]) for a, k in zip(gy, ("dx", "dw", "db", "dresidual")))
    y = cc.add_norm_fn(leaves[0], leaves[1], leaves[2], residual=leaves[3])  # the sum not returned
    g = torch.autograd.grad(y, leaves, p["dy"])
    assert all(torch.equal(a, zero[k]) for a, k in zip(g, ("dx", "dw", "db", "dresidual")))
    y, s = cc.add_norm_fn(p["x"].detach().requires_grad_(), p["weight"], residual=p["residual"], return_residual=True)
    assert y.requires_grad and s.requires_grad


@pytest.mark.parametrize("hole", [float("nan"), float("inf")])
@pytest.mark.parametrize("dim", [64, 300, 2560])
def test_rows_keep_to_themselves(dim, hole):
    p = make(9, dim, BF16, "fp32")
    want = own(p)
    p["x"][4, dim // 2] = hole
    got = own(p)
    rest = [0, 1, 2, 3, 5, 6, 7, 8]
    for k in ("out", "sum", "dx", "dresidual"):
        assert torch.equal(got[k][rest], want[k][rest]), k
    assert not torch.isfinite(got["out"][4]).all()


def test_large_offsets_and_small_spread():
    """A mean far above the spread: the variance is taken around the mean."""
    p = make(7, 1000, FP32, "none")
    p["x"] = 1000.0 + 0.01 * p["x"]
    check(p)
    p["x"] = torch.zeros(7, 1000, device=DEV)  # rstd = 1 / sqrt(eps)
    check(p)


def test_same_bits_every_time():
    p = make(3001, 777, BF16, "fp32")
    first = own(p)
    for _ in range(3):
        for k, v in own(p).items():
            assert torch.equal(v, first[k]), k


def test_past_32_bits():
    rows, dim = 65600, 32768  # 2.15e9 values
    x = torch.zeros(rows, dim, dtype=BF16, device=DEV)
    p = make(2, dim, BF16, "none")
    x[-2:] = p["x"]
    out = cc.add_norm_fn(x, p["weight"], p["bias"])
    assert torch.equal(out[-2:], cc.add_norm_fn(p["x"], p["weight"], p["bias"]))


def test_more_rows_than_one_turn_of_the_grid():
    """Eight lanes a row: 2**29 rows are more threads than a launch counts, and blocks take several turns."""
    rows = (1 << 29) + 3
    x = torch.randn(4099, 1, device=DEV).bfloat16().repeat(rows // 4099 + 1, 1)[:rows].requires_grad_()
    w, b = torch.tensor([1.5], device=DEV), torch.tensor([0.25], device=DEV)
    y = cc.add_norm_fn(x, w, b, rms=True)
    few = x.detach()[:4099].requires_grad_()
    want = cc.add_norm_fn(few, w, b, rms=True)
    dx, = torch.autograd.grad(y, x, x.detach())
    dwant, = torch.autograd.grad(want, few, few.detach())
    for got, exact in ((y, want), (dx, dwant)):
        for part in got.split(1 << 26):
            at = part.storage_offset() % 4099
            assert torch.equal(part, exact.roll(-at, 0).repeat(part.shape[0] // 4099 + 1, 1)[:part.shape[0]])


def test_graph_compile_and_side_stream():
    p = make(33, 2560, BF16, "fp32")
    want = own(p)
    names = ("x", "weight", "bias", "residual")
    leaves = [p[k].detach().clone().requires_grad_() for k in names]

    def step():
        r = cc.add_norm_fn(leaves[0], leaves[1], leaves[2], residual=leaves[3], return_residual=True)
        return (*r, *torch.autograd.grad(r, leaves, (p["dy"], p["dsum"])))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    order = ("out", "sum", "dx", "dw", "db", "dresidual")
    assert all(torch.equal(a, want[k]) for a, k in zip(got, order))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        outs = step()
    for seed in (0, 1, 2):
        new = make(33, 2560, BF16, "fp32", seed=seed)
        for k, t in zip(names, leaves):
            t.data.copy_(new[k])
        p["dy"].copy_(new["dy"])
        p["dsum"].copy_(new["dsum"])
        graph.replay()
        torch.cuda.synchronize()
        want = own(new)
        assert all(torch.equal(a, want[k]) for a, k in zip(outs, order)), seed
    leaves = [t.detach().clone().requires_grad_() for t in leaves]
    f = lambda x, w, b, r: cc.add_norm_fn(x, w, b, residual=r, return_residual=True)[0] * 2.0  # noqa: E731
    got = torch.compile(f, backend="aot_eager", fullgraph=True)(*leaves)
    eager = f(*leaves)
    assert torch.equal(got, eager)
    for a, b in zip(torch.autograd.grad(got, leaves, p["dy"]), torch.autograd.grad(eager, leaves, p["dy"])):
        assert torch.equal(a, b)


def test_ops_pass_opcheck():
    from test_scan_gpu import make as scan_make

    p = make(9, 100, BF16, "fp32")
    ops = torch.ops.causal_conv1d_amd
    y, s, st = torch.empty_like(p["x"]), torch.empty_like(p["residual"]), torch.empty(9, 2, device=DEV)
    torch.library.opcheck(ops._norm_fwd_inplace.default, (p["x"], p["weight"], p["bias"], p["residual"], 1e-5, False, y, s, st))
    dx, dr, dw, db = (torch.empty_like(p[k]) for k in ("x", "residual", "weight", "bias"))
    torch.library.opcheck(ops._norm_bwd_inplace.default,
                          (p["x"], p["weight"], p["residual"], st, False, p["dy"], p["dsum"], dx, dr, dw, db))
    q = scan_make(1, 8, 70, 16, 1, BF16)
    out, fin, tiles = torch.empty_like(q["u"]), torch.empty_like(q["init"]), torch.empty(8 * 16, device=DEV)
    args = (q["u"], q["delta"], q["A"], q["B"], q["C"], q["D"], q["z"], q["bias"], None, None)
    torch.library.opcheck(ops._scan_fwd_inplace.default, (*args, q["init"], True, out, fin, tiles))
    new = [torch.empty_like(q[k]) for k in ("u", "delta", "A", "B", "C", "D", "z", "bias", "init")]
    torch.library.opcheck(ops._scan_bwd_inplace.default, (*args, tiles, q["dout"], q["dfinal"], True, *new))
