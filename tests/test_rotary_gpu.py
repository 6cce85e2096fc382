"""head_norm_rotary_fn on the GPU against its definition in float64."""

from __future__ import annotations

import pytest
import torch

import causal_conv1d_amd as cc
from _attn import close, rotary64

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
TYPES = pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])


def make(lead, H, K, dim, rotated, dtype, norm="qk", reach=0, train=False, seed=0):
    gen = torch.Generator().manual_seed(seed + dim)
    r = lambda *s: torch.randn(*s, generator=gen)  # noqa: E731
    p = {"q": r(*lead, H, dim).to(dtype).to(DEV), "k": r(*lead, K, dim).to(dtype).to(DEV),
         "wq": (1 + 0.2 * r(dim)).to(DEV) if "q" in norm else None, "wk": (1 + 0.2 * r(dim)).to(DEV) if "k" in norm else None,
         "freq": cc.rotary_frequencies(rotated, device=DEV)[0] if rotated else None, "pos": None}
    if reach or len(lead) == 1:
        p["pos"] = torch.randint(0, reach + 1, lead, generator=gen).to(DEV)
    p["dq"] = r(*lead, H, dim).to(dtype).to(DEV) if train else None
    p["dk"] = r(*lead, K, dim).to(dtype).to(DEV) if train else None
    return p


def own(p, **how):
    leaves = {n: p[n] if p[n] is None or p["dq"] is None else p[n].detach().requires_grad_() for n in ("q", "k", "wq", "wk")}
    q, k = cc.head_norm_rotary_fn(leaves["q"], leaves["k"], leaves["wq"], leaves["wk"], p["freq"], p["pos"], **how)
    got = {"q": q, "k": k}
    if p["dq"] is not None:
        wanted = {n: t for n, t in leaves.items() if t is not None}
        got.update({"d" + n: g for n, g in zip(wanted, torch.autograd.grad((q, k), list(wanted.values()), (p["dq"], p["dk"])))})
    return got


def check(p, **how):
    got = own(p, **how)
    e, m = rotary64(p["q"], p["k"], p["wq"], p["wk"], p["freq"], p["pos"], dq=p["dq"], dk=p["dk"], **how)
    for n, t in got.items():
        assert t.is_contiguous()
        # a weight's gradient is a sum over the heads of every token
        close(t, e[n], m[n], p[n[-1]].numel() // p["q"].shape[-1] if n.startswith("dw") else 1, n, drift(p, n, m[n]))
    return got


def drift(p, n, mag):
    """What 64 bits leave of an angle: the definition's product position * frequency (at most the position: frequencies
    are 1 and less) is off by 2**-53 of it, the kernel's product, its factor 2 / pi and their product by 3 * 2**-53, a
    cosine or sine by as much as its angle."""
    if p["pos"] is None or n.startswith("dw"):
        return 0.0
    return 2.0**-51 * p["pos"].double().abs().cpu()[..., None, None] * mag


SIZES = [((1, 1), 1, 1, 1, 0), ((2, 5), 4, 2, 64, 64), ((3, 7), 5, 1, 128, 128), ((1, 9), 3, 3, 256, 256), ((2, 3), 2, 7, 80, 36),
         ((1, 4), 1, 2, 2, 2), ((2, 2), 3, 1, 67, 34), ((1, 3), 9, 9, 256, 252), ((5, 1), 2, 2, 96, 30), ((1, 2), 2, 1, 253, 4),
         ((33, 5), 2, 2, 8, 8), ((1, 6), 40, 8, 128, 64)]


@TYPES
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_sizes(size, interleaved, dtype):
    check(make(*size, dtype), interleaved=interleaved)
    check(make(*size, dtype, train=True), interleaved=interleaved)


@TYPES
@pytest.mark.parametrize("norm", ["", "q", "k"])
@pytest.mark.parametrize("train", [False, True])
def test_without_a_norm(norm, train, dtype):
    check(make((2, 9), 4, 2, 64, 48, dtype, norm, train=train), eps=1e-3)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("integer", [torch.int32, torch.int64])
def test_far_positions(integer, interleaved):
    """Angles of a million turns and more: as exact as near ones."""
    p = make((4, 50), 2, 2, 64, 64, FP32, reach=2**31 - 1, train=True)
    p["pos"][0, 0], p["pos"][0, 1] = 0, -5
    p["pos"] = p["pos"].to(integer)
    check(p, interleaved=interleaved, amplitude=1.25)


def test_positions_past_32_bits():
    p = make((1, 5), 2, 2, 64, 64, FP32)
    p["pos"] = torch.tensor([[2**31, 2**33 + 1, 2**40 + 7, -2**35, 3]], device=DEV)
    check(p)


@TYPES
def test_single_tokens(dtype):
    check(make((7,), 6, 2, 128, 128, dtype, reach=100000))
    check(make((7,), 6, 2, 128, 128, dtype, reach=100000, train=True))


@pytest.mark.parametrize("tokens", [(1, 8200), (3, 2900)], ids=str)
def test_many_tokens(tokens):
    """More tokens than wavefronts at once: the walk over tokens, and the weights' sums over them."""
    check(make(tokens, 3, 1, 32, 32, BF16, train=True))


def test_strides():
    """q, k and their gradients as slices of one projection, heads and values any distance apart."""
    p = make((2, 6), 4, 2, 64, 32, BF16, train=True)
    one = torch.cat([p["q"].flatten(2), p["k"].flatten(2)], 2)
    q, k = one[..., :256].unflatten(2, (4, 64)), one[..., 256:].unflatten(2, (2, 64))
    check({**p, "q": q, "k": k})
    apart = {n: torch.stack([p[n], p[n]], -1)[..., 1] for n in ("q", "k", "dq", "dk")}
    check({**p, **apart})
    check({**p, "dq": p["dq"][:, :, :1].expand(-1, -1, 4, -1), "pos": torch.arange(6, device=DEV).expand(2, 6)})


def test_rows_that_hold_nothing():
    """A head of zeros: the norm's epsilon keeps it, and its gradient, finite."""
    p = make((1, 3), 2, 2, 64, 64, BF16, train=True)
    p["q"][0, 1] = 0
    check(p)


def test_one_value_that_is_not_finite_stays_in_its_head():
    p = make((1, 4), 3, 2, 64, 64, FP32, train=True)
    want = own(p)
    p["q"][0, 2, 1, 5] = float("nan")
    got = own(p)
    hit = torch.zeros(1, 4, 3, dtype=torch.bool, device=DEV)
    hit[0, 2, 1] = True
    for n in ("q", "dq"):
        assert got[n][hit].isnan().all() and torch.equal(got[n][~hit], want[n][~hit])
    assert torch.equal(got["k"], want["k"]) and torch.equal(got["dwk"], want["dwk"])


def test_empty():
    p = make((2, 0), 3, 2, 64, 64, BF16, train=True)
    got = own(p)
    assert got["q"].shape == (2, 0, 3, 64) and (got["dwq"] == 0).all() and (got["dwk"] == 0).all()


def test_the_same_bits_again():
    p = make((2, 700), 4, 2, 128, 128, BF16, train=True)
    a, b = own(p), own(p)
    assert all(torch.equal(a[n], b[n]) for n in a)


def test_graph_and_side_stream():
    p = make((2, 40), 4, 2, 64, 64, BF16)
    want = own(p)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = own(p)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(got[n], want[n]) for n in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = own(p)
    for seed in range(3):
        p["q"].copy_(make((2, 40), 4, 2, 64, 64, BF16, seed=seed)["q"])
        want = own(p)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(got[n], want[n]) for n in got)
