"""linear_attn_update on the GPU against its definition in float64, and against linear_attn_fn over the same tokens."""

from __future__ import annotations

import math

import pytest
import torch

import causal_conv1d_amd as cc
from _attn import attn64, close

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def make(batch, T, H, K, dk, dv, dtype, rows=None, seed=0):
    gen = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen).to(DEV)  # noqa: E731
    lead = (batch,) if T is None else (batch, T)
    return {"q": r(*lead, K, dk).to(dtype), "state": r(rows or batch, H, dk, dv), "k": r(*lead, K, dk).to(dtype),
            "v": r(*lead, H, dv).to(dtype), "g": (-r(*lead, H).abs()).to(dtype)}


def call(p, idx=None, scale=None):
    return cc.linear_attn_update(p["q"], p["state"], p["k"], p["v"], p["g"], scale, idx)


def check(p, idx=None, scale=None):
    before = p["state"].clone()
    rows = torch.arange(p["q"].shape[0], device=DEV) if idx is None else idx.long()
    live = (rows >= 0) & (rows < before.shape[0])
    timed = p["q"].dim() == 4
    q = [p[n][live] if timed else p[n][live].unsqueeze(1) for n in ("q", "k", "v", "g")]
    s = p["q"].shape[-1] ** -0.5 if scale is None else scale
    e, m = (attn64(*q, s, before[rows[live]], mag=x) for x in (False, True))
    out = call(p, idx, scale)
    assert out.shape == p["v"].shape and out.is_contiguous()
    T = q[0].shape[1]
    shape = p["v"][live].shape
    close(out[live], e["out"].reshape(shape), m["out"].reshape(shape), T, "out")
    close(p["state"][rows[live]], e["final"], m["final"], T, "state")
    assert (out[~live] == 0).all()
    rest = torch.ones(before.shape[0], dtype=torch.bool, device=DEV)
    rest[rows[live]] = False
    assert torch.equal(p["state"][rest], before[rest])


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T", [None, 1, 4])
@pytest.mark.parametrize("size", [(1, 1, 1, 1, 1), (2, 4, 4, 64, 64), (3, 6, 2, 128, 128), (1, 2, 1, 17, 5), (5, 3, 3, 80, 72),
                                  (2, 8, 1, 128, 64), (1, 2, 2, 127, 126), (4, 1, 1, 3, 128), (9, 2, 2, 128, 4), (2, 5, 5, 64, 33)],
                         ids=str)
def test_sizes(size, T, dtype):
    batch, H, K, dk, dv = size
    check(make(batch, T, H, K, dk, dv, dtype, seed=dk))


@pytest.mark.parametrize("T", [None, 3])
@pytest.mark.parametrize("dv", [64, 30])
def test_pool_with_padding(dv, T):
    p = make(7, T, 4, 2, 64, dv, BF16, rows=12)
    idx = torch.tensor([11, -1, 0, 3, -7, 12, 5], dtype=torch.int32, device=DEV)  # 12: outside the pool
    for n in ("q", "k", "v", "g"):
        p[n][[1, 4, 5]] = float("nan")  # unused slots hold anything
    check(p, idx)
    check(make(2, T, 4, 2, 64, dv, BF16, rows=3), torch.tensor([-1, -1], dtype=torch.int32, device=DEV))


def test_empty_pool_and_batch():
    p = make(2, None, 2, 2, 16, 16, BF16)
    p["state"] = torch.zeros(0, 2, 16, 16, device=DEV)
    assert (call(p, torch.tensor([0, -1], dtype=torch.int32, device=DEV)) == 0).all()
    assert call(make(0, None, 2, 2, 16, 16, BF16)).shape == (0, 2, 16)
    p = make(2, 0, 2, 2, 16, 16, BF16)
    before = p["state"].clone()
    assert call(p).shape == (2, 0, 2, 16) and torch.equal(p["state"], before)


@pytest.mark.parametrize("dv", [48, 50])
def test_strides(dv):
    """States and tokens read and written through any strides."""
    p = make(3, 2, 4, 2, 24, dv, FP32, rows=4)
    big = torch.zeros(4, 5, dv, 24, 2, device=DEV)
    state = big[:, 1:, :, :, 1].transpose(2, 3)
    state.copy_(p["state"])
    both = torch.stack([p["q"], p["k"]], -1)  # values two apart
    idx = torch.tensor([3, 0, 1], dtype=torch.int32, device=DEV)
    check({**p, "state": state, "q": both[..., 0], "k": both[..., 1], "v": p["v"].transpose(1, 2).contiguous().transpose(1, 2),
           "g": p["g"][:, :, :1].expand(-1, -1, 4)}, idx)
    assert (big[:, :1] == 0).all() and (big[..., 0] == 0).all()  # nothing beside the state
    p = make(3, None, 4, 2, 24, dv, BF16)
    off = torch.zeros(3 * 4 * 24 * dv + 1, device=DEV)[1:].view(3, 4, 24, dv)  # off the 16-byte grid
    check({**p, "state": off.copy_(p["state"])})


@pytest.mark.parametrize("g", [-math.inf, -1e4, 0.0, 0.3])
def test_decays(g):
    p = make(2, 3, 2, 1, 16, 16, FP32)
    p["g"][:, 1] = g
    check(p, scale=0.5)


def test_tokens_one_by_one_are_the_whole():
    """Prompt by linear_attn_fn, then tokens by the update: what linear_attn_fn over all of them gives."""
    p = make(2, 150, 4, 2, 64, 48, FP32)
    q, k, v, g = (p[n] for n in ("q", "k", "v", "g"))
    whole, final = cc.linear_attn_fn(q, k, v, g, return_final_states=True)
    out, state = cc.linear_attn_fn(q[:, :140], k[:, :140], v[:, :140], g[:, :140], return_final_states=True)
    torch.testing.assert_close(out, whole[:, :140], rtol=1e-5, atol=1e-5)
    for t in range(140, 146):
        o = cc.linear_attn_update(q[:, t], state, k[:, t], v[:, t], g[:, t])
        torch.testing.assert_close(o, whole[:, t], rtol=1e-4, atol=1e-4)
    o = cc.linear_attn_update(q[:, 146:], state, k[:, 146:], v[:, 146:], g[:, 146:])
    torch.testing.assert_close(o, whole[:, 146:], rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(state, final, rtol=1e-4, atol=1e-4)


def test_large_pool_past_32_bits():
    """A pool of more than 2**31 states: the last row is found."""
    rows = 1030
    state = torch.zeros(rows, 128, 128, 128, device=DEV)  # 2.16e9 states, 8.6 GB
    p = make(2, None, 128, 128, 128, 128, BF16, rows=2)
    state[-1].copy_(p["state"][0])
    state[0].copy_(p["state"][1])
    small = p["state"].clone()
    p["state"] = state
    out = call(p, torch.tensor([rows - 1, 0], dtype=torch.int32, device=DEV))
    q = {**p, "state": small}
    assert torch.equal(out, call(q)) and torch.equal(state[-1], small[0]) and torch.equal(state[0], small[1])


def test_graph_and_side_stream():
    p = make(5, None, 4, 2, 64, 64, BF16, rows=8)
    idx = torch.tensor([7, 2, -1, 0, 5], dtype=torch.int32, device=DEV)
    want = {n: v.clone() for n, v in p.items()}
    outs = [call(want, idx).clone() for _ in range(3)]
    side = torch.cuda.Stream()
    scratch = {n: v.clone() for n, v in p.items()}
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(scratch, idx)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(scratch["state"][[7, 2]], scratch["state"][[7, 2]])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(p, idx)
    for o in outs:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, o)
    assert torch.equal(p["state"], want["state"])
