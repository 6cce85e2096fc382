"""ssm_scan_update on the GPU against its definition in float64, and against the scan over the same tokens."""

from __future__ import annotations

import pytest
import torch

import causal_conv1d_amd as cc
from _ssm import close, scan64

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def make(batch, D, N, G, T, dtype, rows=None, seed=0, gate=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
    tail = () if T is None else (T,)
    return {"u": r(batch, D, *tail).to(dtype), "state": r(rows or batch, D, N), "delta": (0.5 * r(batch, D, *tail)).to(dtype),
            "A": -2.0 * r(D, N).abs(), "B": r(batch, G, N, *tail).to(dtype), "C": r(batch, G, N, *tail).to(dtype),
            "D": r(D), "z": r(batch, D, *tail).to(dtype) if gate else None, "bias": 0.5 * r(D)}


def call(p, idx=None, softplus=True):
    return cc.ssm_scan_update(p["u"], p["state"], p["delta"], p["A"], p["B"], p["C"], D=p["D"], z=p["z"],
                              delta_bias=p["bias"], delta_softplus=softplus, ssm_state_indices=idx)


def exact(p, rows, softplus=True):
    """(values, magnitudes) of the live entries, whose states are p's rows."""
    f = (lambda t: None if t is None else (t if t.dim() == p["u"].dim() + 2 or p["u"].dim() == 3 else t[..., None]))
    args = [f(p["u"]), f(p["delta"]), p["A"], f(p["B"]), f(p["C"]), p["D"], f(p["z"]), p["bias"]]
    return [scan64(*args, softplus, None, p["state"][rows], mag=m) for m in (False, True)]


def check(p, idx=None, softplus=True):
    before = p["state"].clone()
    rows = torch.arange(p["u"].shape[0], device=DEV) if idx is None else idx.long()
    live = (rows >= 0) & (rows < before.shape[0])
    q = {k: (v[live] if k in ("u", "delta", "B", "C", "z") and v is not None else v) for k, v in p.items()}
    e, s = exact(q, rows[live], softplus)
    out = call(p, idx, softplus)
    T = 1 if p["u"].dim() == 2 else p["u"].shape[2]
    shape = p["u"][live].shape
    close(out[live], e["out"].reshape(shape), s["out"].reshape(shape), T, "out")
    close(p["state"][rows[live]], e["final"], s["final"], T, "state")
    assert (out[~live] == 0).all()
    rest = torch.ones(before.shape[0], dtype=torch.bool, device=DEV)
    rest[rows[live]] = False
    assert torch.equal(p["state"][rest], before[rest])


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("T", [None, 1, 4])
@pytest.mark.parametrize("size", [(1, 1, 1, 1), (2, 64, 16, 1), (3, 30, 5, 3), (1, 257, 16, 1), (5, 48, 64, 8), (2, 10, 128, 1),
                                  (2, 7, 256, 1), (33, 72, 16, 2), (2, 9, 40, 1), (1, 6, 130, 1), (4, 33, 8, 1)], ids=str)
def test_sizes(size, T, dtype):
    batch, D, N, G = size
    check(make(batch, D, N, G, T, dtype, seed=D))


@pytest.mark.parametrize("softplus", [False, True])
@pytest.mark.parametrize("absent", ["z", "D", "bias", None])
def test_options(absent, softplus):
    p = make(3, 40, 16, 1, None, BF16)
    if absent:
        p[absent] = None
    check(p, softplus=softplus)


@pytest.mark.parametrize("T", [None, 3])
@pytest.mark.parametrize("N", [16, 6])
def test_pool_with_padding(N, T):
    p = make(7, 40, N, 1, T, BF16, rows=12)
    idx = torch.tensor([11, -1, 0, 3, -7, 12, 5], dtype=torch.int32, device=DEV)  # 12: outside the pool
    for k in ("u", "delta", "z", "B", "C"):
        p[k][[1, 4, 5]] = float("nan")  # unused slots hold anything
    check(p, idx)
    check(make(2, 40, N, 1, T, BF16, rows=3), torch.tensor([-1, -1], dtype=torch.int32, device=DEV))


def test_empty_pool_and_batch():
    p = make(2, 40, 16, 1, None, BF16)
    p["state"] = torch.zeros(0, 40, 16, device=DEV)
    assert (call(p, torch.tensor([0, -1], dtype=torch.int32, device=DEV)) == 0).all()
    p = make(0, 40, 16, 1, None, BF16)
    assert call(p).shape == (0, 40)


@pytest.mark.parametrize("N", [16, 12])
def test_strides(N):
    """States, parameters and tokens read and written through any strides."""
    p = make(3, 36, N, 2, 2, FP32, rows=4)
    big = torch.zeros(4, N + 1, 36, 2, device=DEV)
    state = big[:, 1:, :, 1].transpose(1, 2)
    state.copy_(p["state"])
    q = {**p, "state": state, "A": p["A"].t().contiguous().t(), "u": p["u"].transpose(1, 2).contiguous().transpose(1, 2),
         "B": p["B"].permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)[..., :2],
         "D": torch.stack([p["D"], p["D"]], 1)[:, 0]}
    idx = torch.tensor([3, 0, 1], dtype=torch.int32, device=DEV)
    check(q, idx)
    assert (big[:, :1] == 0).all() and (big[..., 0] == 0).all()  # nothing beside the state
    p = make(3, 36, N, 2, None, BF16)
    off = torch.zeros(3 * 36 * N + 1, device=DEV)[1:].view(3, 36, N)  # off the 16-byte grid
    check({**p, "state": off.copy_(p["state"])})


def test_one_state_row_shared_by_expand_reads():
    p = make(4, 36, 16, 1, None, BF16)
    check({**p, "A": p["A"][:, :1].expand(-1, 16), "B": p["B"][:1].expand(4, -1, -1)})


def test_tokens_one_by_one_are_the_scan():
    """Prompt by the scan, then tokens by the update: what the scan over all of them gives."""
    D, N, L, P = 48, 16, 40, 30
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g).to(DEV)  # noqa: E731
    u, delta, z, B, C = r(2, D, L), 0.5 * r(2, D, L), r(2, D, L), r(2, 1, N, L), r(2, 1, N, L)
    A, skip, bias = -2.0 * r(D, N).abs(), r(D), r(D)
    whole, final = cc.ssm_scan_fn(u, delta, A, B, C, skip, z, bias, True, return_final_states=True)
    out, state = cc.ssm_scan_fn(u[..., :P], delta[..., :P], A, B[..., :P], C[..., :P], skip, z[..., :P], bias, True,
                                return_final_states=True)
    torch.testing.assert_close(out, whole[..., :P], rtol=1e-5, atol=1e-5)
    for t in range(P, P + 4):
        o = cc.ssm_scan_update(u[..., t], state, delta[..., t], A, B[..., t], C[..., t], skip, z[..., t], bias, True)
        torch.testing.assert_close(o, whole[..., t], rtol=1e-4, atol=1e-4)
    o = cc.ssm_scan_update(u[..., P + 4:], state, delta[..., P + 4:], A, B[..., P + 4:], C[..., P + 4:], skip,
                           z[..., P + 4:], bias, True)
    torch.testing.assert_close(o, whole[..., P + 4:], rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(state, final, rtol=1e-4, atol=1e-4)


def test_large_pool_past_32_bits():
    """A pool of more than 2**31 states: the last row is found."""
    rows, D, N = 1040, 8192, 256  # 2.18e9 states, 8.7 GB
    state = torch.zeros(rows, D, N, device=DEV)
    p = make(2, D, N, 1, None, BF16, rows=2)
    state[-1].copy_(p["state"][0])
    state[0].copy_(p["state"][1])
    small = p["state"].clone()
    p["state"] = state
    out = call(p, torch.tensor([rows - 1, 0], dtype=torch.int32, device=DEV))
    q = {**p, "state": small}
    assert torch.equal(out, call(q)) and torch.equal(state[-1], small[0]) and torch.equal(state[0], small[1])


def test_graph_and_side_stream():
    p = make(5, 64, 16, 1, None, BF16, rows=8)
    idx = torch.tensor([7, 2, -1, 0, 5], dtype=torch.int32, device=DEV)
    want = {k: v.clone() for k, v in p.items()}
    outs = [call(want, idx).clone() for _ in range(3)]
    side = torch.cuda.Stream()
    scratch = {k: v.clone() for k, v in p.items()}
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(scratch, idx)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = call(p, idx)
    for i in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, outs[i])
        torch.zeros(1000, device=DEV).sum().item()
    assert torch.equal(p["state"], want["state"])


def test_wide_batch():
    """More batch entries than a grid's second axis holds."""
    p = make(70000, 4, 2, 1, None, FP32)
    check(p)
