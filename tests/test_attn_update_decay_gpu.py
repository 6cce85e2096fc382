"""linear_attn_update's decay."""

from __future__ import annotations

import math

import pytest
import torch

import causal_conv1d_amd as cc

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32], ids=["bf16", "fp16", "fp32"])
def test_a_decay_is_exp_of_g(dtype):
    """A state of ones after a token without a key: the exponential's two roundings and that of its correction, 2**-22."""
    n = 4096
    g = -torch.logspace(-4, math.log10(87.0), n, device=DEV).to(dtype)
    state = torch.ones(n, 1, 1, 1, device=DEV)
    zero = torch.zeros(n, 1, 1, dtype=dtype, device=DEV)
    cc.linear_attn_update(zero, state, zero, zero, g.view(n, 1))
    want = torch.exp(g.double())
    off = (state.flatten().double() - want).abs() / want
    assert off.max().item() <= 2.0**-22, (g[off.argmax()].item(), off.max().item() * 2**24)


def test_decays_beyond():
    g = torch.tensor([-math.inf, -1e30, -1e5, -1000.0, 0.0, 1000.0, math.inf, math.nan], device=DEV)
    state = torch.ones(8, 1, 1, 1, device=DEV)
    zero = torch.zeros(8, 1, 1, device=DEV)
    cc.linear_attn_update(zero, state, zero, zero, g.view(8, 1))
    s = state.flatten().tolist()
    assert s[:6] == [0.0, 0.0, 0.0, 0.0, 1.0, math.inf] and s[6] == math.inf and math.isnan(s[7])
