"""linear_attn_update on a stream that is not the current one."""

from __future__ import annotations

import pytest
import torch

from test_attn_update_gpu import BF16, DEV, call, make

pytestmark = pytest.mark.gpu


def test_side_stream():
    """Output and state of a call on another stream, which the inputs are written on as well, are those of the current one."""
    p = make(5, None, 4, 2, 64, 64, BF16, rows=8)
    idx = torch.tensor([7, 2, -1, 0, 5], dtype=torch.int32, device=DEV)
    want = {n: v.clone() for n, v in p.items()}
    out = call(want, idx)
    side = torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device=DEV)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(4):
            busy = busy @ busy * 1e-4  # the inputs are there when this is done, and no sooner
        got = {n: torch.where(busy.isnan().any(), v, v) for n, v in p.items()}
        there = call(got, idx)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert torch.equal(there, out) and torch.equal(got["state"], want["state"]) and not torch.equal(got["state"], p["state"])
