"""The example model: training lowers its loss, and decoding continues a packed
prefill as prefills of the longer prompts do.

Tolerance of the comparison (fp32 model): both sides evaluate the same formulas in
fp32; an operator's result is off by at most (64 + 4 sqrt(L)) 2**-24 of its terms'
magnitude, 7e-6 here, about six follow each other in each of two layers, and a norm
scales errors and values alike, with up to ten times cancellation in between: 1e-3 of
the largest logit.
"""

from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "causal-conv1d-mojo_amd" / "examples"))

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
def test_training_lowers_the_loss(dtype):
    from state_space_lm import StateSpaceLM, train

    torch.manual_seed(0)
    model = StateSpaceLM(vocab=64, dim=64, dtype=dtype)
    tokens = torch.randint(64, (2, 130), device="cuda")
    ids = (torch.arange(130, device="cuda") >= 50).int().expand(2, -1).contiguous()
    losses = train(model, tokens, ids, 40)
    assert losses[-1] < 0.5 * losses[0], losses
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in model.parameters())


def test_decoding_continues_a_packed_prefill():
    from state_space_lm import StateSpaceLM

    torch.manual_seed(1)
    model = StateSpaceLM(vocab=64, dim=64, dtype=torch.float32)
    tokens = torch.randint(64, (3, 40))
    lengths = (33, 1, 7)
    rows = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
    cache = model.new_cache(6)
    logits = model.prefill([t[:n] for t, n in zip(tokens, lengths)], cache, rows)
    untouched = [s[[1, 3, 5]].clone() for s in cache.ssm]
    # a fourth slot of the decoding batch is free
    padded = torch.cat((rows, torch.tensor([-1], dtype=torch.int32, device="cuda")))
    for step in range(5):
        for i, n in enumerate(lengths):
            whole = model(tokens[i:i + 1, :n + step].cuda())[0, -1]
            assert (logits[i] - whole).abs().max() <= 1e-3 * whole.abs().max(), (step, i)
        new = torch.stack([t[n + step] for t, n in zip(tokens, lengths)] + [tokens[0, 0]])
        logits = model.decode(new.cuda(), cache, padded)
    assert all(torch.equal(a, s[[1, 3, 5]]) for a, s in zip(untouched, cache.ssm))
