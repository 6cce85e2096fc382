"""The example model: it trains, its gradients are those of the plain forms, and decoding continues a packed prefill as
prefills of the longer prompts do.

Tolerance of the comparisons (fp32 model): both sides evaluate the same formulas in fp32; an operator's result is off by
at most (64 + 4 sqrt(L)) 2**-24 of its terms' magnitude, 7e-6 here, about six follow each other in each of two layers
(twice as many where gradients go back through them), and a norm scales errors and values alike, with up to ten times
cancellation in between: 1e-3 of the largest value.
"""

from __future__ import annotations

import sys
from pathlib import Path

import pytest
import torch

import causal_conv1d_amd as cc

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "causal-conv1d-mojo_amd" / "examples"))

pytestmark = pytest.mark.gpu


def model_of(dtype, seed=0):
    from linear_attn_lm import LinearAttnLM

    torch.manual_seed(seed)
    return LinearAttnLM(vocab=64, dim=64, dtype=dtype)


@pytest.mark.parametrize("dtype", (torch.bfloat16, torch.float32))
def test_it_trains(dtype):
    from linear_attn_lm import Pack, train

    model = model_of(dtype)
    before = {n: p.detach().clone() for n, p in model.named_parameters()}
    lengths = [70, 1, 130]
    losses = train(model, torch.randint(64, (1, sum(lengths)), device="cuda"), Pack.of(lengths), 3)
    assert all(0 < x < 100 for x in losses)
    for n, p in model.named_parameters():
        assert torch.isfinite(p.grad).all() and p.grad.any(), n
        assert not torch.equal(p, before[n]), n


def test_gradients_are_the_plain_forms(monkeypatch):
    from linear_attn_lm import Pack, loss_of

    model = model_of(torch.float32)
    lengths = [70, 1, 130]
    tokens, pack = torch.randint(64, (1, sum(lengths)), device="cuda"), Pack.of(lengths)

    def grads():
        model.zero_grad()
        loss_of(model, tokens, pack).backward()
        return {n: p.grad.clone() for n, p in model.named_parameters()}

    got = grads()
    monkeypatch.setattr(cc, "linear_attn_fn", cc.linear_attn_ref)
    monkeypatch.setattr(cc, "head_norm_rotary_fn", cc.head_norm_rotary_ref)
    want = grads()
    for n, g in got.items():
        assert (g - want[n]).abs().max() <= 1e-3 * want[n].abs().max(), n


def test_decoding_continues_a_packed_prefill():
    from linear_attn_lm import Pack

    model = model_of(torch.float32, 1)
    tokens = torch.randint(64, (3, 140))
    lengths = (133, 1, 7)
    rows = torch.tensor([4, 0, 2], dtype=torch.int32, device="cuda")
    cache = model.new_cache(6)
    logits = model.prefill([t[:n] for t, n in zip(tokens, lengths)], cache, rows)
    untouched = [s[[1, 3, 5]].clone() for s in cache.attn]
    # a fourth slot of the decoding batch is free
    padded = torch.cat((rows, torch.tensor([-1], dtype=torch.int32, device="cuda")))
    for step in range(5):
        for i, n in enumerate(lengths):
            whole = model(tokens[i:i + 1, :n + step].cuda(), Pack.of([n + step]))[0, -1]
            assert (logits[i] - whole).abs().max() <= 1e-3 * whole.abs().max(), (step, i)
        new = torch.stack([t[n + step] for t, n in zip(tokens, lengths)] + [tokens[0, 0]])
        positions = torch.tensor([n + step for n in lengths] + [0], device="cuda")
        logits = model.decode(new.cuda(), positions, cache, padded)
    assert all(torch.equal(a, s[[1, 3, 5]]) for a, s in zip(untouched, cache.attn))
