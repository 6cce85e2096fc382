"""A small state space language model on the package's operators: trained for a few
steps, then served (prompts of several lengths packed into one prefill, and decode
steps on a pool of states).

    python causal-conv1d-mojo_amd/examples/state_space_lm.py

Activations are (batch, seqlen, channels) out of every projection; the convolution and
the scan take them as they lie (channel-last views, B and C as slices), so nothing is
copied between the operators.
"""

from __future__ import annotations

import math
import sys
from dataclasses import dataclass
from pathlib import Path

import torch
import torch.nn.functional as F
from torch import nn

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import causal_conv1d_amd as cc  # noqa: E402

WIDTH = 4  # of the convolution


@dataclass
class Cache:
    """The states of every layer, a row per served sequence."""

    conv: list[torch.Tensor]  # (rows, inner, WIDTH - 1)
    ssm: list[torch.Tensor]  # (rows, inner, dstate) fp32


class Layer(nn.Module):
    def __init__(self, dim: int, dstate: int, dtype: torch.dtype, device: str) -> None:
        super().__init__()
        inner, rank = 2 * dim, max(1, dim // 16)
        self.split = (rank, dstate, dstate)
        like = {"dtype": dtype, "device": device}
        self.norm = nn.Parameter(torch.ones(dim, device=device))
        self.into = nn.Linear(dim, 2 * inner, bias=False, **like)
        self.conv_weight = nn.Parameter(torch.randn(inner, WIDTH, **like) / WIDTH**0.5)
        self.conv_bias = nn.Parameter(torch.zeros(inner, **like))
        self.select = nn.Linear(inner, rank + 2 * dstate, bias=False, **like)
        self.step = nn.Linear(rank, inner, bias=False, **like)
        self.out = nn.Linear(inner, dim, bias=False, **like)
        # decays -1 .. -dstate, steps between 1e-3 and 1e-1 before the inputs move them
        self.log_decay = nn.Parameter(torch.arange(1, dstate + 1, device=device).float().log().repeat(inner, 1))
        dt = torch.exp(torch.rand(inner, device=device) * math.log(100.0) + math.log(1e-3))
        self.step_bias = nn.Parameter(dt + torch.log(-torch.expm1(-dt)))
        self.skip = nn.Parameter(torch.ones(inner, device=device))

    def selected(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        rank, B, C = self.select(x).split(self.split, dim=-1)
        return self.step(rank), B, C

    def forward(self, h, stream, ids=None, cu=None, cache=None):
        """h (batch, seqlen, dim), the residual stream so far; ``cu`` and ``cache``: (conv states, ssm states) to fill."""
        h, stream = cc.add_norm_fn(h, self.norm, None, stream, rms=True, return_residual=True)
        x, z = self.into(h).chunk(2, dim=-1)
        if cache is not None:
            cache[0].copy_(cc.causal_conv1d_varlen_states(x[0], cu, WIDTH - 1))
        x = cc.causal_conv1d_fn(x.transpose(1, 2), self.conv_weight, self.conv_bias, seq_idx=ids, activation="silu")
        step, B, C = self.selected(x.transpose(1, 2))
        y = cc.ssm_scan_fn(x, step.transpose(1, 2), -self.log_decay.exp(), B.transpose(1, 2), C.transpose(1, 2),
                           D=self.skip, z=z.transpose(1, 2), delta_bias=self.step_bias, delta_softplus=True,
                           seq_idx=None if cache is not None else ids, cu_seqlens=cu,
                           return_final_states=cache is not None)
        if cache is not None:
            y, states = y
            cache[1].copy_(states)
        return self.out(y.transpose(1, 2)), stream

    def decode(self, h, stream, conv, ssm, rows):
        """One token of each sequence: h (batch, dim); rows (batch,) int32, those of the states (< 0: a free slot)."""
        h, stream = cc.add_norm_fn(h, self.norm, None, stream, rms=True, return_residual=True)
        x, z = self.into(h).chunk(2, dim=-1)
        x = cc.causal_conv1d_update(x, conv, self.conv_weight, self.conv_bias, activation="silu", conv_state_indices=rows)
        step, B, C = self.selected(x)
        y = cc.ssm_scan_update(x, ssm, step, -self.log_decay.exp(), B, C, D=self.skip, z=z, delta_bias=self.step_bias,
                               delta_softplus=True, ssm_state_indices=rows)
        return self.out(y), stream


class StateSpaceLM(nn.Module):
    def __init__(self, vocab=256, dim=128, layers=2, dstate=16, dtype=torch.bfloat16, device="cuda") -> None:
        super().__init__()
        self.embed = nn.Embedding(vocab, dim, dtype=dtype, device=device)
        self.layers = nn.ModuleList(Layer(dim, dstate, dtype, device) for _ in range(layers))
        self.norm = nn.Parameter(torch.ones(dim, device=device))
        self.head = nn.Linear(dim, vocab, bias=False, dtype=dtype, device=device)

    def forward(self, tokens: torch.Tensor, ids: torch.Tensor | None = None) -> torch.Tensor:
        """Logits of (batch, seqlen) tokens; ``ids`` marks documents packed into a row."""
        h = self.embed(tokens)
        stream = torch.zeros_like(h, dtype=torch.float32)  # the residual stream stays in 32 bits
        for layer in self.layers:
            h, stream = layer(h, stream, ids)
        return self.head(cc.add_norm_fn(h, self.norm, None, stream, rms=True))

    def new_cache(self, rows: int) -> Cache:
        first = self.layers[0]
        inner, dstate = first.log_decay.shape
        like = {"device": first.skip.device}
        return Cache([torch.zeros(rows, inner, WIDTH - 1, dtype=first.conv_bias.dtype, **like) for _ in self.layers],
                     [torch.zeros(rows, inner, dstate, **like) for _ in self.layers])

    @torch.no_grad()
    def prefill(self, prompts: list[torch.Tensor], cache: Cache, rows: torch.Tensor) -> torch.Tensor:
        """Prompts of any lengths as one packed row; their states go to ``rows``. Logits after each prompt."""
        lengths = torch.tensor([len(p) for p in prompts])
        cu = F.pad(lengths.cumsum(0), (1, 0)).to(torch.int32).to(rows.device)
        ids = torch.repeat_interleave(torch.arange(len(prompts), dtype=torch.int32), lengths).to(rows.device)[None]
        h = self.embed(torch.cat(prompts).to(rows.device)[None])
        stream = torch.zeros_like(h, dtype=torch.float32)
        for layer, conv, ssm in zip(self.layers, cache.conv, cache.ssm):
            new = conv.new_empty(len(prompts), *conv.shape[1:]), ssm.new_empty(len(prompts), *ssm.shape[1:])
            h, stream = layer(h, stream, ids, cu, new)
            conv[rows.long()], ssm[rows.long()] = new
        last = (cu[1:] - 1).long()
        return self.head(cc.add_norm_fn(h[0, last], self.norm, None, stream[0, last], rms=True))

    @torch.no_grad()
    def decode(self, tokens: torch.Tensor, cache: Cache, rows: torch.Tensor) -> torch.Tensor:
        """Logits after one more token (batch,) of the sequences whose states are ``rows``."""
        h = self.embed(tokens)
        stream = torch.zeros_like(h, dtype=torch.float32)
        for layer, conv, ssm in zip(self.layers, cache.conv, cache.ssm):
            h, stream = layer.decode(h, stream, conv, ssm, rows)
        return self.head(cc.add_norm_fn(h, self.norm, None, stream, rms=True))


def train(model: StateSpaceLM, tokens: torch.Tensor, ids: torch.Tensor | None, steps: int, lr: float = 3e-3) -> list[float]:
    """Next-token training on one batch; the loss of each step."""
    opt = torch.optim.AdamW(model.parameters(), lr=lr)
    losses = []
    for _ in range(steps):
        logits = model(tokens[:, :-1], None if ids is None else ids[:, :-1])
        loss = F.cross_entropy(logits.float().flatten(0, 1), tokens[:, 1:].flatten())
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    return losses


def main() -> None:
    torch.manual_seed(0)
    model = StateSpaceLM()
    tokens = torch.randint(256, (4, 257), device="cuda")
    ids = (torch.arange(257, device="cuda") >= 100).int().expand(4, -1).contiguous()  # two documents a row
    losses = train(model, tokens, ids, 40)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f}")

    rows = torch.tensor([5, 0, 3], dtype=torch.int32, device="cuda")
    cache = model.new_cache(8)
    token = model.prefill([tokens[0, :100].cpu(), tokens[1, 100:140].cpu(), tokens[2, :3].cpu()], cache, rows).argmax(-1)
    out = [token]
    for _ in range(15):
        token = model.decode(token, cache, rows).argmax(-1)
        out.append(token)
    for text in torch.stack(out, 1).tolist():
        print(*text)


if __name__ == "__main__":
    main()
