"""A small language model of convolutions and linear attention on the package's operators:
trained for a few steps on packed documents, then served (prompts of several lengths
packed into one prefill, and decode steps on a pool of states).

    python causal-conv1d-mojo_amd/examples/linear_attn_lm.py

Documents lie one behind another in one row of tokens, (1, tokens); every operator takes
slices of the projections as they lie, so nothing is copied between them.
"""

from __future__ import annotations

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
class Pack:
    """Where the documents of a row of tokens begin, and each token's place in its own."""

    cu: torch.Tensor  # (documents + 1,) int32
    ids: torch.Tensor  # (1, tokens) int32
    positions: torch.Tensor  # (1, tokens)

    @classmethod
    def of(cls, lengths: list[int], device: str = "cuda") -> Pack:
        n = torch.tensor(lengths)
        cu = F.pad(n.cumsum(0), (1, 0))
        ids = torch.repeat_interleave(torch.arange(len(lengths)), n)
        positions = torch.arange(int(cu[-1])) - cu[ids]
        return cls(cu.to(torch.int32).to(device), ids.to(torch.int32).to(device)[None], positions.to(device)[None])


@dataclass
class Cache:
    """The states of every layer, a row per served sequence."""

    conv: list[torch.Tensor]  # (rows, channels, WIDTH - 1)
    attn: list[torch.Tensor]  # (rows, heads, dk, dv) fp32


class Layer(nn.Module):
    def __init__(self, dim: int, heads: int, key_heads: int, head: int, dtype: torch.dtype, device: str) -> None:
        super().__init__()
        self.heads, self.key_heads, self.head = heads, key_heads, head
        keys, values = key_heads * head, heads * head
        self.sizes, self.mixed = (2 * keys + values, values, heads), (keys, keys, values)
        like = {"dtype": dtype, "device": device}
        self.norm = nn.Parameter(torch.ones(dim, device=device))
        self.into = nn.Linear(dim, sum(self.sizes), bias=False, **like)
        self.conv_weight = nn.Parameter(torch.randn(self.sizes[0], WIDTH, **like) / WIDTH**0.5)
        self.conv_bias = nn.Parameter(torch.zeros(self.sizes[0], **like))
        self.q_norm = nn.Parameter(torch.ones(head, device=device))
        self.k_norm = nn.Parameter(torch.full((head,), head**-0.5, device=device))
        # decays of the heads between exp(-0.01) and exp(-1) before the inputs move them
        self.decay_bias = nn.Parameter(torch.logspace(-2, 0, heads, device=device).expm1().log().to(dtype))
        self.out = nn.Linear(values, dim, bias=False, **like)

    def split(self, x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        q, k, v = x.split(self.mixed, dim=-1)
        return tuple(t.unflatten(-1, (n, self.head)) for t, n in ((q, self.key_heads), (k, self.key_heads), (v, self.heads)))

    def log_decay(self, x: torch.Tensor) -> torch.Tensor:
        return -F.softplus(x + self.decay_bias)

    def forward(self, h, stream, pack: Pack, freq, cache=None):
        """h (1, tokens, dim), the residual stream so far; ``cache``: (conv states, attention states) to fill."""
        h, stream = cc.add_norm_fn(h, self.norm, None, stream, rms=True, return_residual=True)
        x, gate, decay = self.into(h).split(self.sizes, dim=-1)
        if cache is not None:
            cache[0].copy_(cc.causal_conv1d_varlen_states(x[0], pack.cu, WIDTH - 1))
        x = cc.causal_conv1d_fn(x.transpose(1, 2), self.conv_weight, self.conv_bias, seq_idx=pack.ids, activation="silu")
        q, k, v = self.split(x.transpose(1, 2))
        q, k = cc.head_norm_rotary_fn(q, k, self.q_norm, self.k_norm, freq, pack.positions)
        y = cc.linear_attn_fn(q, k, v, self.log_decay(decay), cu_seqlens=pack.cu, return_final_states=cache is not None)
        if cache is not None:
            y, states = y
            cache[1].copy_(states)
        return self.out(y.flatten(-2) * F.silu(gate)), stream

    def decode(self, h, stream, conv, attn, rows, freq, positions):
        """One token of each sequence: h (batch, dim), positions (batch,); rows (batch,) int32 (< 0: a free slot)."""
        h, stream = cc.add_norm_fn(h, self.norm, None, stream, rms=True, return_residual=True)
        x, gate, decay = self.into(h).split(self.sizes, dim=-1)
        x = cc.causal_conv1d_update(x, conv, self.conv_weight, self.conv_bias, activation="silu", conv_state_indices=rows)
        q, k, v = self.split(x)
        q, k = cc.head_norm_rotary_fn(q, k, self.q_norm, self.k_norm, freq, positions)
        y = cc.linear_attn_update(q, attn, k, v, self.log_decay(decay), attn_state_indices=rows)
        return self.out(y.flatten(-2) * F.silu(gate)), stream


class LinearAttnLM(nn.Module):
    def __init__(self, vocab=256, dim=128, layers=2, heads=4, key_heads=2, head=64,
                 dtype=torch.bfloat16, device="cuda") -> None:
        super().__init__()
        self.embed = nn.Embedding(vocab, dim, dtype=dtype, device=device)
        self.layers = nn.ModuleList(Layer(dim, heads, key_heads, head, dtype, device) for _ in range(layers))
        self.norm = nn.Parameter(torch.ones(dim, device=device))
        self.head = nn.Linear(dim, vocab, bias=False, dtype=dtype, device=device)
        self.register_buffer("freq", cc.rotary_frequencies(head // 2, device=device)[0])

    def hidden(self, tokens: torch.Tensor, pack: Pack, caches=None) -> torch.Tensor:
        h = self.embed(tokens)
        stream = torch.zeros_like(h, dtype=torch.float32)  # the residual stream stays in 32 bits
        for i, layer in enumerate(self.layers):
            h, stream = layer(h, stream, pack, self.freq, None if caches is None else caches[i])
        return cc.add_norm_fn(h, self.norm, None, stream, rms=True)

    def forward(self, tokens: torch.Tensor, pack: Pack) -> torch.Tensor:
        """Logits of (1, tokens) tokens."""
        return self.head(self.hidden(tokens, pack))

    def new_cache(self, rows: int) -> Cache:
        f = self.layers[0]
        like = {"device": f.norm.device}
        return Cache([torch.zeros(rows, f.sizes[0], WIDTH - 1, dtype=f.conv_bias.dtype, **like) for _ in self.layers],
                     [torch.zeros(rows, f.heads, f.head, f.head, **like) for _ in self.layers])

    @torch.no_grad()
    def prefill(self, prompts: list[torch.Tensor], cache: Cache, rows: torch.Tensor) -> torch.Tensor:
        """Prompts of any lengths as one packed row; their states go to ``rows``. Logits after each prompt."""
        pack = Pack.of([len(p) for p in prompts], str(rows.device))
        new = [(c.new_empty(len(prompts), *c.shape[1:]), a.new_empty(len(prompts), *a.shape[1:]))
               for c, a in zip(cache.conv, cache.attn)]
        h = self.hidden(torch.cat(prompts).to(rows.device)[None], pack, new)
        for (c, a), conv, attn in zip(new, cache.conv, cache.attn):
            conv[rows.long()], attn[rows.long()] = c, a
        return self.head(h[0, (pack.cu[1:] - 1).long()])

    @torch.no_grad()
    def decode(self, tokens: torch.Tensor, positions: torch.Tensor, cache: Cache, rows: torch.Tensor) -> torch.Tensor:
        """Logits after one more token (batch,), at ``positions``, of the sequences whose states are ``rows``."""
        h = self.embed(tokens)
        stream = torch.zeros_like(h, dtype=torch.float32)
        for layer, conv, attn in zip(self.layers, cache.conv, cache.attn):
            h, stream = layer.decode(h, stream, conv, attn, rows, self.freq, positions)
        return self.head(cc.add_norm_fn(h, self.norm, None, stream, rms=True))


def loss_of(model: LinearAttnLM, tokens: torch.Tensor, pack: Pack) -> torch.Tensor:
    """Next-token loss; a document's last token predicts nothing."""
    logits = model(tokens, pack)[0, :-1]
    inside = pack.ids[0, 1:] == pack.ids[0, :-1]
    return F.cross_entropy(logits[inside].float(), tokens[0, 1:][inside])


def train(model: LinearAttnLM, tokens: torch.Tensor, pack: Pack, steps: int, lr: float = 3e-3) -> list[float]:
    opt = torch.optim.AdamW(model.parameters(), lr=lr)
    losses = []
    for _ in range(steps):
        loss = loss_of(model, tokens, pack)
        opt.zero_grad()
        loss.backward()
        opt.step()
        losses.append(loss.item())
    return losses


def main() -> None:
    torch.manual_seed(0)
    model = LinearAttnLM()
    lengths = [300, 17, 512, 195]
    tokens = torch.randint(256, (1, sum(lengths)), device="cuda")
    losses = train(model, tokens, Pack.of(lengths), 40)
    print(f"loss {losses[0]:.3f} -> {losses[-1]:.3f}")

    rows = torch.tensor([5, 0, 3], dtype=torch.int32, device="cuda")
    prompts = [tokens[0, :100].cpu(), tokens[0, 300:317].cpu(), tokens[0, 317:320].cpu()]
    cache = model.new_cache(8)
    token = model.prefill(prompts, cache, rows).argmax(-1)
    positions = torch.tensor([len(p) for p in prompts], device="cuda")
    out = [token]
    for _ in range(15):
        token = model.decode(token, positions, cache, rows).argmax(-1)
        positions = positions + 1
        out.append(token)
    for text in torch.stack(out, 1).tolist():
        print(*text)


if __name__ == "__main__":
    main()
