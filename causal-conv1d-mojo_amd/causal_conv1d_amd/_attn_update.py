"""``linear_attn_update``: linear attention with a decay for each head, for the
new tokens of a decode batch, on a state pool updated in place (the counterpart
of ``ssm_scan_update``). No autograd.
"""

from __future__ import annotations

import torch

from causal_conv1d_amd import _host
from causal_conv1d_amd._attn import _check_heads, _flat
from causal_conv1d_amd._native import native_attn_update
from causal_conv1d_amd._scan import _check_int32, _check_like


def _attn_update_impl(
    q: torch.Tensor,
    attn_state: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    scale: float,
    attn_state_indices: torch.Tensor | None,
    out: torch.Tensor,
) -> None:
    native_attn_update(q, attn_state, k, v, g, scale, attn_state_indices, out)


def _attn_update_fake(
    q: torch.Tensor,
    attn_state: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    scale: float,
    attn_state_indices: torch.Tensor | None,
    out: torch.Tensor,
) -> None:
    return None


_attn_update_inplace = torch.library.custom_op(
    "causal_conv1d_amd::_attn_update_inplace",
    mutates_args=("attn_state", "out"),
)(_attn_update_impl)
_attn_update_inplace.register_fake(_attn_update_fake)


def linear_attn_update(
    q: torch.Tensor,
    attn_state: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    scale: float | None = None,
    attn_state_indices: torch.Tensor | None = None,
) -> torch.Tensor:
    """
    q, k: (batch, key_heads, dk) or (batch, tokens, key_heads, dk) -- the new tokens, fp16 / bf16 / fp32
    attn_state: (batch_or_pool_size, heads, dk, dv) fp32; mutated in place, as autograd is told: a backward of
        ``linear_attn_fn`` that went on from this buffer before raises
    v: (batch, [tokens,] heads, dv), g: (batch, [tokens,] heads), as in ``linear_attn_fn``
    scale: on the outputs; dk ** -0.5 if None
    attn_state_indices: (batch,) int32 or None -- state row per batch entry, distinct; < 0 marks padding

    Returns: out, shape of v, contiguous (0 for padding, whose state rows stay as they are).
    """
    if getattr(q, "is_cuda", False) and not torch.compiler.is_compiling():
        # an ordinary call, checked and launched in native code
        out = _host.native().linear_attn_update(q, attn_state, k, v, g, scale, attn_state_indices)
        if out is not NotImplemented:
            return out
    if q.dim() not in (3, 4) or attn_state.dim() != 4:
        raise ValueError(
            f"expected q (batch, [tokens,] key_heads, dk) and attn_state (rows, heads, dk, dv); "
            f"got q {tuple(q.shape)}, attn_state {tuple(attn_state.shape)}"
        )
    _check_heads(q, k, v, g, "batch[, tokens]")
    batch, dk = q.shape[0], q.shape[-1]
    heads, dv = v.shape[-2:]
    rows = batch if attn_state_indices is None else attn_state.shape[0]
    _check_like("attn_state", attn_state, q, (rows, heads, dk, dv), torch.float32)
    if attn_state_indices is not None:
        attn_state_indices = _check_int32("attn_state_indices", attn_state_indices, q, (batch,))
    with torch.no_grad():
        out = _flat(v)
        parts = (q, k, v, g, out) if q.dim() == 4 else tuple(t.unsqueeze(1) for t in (q, k, v, g, out))
        torch.ops.causal_conv1d_amd._attn_update_inplace(
            parts[0], attn_state, *parts[1:4], dk**-0.5 if scale is None else float(scale), attn_state_indices, parts[4])
        return out
