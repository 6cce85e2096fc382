"""``linear_attn_fn``: linear attention with a decay for each head over prompts,
forward and autograd backward on MI355X.

The mixer that has a matrix of state where the selective scan has a vector.
Per head, with ``g`` the log of the decay::

    S[t] = exp(g[t]) S[t-1] + k[t] v[t]^T        (dk x dv)
    out[t] = scale * q[t]^T S[t]

The kernel takes chunks of positions on the matrix cores (csrc/cc1d_attn_kernels.hpp).
Tensors are read in the caller's layout on the current stream; nothing is
allocated but outputs and per-call workspaces, and sums run in a fixed order
(the same inputs give the same bits). States are fp32.
"""

from __future__ import annotations

import torch

from causal_conv1d_amd import _host
from causal_conv1d_amd._dtype import _DTYPE_CODE
from causal_conv1d_amd._native import native_attn_bwd, native_attn_fwd
from causal_conv1d_amd._scan import _check_int32, _check_like

MAX_HEAD_DIM = 128


def _attn_fwd_impl(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    cu_seqlens: torch.Tensor | None,
    initial_states: torch.Tensor | None,
    scale: float,
    out: torch.Tensor,
    final_states: torch.Tensor | None,
) -> None:
    native_attn_fwd(q, k, v, g, cu_seqlens, initial_states, scale, out, final_states)


def _attn_fwd_fake(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    cu_seqlens: torch.Tensor | None,
    initial_states: torch.Tensor | None,
    scale: float,
    out: torch.Tensor,
    final_states: torch.Tensor | None,
) -> None:
    return None


_attn_fwd_inplace = torch.library.custom_op(
    "causal_conv1d_amd::_attn_fwd_inplace",
    mutates_args=("out", "final_states"),
)(_attn_fwd_impl)
_attn_fwd_inplace.register_fake(_attn_fwd_fake)


def _attn_bwd_impl(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    cu_seqlens: torch.Tensor | None,
    initial_states: torch.Tensor | None,
    scale: float,
    dout: torch.Tensor,
    dfinal_states: torch.Tensor | None,
    dq: torch.Tensor,
    dk: torch.Tensor,
    dv: torch.Tensor,
    dg: torch.Tensor,
    dinitial_states: torch.Tensor | None,
) -> None:
    native_attn_bwd(q, k, v, g, cu_seqlens, initial_states, scale, dout, dfinal_states, dq, dk, dv, dg,
                    dinitial_states)


def _attn_bwd_fake(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    cu_seqlens: torch.Tensor | None,
    initial_states: torch.Tensor | None,
    scale: float,
    dout: torch.Tensor,
    dfinal_states: torch.Tensor | None,
    dq: torch.Tensor,
    dk: torch.Tensor,
    dv: torch.Tensor,
    dg: torch.Tensor,
    dinitial_states: torch.Tensor | None,
) -> None:
    return None


_attn_bwd_inplace = torch.library.custom_op(
    "causal_conv1d_amd::_attn_bwd_inplace",
    mutates_args=("dq", "dk", "dv", "dg", "dinitial_states"),
)(_attn_bwd_impl)
_attn_bwd_inplace.register_fake(_attn_bwd_fake)


def _flat(t: torch.Tensor | None) -> torch.Tensor | None:
    """Contiguous and empty, t's shape and dtype."""
    return None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)


class _LinearAttnFn(torch.autograd.Function):
    """Saves the inputs; the backward recomputes the states."""

    @staticmethod
    def forward(ctx, q, k, v, g, cu_seqlens, initial_states, scale, final_states):
        out = _flat(v)
        torch.ops.causal_conv1d_amd._attn_fwd_inplace(q, k, v, g, cu_seqlens, initial_states, scale, out, final_states)
        ctx.save_for_backward(q, k, v, g, cu_seqlens, initial_states)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        if final_states is not None:
            return out, final_states
        return out

    @staticmethod
    def backward(ctx, *grads):
        q, k, v, g, cu_seqlens, initial_states = ctx.saved_tensors
        dout, dfinal = grads[0], grads[1] if len(grads) > 1 else None
        if dout is None:
            if dfinal is None:
                return (None,) * 8
            dout = torch.zeros(v.shape, dtype=v.dtype, device=v.device)
        dq, dk, dv, dg, dinitial = (_flat(t) for t in (q, k, v, g, initial_states))
        torch.ops.causal_conv1d_amd._attn_bwd_inplace(q, k, v, g, cu_seqlens, initial_states, ctx.scale, dout, dfinal,
                                                      dq, dk, dv, dg, dinitial)
        return dq, dk, dv, dg, None, dinitial, None, None


def _check_heads(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, layout: str) -> None:
    """q, k, v (.., heads, size) and g (.., heads) against each other."""
    if q.dtype not in _DTYPE_CODE:
        raise NotImplementedError(f"unsupported dtype {q.dtype}; only fp16/bf16/fp32 are supported")
    if v.dim() != q.dim():
        raise ValueError(f"expected q, k and v of shape ({layout}, heads, size); got {tuple(q.shape)}, {tuple(v.shape)}")
    key_heads, dk = q.shape[-2:]
    heads, dv = v.shape[-2:]
    for name, d in (("q", dk), ("v", dv)):
        if d < 1 or d > MAX_HEAD_DIM:
            raise NotImplementedError(f"{name}'s head size must be in 1..{MAX_HEAD_DIM} (got {d})")
    if key_heads < 1 or heads % key_heads != 0:
        raise ValueError(f"v's heads ({heads}) must be a multiple of q's ({key_heads})")
    lead = q.shape[:-2]
    _check_like("k", k, q, q.shape, q.dtype)
    _check_like("v", v, q, (*lead, heads, dv), q.dtype)
    _check_like("g", g, q, (*lead, heads), q.dtype)


def linear_attn_fn(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    g: torch.Tensor,
    scale: float | None = None,
    cu_seqlens: torch.Tensor | None = None,
    initial_states: torch.Tensor | None = None,
    return_final_states: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """
    q, k: (batch, seqlen, key_heads, dk), fp16 / bf16 / fp32, dk in 1..128, any strides (values of a head next to
        each other are fast)
    v: (batch, seqlen, heads, dv), dtype of q, dv in 1..128; heads a multiple of key_heads: head h reads key head
        h // (heads // key_heads)
    g: (batch, seqlen, heads), dtype of q: log of the decay, 0 or less (-inf keeps nothing); a decay that is the same
        everywhere may be expanded
    scale: on the outputs; dk ** -0.5 if None
    cu_seqlens: (sequences + 1,) int32, non-decreasing from 0 to seqlen: sequences packed into one batch row
        (batch == 1), each with its own states; positions that no sequence covers give 0
    initial_states: (batch or sequences, heads, dk, dv) fp32
    return_final_states: also return the states after the last positions, (batch or sequences, heads, dk, dv) fp32
        (the initial ones for a sequence of no positions)

    Returns out (batch, seqlen, heads, dv), contiguous, or (out, final_states). Gradients reach every float argument
    and flow through final_states.
    """
    if getattr(q, "is_cuda", False) and not torch.compiler.is_compiling():
        # an ordinary call, checked, recorded and launched in native code
        r = _host.native().linear_attn(q, k, v, g, scale, cu_seqlens, initial_states, return_final_states)
        if r is not NotImplemented:
            return r
    if q.dim() != 4:
        raise ValueError(f"expected q of shape (batch, seqlen, key_heads, dk); got {tuple(q.shape)}")
    _check_heads(q, k, v, g, "batch, seqlen")
    batch, seqlen, _, dk = q.shape
    heads, dv = v.shape[2:]
    sequences = batch
    if cu_seqlens is not None:
        if batch != 1:
            raise ValueError(f"cu_seqlens needs batch == 1 (got {batch})")
        if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < (2 if seqlen else 1):
            raise ValueError(f"cu_seqlens shape {tuple(cu_seqlens.shape)}: expected (sequences + 1,)")
        cu_seqlens = _check_int32("cu_seqlens", cu_seqlens, q, cu_seqlens.shape)
        sequences = cu_seqlens.shape[0] - 1
    _check_like("initial_states", initial_states, q, (sequences, heads, dk, dv), torch.float32)
    final_states = None
    if return_final_states:
        final_states = torch.empty(sequences, heads, dk, dv, dtype=torch.float32, device=q.device)
    return _LinearAttnFn.apply(q, k, v, g, cu_seqlens, initial_states, dk**-0.5 if scale is None else float(scale),
                               final_states)
