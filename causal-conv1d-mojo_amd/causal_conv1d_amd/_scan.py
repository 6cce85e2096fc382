"""``ssm_scan_fn``: the selective state space scan over prompts, forward and
autograd backward on MI355X.

What a state space layer runs on the convolution's output. Per channel, with
``dt = softplus(delta + delta_bias)`` and ``dstate`` values of state::

    h[t] = exp(dt[t] A) h[t-1] + dt[t] u[t] B[t]
    y[t] = sum_n C[t, n] h[t, n] + D u[t]
    out[t] = y[t] * silu(z[t])          (y[t] without z)

As for the convolution, the kernels read and write tensors in the caller's
layout on the current stream, allocate nothing but outputs and per-call
workspaces, and run their sums in a fixed order (the same inputs give the
same bits). States, parameters and all arithmetic are fp32.
"""

from __future__ import annotations

import torch

from causal_conv1d_amd import _host
from causal_conv1d_amd._dtype import _DTYPE_CODE
from causal_conv1d_amd._fn import _match_layout
from causal_conv1d_amd._native import native_scan_bwd, native_scan_fwd

MAX_DSTATE = 256


def scan_tile(seqlen: int) -> int:
    """Positions between the states that a training forward keeps for the backward (csrc/cc1d_scan_device.hpp)."""
    return 256 if seqlen <= 256 else 512


def scan_tile_floats(u: torch.Tensor, A: torch.Tensor, cu_seqlens: torch.Tensor | None) -> int:
    """cc1d_scan_tile_floats of these inputs, in arithmetic that torch.compile can trace."""
    batch, dim, seqlen = u.shape
    tile = scan_tile(seqlen)
    if cu_seqlens is not None:
        return (seqlen // tile + cu_seqlens.shape[0] - 1) * dim * A.shape[1]
    return batch * ((seqlen + tile - 1) // tile) * dim * A.shape[1]


def _scan_fwd_impl(
    u: torch.Tensor,
    delta: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: torch.Tensor | None,
    z: torch.Tensor | None,
    delta_bias: torch.Tensor | None,
    seq_idx: torch.Tensor | None,
    cu_seqlens: torch.Tensor | None,
    initial_states: torch.Tensor | None,
    delta_softplus: bool,
    out: torch.Tensor,
    final_states: torch.Tensor | None,
    tile_states: torch.Tensor | None,
) -> None:
    native_scan_fwd(u, delta, A, B, C, D, z, delta_bias, seq_idx, cu_seqlens, initial_states, delta_softplus, out,
                    final_states, tile_states)


def _scan_fwd_fake(
    u: torch.Tensor,
    delta: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: torch.Tensor | None,
    z: torch.Tensor | None,
    delta_bias: torch.Tensor | None,
    seq_idx: torch.Tensor | None,
    cu_seqlens: torch.Tensor | None,
    initial_states: torch.Tensor | None,
    delta_softplus: bool,
    out: torch.Tensor,
    final_states: torch.Tensor | None,
    tile_states: torch.Tensor | None,
) -> None:
    return None


_scan_fwd_inplace = torch.library.custom_op(
    "causal_conv1d_amd::_scan_fwd_inplace",
    mutates_args=("out", "final_states", "tile_states"),
)(_scan_fwd_impl)
_scan_fwd_inplace.register_fake(_scan_fwd_fake)


def _scan_bwd_impl(
    u: torch.Tensor,
    delta: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: torch.Tensor | None,
    z: torch.Tensor | None,
    delta_bias: torch.Tensor | None,
    seq_idx: torch.Tensor | None,
    cu_seqlens: torch.Tensor | None,
    tile_states: torch.Tensor,
    dout: torch.Tensor,
    dfinal_states: torch.Tensor | None,
    delta_softplus: bool,
    du: torch.Tensor,
    ddelta: torch.Tensor,
    dA: torch.Tensor,
    dB: torch.Tensor,
    dC: torch.Tensor,
    dD: torch.Tensor | None,
    dz: torch.Tensor | None,
    ddelta_bias: torch.Tensor | None,
    dinitial_states: torch.Tensor | None,
) -> None:
    native_scan_bwd(u, delta, A, B, C, D, z, delta_bias, seq_idx, cu_seqlens, tile_states, dout, dfinal_states,
                    delta_softplus, du, ddelta, dA, dB, dC, dD, dz, ddelta_bias, dinitial_states)


def _scan_bwd_fake(
    u: torch.Tensor,
    delta: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: torch.Tensor | None,
    z: torch.Tensor | None,
    delta_bias: torch.Tensor | None,
    seq_idx: torch.Tensor | None,
    cu_seqlens: torch.Tensor | None,
    tile_states: torch.Tensor,
    dout: torch.Tensor,
    dfinal_states: torch.Tensor | None,
    delta_softplus: bool,
    du: torch.Tensor,
    ddelta: torch.Tensor,
    dA: torch.Tensor,
    dB: torch.Tensor,
    dC: torch.Tensor,
    dD: torch.Tensor | None,
    dz: torch.Tensor | None,
    ddelta_bias: torch.Tensor | None,
    dinitial_states: torch.Tensor | None,
) -> None:
    return None


_scan_bwd_inplace = torch.library.custom_op(
    "causal_conv1d_amd::_scan_bwd_inplace",
    mutates_args=("du", "ddelta", "dA", "dB", "dC", "dD", "dz", "ddelta_bias", "dinitial_states"),
)(_scan_bwd_impl)
_scan_bwd_inplace.register_fake(_scan_bwd_fake)


class _SsmScanFn(torch.autograd.Function):
    """Saves the inputs and the states at the kernel's tile boundaries; the
    backward recomputes the states inside a tile."""

    @staticmethod
    def forward(ctx, u, delta, A, B, C, D, z, delta_bias, seq_idx, cu_seqlens, initial_states, delta_softplus,
                final_states):
        out = torch.empty_like(u)
        tiles = None
        if any(ctx.needs_input_grad):
            n = scan_tile_floats(u, A, cu_seqlens)
            tiles = torch.empty(n, dtype=torch.float32, device=u.device)
        torch.ops.causal_conv1d_amd._scan_fwd_inplace(
            u, delta, A, B, C, D, z, delta_bias, seq_idx, cu_seqlens, initial_states, delta_softplus, out,
            final_states, tiles
        )
        ctx.save_for_backward(u, delta, A, B, C, D, z, delta_bias, seq_idx, cu_seqlens, initial_states, tiles)
        ctx.delta_softplus = delta_softplus
        ctx.has_final = final_states is not None
        if final_states is not None:
            return out, final_states
        return out

    @staticmethod
    def backward(ctx, *grad_outputs):
        u, delta, A, B, C, D, z, delta_bias, seq_idx, cu_seqlens, initial_states, tiles = ctx.saved_tensors
        dout = _match_layout(grad_outputs[0], u)
        dfinal = grad_outputs[1] if ctx.has_final else None
        new = lambda t: None if t is None else torch.empty_like(t)  # noqa: E731
        flat = lambda t: None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)  # noqa: E731
        du, ddelta, dz = new(u), new(delta), new(z)
        dA, dB, dC, dD, dbias, dinit = (flat(t) for t in (A, B, C, D, delta_bias, initial_states))
        torch.ops.causal_conv1d_amd._scan_bwd_inplace(
            u, delta, A, B, C, D, z, delta_bias, seq_idx, cu_seqlens, tiles, dout, dfinal, ctx.delta_softplus,
            du, ddelta, dA, dB, dC, dD, dz, dbias, dinit
        )
        return du, ddelta, dA, dB, dC, dD, dz, dbias, None, None, dinit, None, None


def _check_like(name: str, t: torch.Tensor | None, u: torch.Tensor, shape: tuple, dtype: torch.dtype) -> None:
    if t is None:
        return
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} shape {tuple(t.shape)} != expected {tuple(shape)}")
    if t.dtype != dtype:
        raise NotImplementedError(f"{name}.dtype must be {dtype} (got {t.dtype})")
    if t.device != u.device:
        raise NotImplementedError(f"{name}.device ({t.device}) must match u.device ({u.device})")


def _check_parameters(u: torch.Tensor, A: torch.Tensor, D, delta_bias, dim: int) -> int:
    """A, D and delta_bias against u and its dim; dstate."""
    if u.dtype not in _DTYPE_CODE:
        raise NotImplementedError(f"unsupported dtype {u.dtype}; only fp16/bf16/fp32 are supported")
    if A.dim() != 2:
        raise ValueError(f"A shape {tuple(A.shape)}: expected (dim, dstate)")
    dstate = A.shape[1]
    if dstate < 1 or dstate > MAX_DSTATE:
        raise NotImplementedError(f"dstate must be in 1..{MAX_DSTATE} (got {dstate})")
    _check_like("A", A, u, (dim, dstate), torch.float32)
    _check_like("D", D, u, (dim,), torch.float32)
    _check_like("delta_bias", delta_bias, u, (dim,), torch.float32)
    return dstate


def _check_int32(name: str, t: torch.Tensor, u: torch.Tensor, shape: tuple) -> torch.Tensor:
    if tuple(t.shape) != tuple(shape):
        raise ValueError(f"{name} shape {tuple(t.shape)} != expected {tuple(shape)}")
    if t.dtype != torch.int32:
        raise ValueError(f"{name}.dtype must be int32 (got {t.dtype})")
    if t.device != u.device:
        raise ValueError(f"{name}.device ({t.device}) must match u.device ({u.device})")
    return t if t.is_contiguous() else t.contiguous()


def ssm_scan_fn(
    u: torch.Tensor,
    delta: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: torch.Tensor | None = None,
    z: torch.Tensor | None = None,
    delta_bias: torch.Tensor | None = None,
    delta_softplus: bool = False,
    seq_idx: torch.Tensor | None = None,
    cu_seqlens: torch.Tensor | None = None,
    initial_states: torch.Tensor | None = None,
    return_final_states: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """
    u, delta, z: (batch, dim, seqlen), fp16 / bf16 / fp32; channel-first and channel-last layouts are fast where
        the three lie alike; B and C may lie either way beside them. Other strides, or one tensor unlike the rest,
        are read element by element (two to three times as long)
    A: (dim, dstate) fp32 (real), dstate in 1..256; D, delta_bias: (dim,) fp32
    B, C: (batch, dstate, seqlen) or (batch, groups, dstate, seqlen), dtype of u; dim a multiple of groups
    delta_softplus: dt = softplus(delta + delta_bias) instead of delta + delta_bias
    seq_idx: (batch, seqlen) int32: the state starts at 0 where the id changes; positions with an id < 0
        (padding) give 0 and take no part
    cu_seqlens: (sequences + 1,) int32, non-decreasing from 0 to seqlen: sequences packed into one batch row
        (batch == 1), each with its own row of states; positions that no sequence covers give 0
    initial_states: (batch or sequences, dim, dstate) fp32
    return_final_states: also return the states after the last positions, (batch or sequences, dim, dstate) fp32
        (the initial ones for a sequence of no positions)

    Returns out (batch, dim, seqlen) in u's dtype and layout, or (out, final_states). Gradients reach every
    float argument and flow through final_states.
    """
    if getattr(u, "is_cuda", False) and not torch.compiler.is_compiling():
        # an ordinary call, checked, recorded and launched in native code
        r = _host.native().ssm_scan(u, delta, A, B, C, D, z, delta_bias, delta_softplus, seq_idx, cu_seqlens,
                                    initial_states, return_final_states)
        if r is not NotImplemented:
            return r
    if u.dim() != 3:
        raise ValueError(f"expected u of shape (batch, dim, seqlen); got {tuple(u.shape)}")
    batch, dim, seqlen = u.shape
    dstate = _check_parameters(u, A, D, delta_bias, dim)
    _check_like("delta", delta, u, u.shape, u.dtype)
    _check_like("z", z, u, u.shape, u.dtype)
    if B.dim() not in (3, 4) or C.dim() != B.dim():
        raise ValueError(
            f"expected B and C of shape (batch, [groups,] dstate, seqlen); got {tuple(B.shape)}, {tuple(C.shape)}"
        )
    if B.dim() == 3:
        B, C = B.unsqueeze(1), C.unsqueeze(1)
    groups = B.shape[1]
    if groups < 1 or dim % groups != 0:
        raise ValueError(f"dim ({dim}) must be a multiple of B's groups ({groups})")
    _check_like("B", B, u, (batch, groups, dstate, seqlen), u.dtype)
    _check_like("C", C, u, (batch, groups, dstate, seqlen), u.dtype)

    if seq_idx is not None:
        if cu_seqlens is not None:
            raise ValueError("seq_idx and cu_seqlens are mutually exclusive")
        if return_final_states or initial_states is not None:
            raise ValueError(
                "seq_idx and initial_states / return_final_states are mutually exclusive "
                "(cu_seqlens gives every packed sequence its states)"
            )
        seq_idx = _check_int32("seq_idx", seq_idx, u, (batch, seqlen))
    sequences = batch
    if cu_seqlens is not None:
        if batch != 1:
            raise ValueError(f"cu_seqlens needs batch == 1 (got {batch})")
        if cu_seqlens.dim() != 1 or cu_seqlens.shape[0] < (2 if seqlen else 1):
            raise ValueError(f"cu_seqlens shape {tuple(cu_seqlens.shape)}: expected (sequences + 1,)")
        cu_seqlens = _check_int32("cu_seqlens", cu_seqlens, u, cu_seqlens.shape)
        sequences = cu_seqlens.shape[0] - 1
    _check_like("initial_states", initial_states, u, (sequences, dim, dstate), torch.float32)
    final_states = None
    if return_final_states:
        final_states = torch.empty(sequences, dim, dstate, dtype=torch.float32, device=u.device)
    return _SsmScanFn.apply(u, delta, A, B, C, D, z, delta_bias, seq_idx, cu_seqlens, initial_states,
                            bool(delta_softplus), final_states)
