"""``add_norm_fn``: residual add and layer / rms norm in one pass, forward and
autograd backward on MI355X -- what stands between two layers::

    r = x + residual
    y = (r - mean) * rstd * weight + bias       (rms: mean = 0)

with the statistics, y and the gradients taken from the fp32 sum; the new
residual stream is that sum in the residual's dtype. The parameter gradients
run in a fixed order (the same inputs give the same bits).
"""

from __future__ import annotations

import torch

from causal_conv1d_amd import _host
from causal_conv1d_amd._dtype import _DTYPE_CODE
from causal_conv1d_amd._native import native_norm_bwd, native_norm_fwd

MAX_NORM_DIM = 32768


def _norm_fwd_impl(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None,
    residual: torch.Tensor | None,
    eps: float,
    rms: bool,
    y: torch.Tensor,
    sum: torch.Tensor | None,
    stats: torch.Tensor | None,
) -> None:
    native_norm_fwd(x, weight, bias, residual, eps, rms, y, sum, stats)


def _norm_fwd_fake(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None,
    residual: torch.Tensor | None,
    eps: float,
    rms: bool,
    y: torch.Tensor,
    sum: torch.Tensor | None,
    stats: torch.Tensor | None,
) -> None:
    return None


_norm_fwd_inplace = torch.library.custom_op(
    "causal_conv1d_amd::_norm_fwd_inplace",
    mutates_args=("y", "sum", "stats"),
)(_norm_fwd_impl)
_norm_fwd_inplace.register_fake(_norm_fwd_fake)


def _norm_bwd_impl(
    x: torch.Tensor | None,
    weight: torch.Tensor,
    residual: torch.Tensor | None,
    stats: torch.Tensor,
    rms: bool,
    dy: torch.Tensor,
    dsum: torch.Tensor | None,
    dx: torch.Tensor,
    dresidual: torch.Tensor | None,
    dweight: torch.Tensor,
    dbias: torch.Tensor | None,
) -> None:
    native_norm_bwd(x, weight, residual, stats, rms, dy, dsum, dx, dresidual, dweight, dbias)


def _norm_bwd_fake(
    x: torch.Tensor | None,
    weight: torch.Tensor,
    residual: torch.Tensor | None,
    stats: torch.Tensor,
    rms: bool,
    dy: torch.Tensor,
    dsum: torch.Tensor | None,
    dx: torch.Tensor,
    dresidual: torch.Tensor | None,
    dweight: torch.Tensor,
    dbias: torch.Tensor | None,
) -> None:
    return None


_norm_bwd_inplace = torch.library.custom_op(
    "causal_conv1d_amd::_norm_bwd_inplace",
    mutates_args=("dx", "dresidual", "dweight", "dbias"),
)(_norm_bwd_impl)
_norm_bwd_inplace.register_fake(_norm_bwd_fake)


class _AddNormFn(torch.autograd.Function):
    """On (rows, dim) tensors. Saves each row's mean and rstd, and the sum:
    the returned one where it is fp32, x and the residual otherwise (a sum
    rounded to 16 bits would put its rounding into the parameter gradients)."""

    @staticmethod
    def forward(ctx, x, weight, bias, residual, eps, rms, return_residual):
        y = torch.empty_like(x)
        total = torch.empty_like(residual) if return_residual else None
        stats = None
        if any(ctx.needs_input_grad):
            stats = torch.empty(x.shape[0], 2, dtype=torch.float32, device=x.device)
        torch.ops.causal_conv1d_amd._norm_fwd_inplace(x, weight, bias, residual, eps, rms, y, total, stats)
        exact = total is not None and total.dtype == torch.float32
        ctx.save_for_backward(None if exact else x, weight, total if exact else residual, stats)
        ctx.rms, ctx.x_dtype, ctx.has_bias, ctx.has_residual = rms, x.dtype, bias is not None, residual is not None
        ctx.set_materialize_grads(False)
        return (y, total) if return_residual else y

    @staticmethod
    def backward(ctx, *grads):
        x, weight, residual, stats = ctx.saved_tensors
        dy = grads[0]
        dsum = grads[1] if len(grads) > 1 else None
        like = x if x is not None else residual
        if dy is None:
            if dsum is None:
                return (None,) * 7
            dy = torch.zeros(like.shape, dtype=ctx.x_dtype, device=like.device)
        dy = _rows(dy)
        if dsum is not None:
            dsum = _rows(dsum)
        dx = torch.empty(like.shape, dtype=ctx.x_dtype, device=like.device)
        # one tensor serves both gradients where their dtypes agree
        apart = ctx.has_residual and residual.dtype != ctx.x_dtype
        dresidual = torch.empty(like.shape, dtype=residual.dtype, device=like.device) if apart else None
        dweight = torch.empty(weight.shape, dtype=weight.dtype, device=like.device)
        dbias = torch.empty_like(dweight) if ctx.has_bias else None
        torch.ops.causal_conv1d_amd._norm_bwd_inplace(x, weight, residual, stats, ctx.rms, dy, dsum, dx, dresidual,
                                                      dweight, dbias)
        if ctx.has_residual and not apart:
            dresidual = dx
        return dx, dweight, dbias, dresidual, None, None, None


def _rows(t: torch.Tensor) -> torch.Tensor:
    """(rows, dim) with contiguous rows."""
    return t if t.stride(1) == 1 or t.shape[1] == 1 else t.contiguous()


def add_norm_fn(
    x: torch.Tensor,
    weight: torch.Tensor,
    bias: torch.Tensor | None = None,
    residual: torch.Tensor | None = None,
    eps: float = 1e-5,
    rms: bool = False,
    return_residual: bool = False,
) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """
    x: (..., dim), fp16 / bf16 / fp32, dim in 1..32768
    weight, bias: (dim,) fp32
    residual: shape of x, x's dtype or fp32; None adds nothing
    rms: root mean square norm (no mean is taken off)
    return_residual: also return x + residual in the residual's dtype (x itself without a residual)

    Returns y (x's dtype), or (y, residual stream). Gradients reach x, weight, bias and residual.
    """
    if getattr(x, "is_cuda", False) and not torch.compiler.is_compiling():
        # an ordinary call, checked, recorded and launched in native code
        r = _host.native().add_norm(x, weight, bias, residual, eps, rms, return_residual)
        if r is not NotImplemented:
            return r
    if x.dtype not in _DTYPE_CODE:
        raise NotImplementedError(f"unsupported dtype {x.dtype}; only fp16/bf16/fp32 are supported")
    if x.dim() < 1:
        raise ValueError("expected x of shape (..., dim)")
    dim = x.shape[-1]
    if dim < 1 or dim > MAX_NORM_DIM:
        raise NotImplementedError(f"dim must be in 1..{MAX_NORM_DIM} (got {dim})")
    for name, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if tuple(t.shape) != (dim,):
            raise ValueError(f"{name} shape {tuple(t.shape)} != expected {(dim,)}")
        if t.dtype != torch.float32:
            raise NotImplementedError(f"{name}.dtype must be torch.float32 (got {t.dtype})")
        if t.device != x.device:
            raise NotImplementedError(f"{name}.device ({t.device}) must match x.device ({x.device})")
    if residual is not None:
        if residual.shape != x.shape:
            raise ValueError(f"residual shape {tuple(residual.shape)} != expected {tuple(x.shape)}")
        if residual.dtype not in (x.dtype, torch.float32):
            raise NotImplementedError(f"residual.dtype ({residual.dtype}) must be x.dtype ({x.dtype}) or torch.float32")
        if residual.device != x.device:
            raise NotImplementedError(f"residual.device ({residual.device}) must match x.device ({x.device})")
    x2 = _rows(x.reshape(-1, dim))
    r2 = None if residual is None else _rows(residual.reshape(-1, dim))
    r = _AddNormFn.apply(x2, weight, bias, r2, float(eps), bool(rms), return_residual and residual is not None)
    if not return_residual:
        return r.reshape(x.shape)
    if residual is None:
        return r.reshape(x.shape), x
    return r[0].reshape(x.shape), r[1].reshape(x.shape)
