"""``head_norm_rotary_fn``: norm of each query and key head and rotation by
position in one pass, forward and autograd backward on MI355X -- what runs on
queries and keys between their projection and the attention::

    x^ = x / sqrt(mean(x^2) + eps) * weight      (x without a weight)
    (a, b) -> amplitude * (a cos t - b sin t, b cos t + a sin t),   t = position * inv_freq[i]

over the pairs of the first ``2 * len(inv_freq)`` values of a head. Angles are
formed in 64 bits, the rest is fp32 and rounded once. The weights' gradients
run in a fixed order (the same inputs give the same bits).
"""

from __future__ import annotations

import math

import torch

from causal_conv1d_amd import _host
from causal_conv1d_amd._attn import _flat
from causal_conv1d_amd._dtype import _DTYPE_CODE
from causal_conv1d_amd._native import native_rotary_bwd, native_rotary_fwd

MAX_ROTARY_DIM = 256


def _rotary_fwd_impl(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor | None,
    k_weight: torch.Tensor | None,
    inv_freq: torch.Tensor | None,
    positions: torch.Tensor | None,
    eps: float,
    interleaved: bool,
    amplitude: float,
    q_out: torch.Tensor,
    k_out: torch.Tensor,
) -> None:
    native_rotary_fwd(q, k, q_weight, k_weight, inv_freq, positions, eps, interleaved, amplitude, q_out, k_out)


def _rotary_fwd_fake(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor | None,
    k_weight: torch.Tensor | None,
    inv_freq: torch.Tensor | None,
    positions: torch.Tensor | None,
    eps: float,
    interleaved: bool,
    amplitude: float,
    q_out: torch.Tensor,
    k_out: torch.Tensor,
) -> None:
    return None


_rotary_fwd_inplace = torch.library.custom_op(
    "causal_conv1d_amd::_rotary_fwd_inplace",
    mutates_args=("q_out", "k_out"),
)(_rotary_fwd_impl)
_rotary_fwd_inplace.register_fake(_rotary_fwd_fake)


def _rotary_bwd_impl(
    q: torch.Tensor | None,
    k: torch.Tensor | None,
    q_weight: torch.Tensor | None,
    k_weight: torch.Tensor | None,
    inv_freq: torch.Tensor | None,
    positions: torch.Tensor | None,
    eps: float,
    interleaved: bool,
    amplitude: float,
    dq_out: torch.Tensor,
    dk_out: torch.Tensor,
    dq: torch.Tensor,
    dk: torch.Tensor,
    dq_weight: torch.Tensor | None,
    dk_weight: torch.Tensor | None,
) -> None:
    native_rotary_bwd(q, k, q_weight, k_weight, inv_freq, positions, eps, interleaved, amplitude, dq_out, dk_out, dq,
                      dk, dq_weight, dk_weight)


def _rotary_bwd_fake(
    q: torch.Tensor | None,
    k: torch.Tensor | None,
    q_weight: torch.Tensor | None,
    k_weight: torch.Tensor | None,
    inv_freq: torch.Tensor | None,
    positions: torch.Tensor | None,
    eps: float,
    interleaved: bool,
    amplitude: float,
    dq_out: torch.Tensor,
    dk_out: torch.Tensor,
    dq: torch.Tensor,
    dk: torch.Tensor,
    dq_weight: torch.Tensor | None,
    dk_weight: torch.Tensor | None,
) -> None:
    return None


_rotary_bwd_inplace = torch.library.custom_op(
    "causal_conv1d_amd::_rotary_bwd_inplace",
    mutates_args=("dq", "dk", "dq_weight", "dk_weight"),
)(_rotary_bwd_impl)
_rotary_bwd_inplace.register_fake(_rotary_bwd_fake)


class _HeadNormRotaryFn(torch.autograd.Function):
    """On (batch, seqlen, heads, dim). Saves q and k where they are normed: a rotation needs no more than its angles."""

    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, inv_freq, positions, eps, interleaved, amplitude):
        q_out, k_out = _flat(q), _flat(k)
        torch.ops.causal_conv1d_amd._rotary_fwd_inplace(q, k, q_weight, k_weight, inv_freq, positions, eps,
                                                        interleaved, amplitude, q_out, k_out)
        ctx.save_for_backward(None if q_weight is None else q, None if k_weight is None else k, q_weight, k_weight,
                              inv_freq, positions)
        ctx.options = eps, interleaved, amplitude
        return q_out, k_out

    @staticmethod
    def backward(ctx, dq_out, dk_out):
        q, k, q_weight, k_weight, inv_freq, positions = ctx.saved_tensors
        dq, dk, dq_weight, dk_weight = (_flat(t) for t in (dq_out, dk_out, q_weight, k_weight))
        torch.ops.causal_conv1d_amd._rotary_bwd_inplace(q, k, q_weight, k_weight, inv_freq, positions, *ctx.options,
                                                        dq_out, dk_out, dq, dk, dq_weight, dk_weight)
        return dq, dk, dq_weight, dk_weight, None, None, None, None, None


def _check_float32(name: str, t: torch.Tensor | None, q: torch.Tensor, shape: tuple) -> torch.Tensor | None:
    if t is None:
        return None
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} shape {tuple(t.shape)} != expected {shape}")
    if t.dtype != torch.float32:
        raise NotImplementedError(f"{name}.dtype must be torch.float32 (got {t.dtype})")
    if t.device != q.device:
        raise NotImplementedError(f"{name}.device ({t.device}) must match q.device ({q.device})")
    return t.contiguous()


def head_norm_rotary_fn(
    q: torch.Tensor,
    k: torch.Tensor,
    q_weight: torch.Tensor | None = None,
    k_weight: torch.Tensor | None = None,
    inv_freq: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    eps: float = 1e-6,
    interleaved: bool = False,
    amplitude: float = 1.0,
) -> tuple[torch.Tensor, torch.Tensor]:
    """
    q: (batch, seqlen, q_heads, dim), or (tokens, q_heads, dim) as in a decode step; k: the same with k_heads.
        fp16 / bf16 / fp32, dim in 1..256, any strides (values of a head next to each other are fast)
    q_weight, k_weight: (dim,) fp32, the weight of the root mean square norm of each head; None: no norm
    inv_freq: (rotated / 2,) fp32, the angle of a pair per position; rotated <= dim, the rest of a head is not turned.
        None: no rotation. Not differentiated. ``rotary_frequencies`` gives it
    positions: (batch, seqlen) or (tokens,), int32 or int64; None: 0 .. seqlen - 1 in every row (not for single tokens)
    interleaved: pairs are values 2 i and 2 i + 1, instead of i and i + rotated / 2
    amplitude: on the rotated values

    Returns (q, k) so treated, contiguous. Gradients reach q, k and the weights.
    """
    if getattr(q, "is_cuda", False) and not torch.compiler.is_compiling():
        # an ordinary call, checked, recorded and launched in native code
        r = _host.native().head_norm_rotary(q, k, q_weight, k_weight, inv_freq, positions, eps, interleaved, amplitude)
        if r is not NotImplemented:
            return r
    if q.dtype not in _DTYPE_CODE:
        raise NotImplementedError(f"unsupported dtype {q.dtype}; only fp16/bf16/fp32 are supported")
    if q.dim() not in (3, 4) or k.dim() != q.dim() or k.shape[:-2] != q.shape[:-2] or k.shape[-1] != q.shape[-1]:
        raise ValueError(
            f"expected q (batch, seqlen, q_heads, dim) or (tokens, q_heads, dim) and k beside it; "
            f"got {tuple(q.shape)}, {tuple(k.shape)}"
        )
    if k.dtype != q.dtype or k.device != q.device:
        raise NotImplementedError(f"k ({k.dtype} on {k.device}) must match q ({q.dtype} on {q.device})")
    dim = q.shape[-1]
    if dim < 1 or dim > MAX_ROTARY_DIM:
        raise NotImplementedError(f"dim must be in 1..{MAX_ROTARY_DIM} (got {dim})")
    q_weight = _check_float32("q_weight", q_weight, q, (dim,))
    k_weight = _check_float32("k_weight", k_weight, q, (dim,))
    if inv_freq is not None:
        if inv_freq.dim() != 1 or 2 * inv_freq.shape[0] > dim:
            raise ValueError(f"inv_freq shape {tuple(inv_freq.shape)}: expected (rotated / 2,) with rotated <= {dim}")
        inv_freq = _check_float32("inv_freq", inv_freq.detach(), q, tuple(inv_freq.shape))
        if positions is None and q.dim() == 3:
            raise ValueError("single tokens need positions")
    if positions is not None:
        if positions.shape != q.shape[:-2]:
            raise ValueError(f"positions shape {tuple(positions.shape)} != expected {tuple(q.shape[:-2])}")
        if positions.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"positions.dtype must be int32 or int64 (got {positions.dtype})")
        if positions.device != q.device:
            raise ValueError(f"positions.device ({positions.device}) must match q.device ({q.device})")
    single = q.dim() == 3
    if single:
        q, k = q.unsqueeze(1), k.unsqueeze(1)
        positions = None if positions is None else positions.unsqueeze(1)
    a, b = _HeadNormRotaryFn.apply(q, k, q_weight, k_weight, inv_freq, positions, float(eps), bool(interleaved),
                                   float(amplitude))
    return (a.squeeze(1), b.squeeze(1)) if single else (a, b)


def rotary_frequencies(
    rotated: int,
    base: float = 10000.0,
    scaling: str = "none",
    factor: float = 1.0,
    trained_length: int = 4096,
    fast_turns: float = 32.0,
    slow_turns: float = 1.0,
    device: torch.device | str | None = None,
) -> tuple[torch.Tensor, float]:
    """The ``inv_freq`` and ``amplitude`` of ``head_norm_rotary_fn``: frequencies base ** (-2 i / rotated).

    scaling, for contexts ``factor`` times as long as the ``trained_length``:
        "none"
        "linear": every frequency divided by the factor (positions moved together)
        "base": the base raised so that the slowest frequency is divided by the factor and the fastest stays
        "ramp": frequencies that turn more than ``fast_turns`` times over the trained length stay, those that turn less
            than ``slow_turns`` times are divided, in between by a linear ramp; amplitude 0.1 ln(factor) + 1
    """
    if rotated < 2 or rotated % 2 != 0:
        raise ValueError(f"rotated must be even and positive (got {rotated})")
    if not base > 0.0 or not factor >= 1.0:
        raise ValueError(f"expected base > 0 and factor >= 1 (got {base}, {factor})")
    if scaling not in ("none", "linear", "base", "ramp"):
        raise ValueError(f'scaling must be "none", "linear", "base" or "ramp" (got {scaling!r})')
    if scaling == "base" and rotated > 2:
        base *= factor ** (rotated / (rotated - 2))
    f = base ** (-torch.arange(0, rotated, 2, dtype=torch.float64) / rotated)
    amplitude = 1.0
    if scaling == "linear":
        f = f / factor
    if scaling == "ramp":
        if not fast_turns > slow_turns:
            raise ValueError(f"fast_turns ({fast_turns}) must be more than slow_turns ({slow_turns})")
        turns = trained_length * f / (2.0 * math.pi)
        keep = ((turns - slow_turns) / (fast_turns - slow_turns)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
        amplitude = 0.1 * math.log(factor) + 1.0
    return f.to(torch.float32).to(device), amplitude
