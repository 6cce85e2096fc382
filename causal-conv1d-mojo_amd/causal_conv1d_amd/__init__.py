"""Depthwise causal conv1d for AMD Instinct MI355X (gfx950).

Drop-in for the public API of ``causal_conv1d_mojo``
(``src/causal_conv1d_mojo/__init__.py:39-60``): the same six names with the
same signatures. ``causal_conv1d_fn`` (forward + autograd backward),
``causal_conv1d_update`` (decode) and ``causal_conv1d_varlen_states`` run
hand-written HIP kernels from ``_lib/libcc1d_amd.so`` through its C ABI
(``include/cc1d.h``) on the current HIP stream; they accept ROCm device
tensors only and raise ``NotImplementedError`` for any other device.
``causal_conv1d_ref`` / ``causal_conv1d_update_ref`` are plain-torch
formulations kept for API parity.

What a state space layer runs around the convolution comes with it, in the
same manner: ``ssm_scan_fn`` (the selective scan over prompts, forward +
autograd backward), ``ssm_scan_update`` (its decode step) and ``add_norm_fn``
(residual add and layer / rms norm, forward + autograd backward), with
plain-torch formulations ``ssm_scan_ref``, ``ssm_scan_update_ref`` and
``add_norm_ref``. So does the mixer whose state is a matrix for each head:
``linear_attn_fn`` (linear attention with a decay for each head over prompts,
forward + autograd backward), ``linear_attn_update`` (its decode step) and
``head_norm_rotary_fn`` (norm of each query and key head and rotation by
position, forward + autograd backward; ``rotary_frequencies`` gives the
frequencies), with ``linear_attn_ref``, ``linear_attn_update_ref`` and
``head_norm_rotary_ref``.
"""

from __future__ import annotations

from causal_conv1d_amd._attn import linear_attn_fn
from causal_conv1d_amd._attn_update import linear_attn_update
from causal_conv1d_amd._fn import causal_conv1d_fn
from causal_conv1d_amd._norm import add_norm_fn
from causal_conv1d_amd._rotary import head_norm_rotary_fn, rotary_frequencies
from causal_conv1d_amd._scan import ssm_scan_fn
from causal_conv1d_amd._scan_update import ssm_scan_update
from causal_conv1d_amd._update import causal_conv1d_update
from causal_conv1d_amd.causal_conv1d_varlen import (
    causal_conv1d_varlen_states,
    causal_conv1d_varlen_states_ref,
)
from causal_conv1d_amd.reference import causal_conv1d_ref, causal_conv1d_update_ref
from causal_conv1d_amd.reference_attn import head_norm_rotary_ref, linear_attn_ref, linear_attn_update_ref
from causal_conv1d_amd.reference_ssm import add_norm_ref, ssm_scan_ref, ssm_scan_update_ref

__version__ = "1.6.1"

__all__ = [
    "add_norm_fn",
    "add_norm_ref",
    "causal_conv1d_fn",
    "causal_conv1d_ref",
    "causal_conv1d_update",
    "causal_conv1d_update_ref",
    "causal_conv1d_varlen_states",
    "causal_conv1d_varlen_states_ref",
    "head_norm_rotary_fn",
    "head_norm_rotary_ref",
    "linear_attn_fn",
    "linear_attn_ref",
    "linear_attn_update",
    "linear_attn_update_ref",
    "rotary_frequencies",
    "ssm_scan_fn",
    "ssm_scan_ref",
    "ssm_scan_update",
    "ssm_scan_update_ref",
]
