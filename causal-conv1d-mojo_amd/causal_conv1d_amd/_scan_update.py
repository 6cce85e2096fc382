"""``ssm_scan_update``: the selective state space scan for new tokens of a
decode batch, on a state pool updated in place (the scan's counterpart of
``causal_conv1d_update``). No autograd.
"""

from __future__ import annotations

import torch

from causal_conv1d_amd import _host
from causal_conv1d_amd._native import native_scan_update
from causal_conv1d_amd._scan import _check_int32, _check_like, _check_parameters


def ssm_scan_update(
    u: torch.Tensor,
    ssm_state: torch.Tensor,
    delta: torch.Tensor,
    A: torch.Tensor,
    B: torch.Tensor,
    C: torch.Tensor,
    D: torch.Tensor | None = None,
    z: torch.Tensor | None = None,
    delta_bias: torch.Tensor | None = None,
    delta_softplus: bool = False,
    ssm_state_indices: torch.Tensor | None = None,
) -> torch.Tensor:
    """
    u, delta, z: (batch, dim) or (batch, dim, seqlen) -- the new tokens, fp16 / bf16 / fp32
    ssm_state: (batch_or_pool_size, dim, dstate) fp32; mutated in place
    A: (dim, dstate) fp32; D, delta_bias: (dim,) fp32
    B, C: (batch, [groups,] dstate) for u (batch, dim), (batch, [groups,] dstate, seqlen) otherwise, dtype of u
    ssm_state_indices: (batch,) int32 or None -- state row per batch entry, distinct; < 0 marks padding

    Returns: out, same shape as u (0 for padding, whose state rows stay as they are).
    """
    if getattr(u, "is_cuda", False) and not torch.compiler.is_compiling():
        # an ordinary call, checked and launched in native code
        out = _host.native().ssm_scan_update(u, ssm_state, delta, A, B, C, D, z, delta_bias, delta_softplus,
                                             ssm_state_indices)
        if out is not NotImplemented:
            return out
    if u.dim() not in (2, 3) or ssm_state.dim() != 3:
        raise ValueError(
            f"expected u (batch, dim[, seqlen]) and ssm_state (rows, dim, dstate); "
            f"got u {tuple(u.shape)}, ssm_state {tuple(ssm_state.shape)}"
        )
    batch, dim = u.shape[:2]
    dstate = _check_parameters(u, A, D, delta_bias, dim)
    _check_like("delta", delta, u, u.shape, u.dtype)
    _check_like("z", z, u, u.shape, u.dtype)
    if B.dim() not in (u.dim(), u.dim() + 1) or C.dim() != B.dim():
        raise ValueError(
            f"expected B and C of shape (batch, [groups,] dstate{', seqlen' if u.dim() == 3 else ''}); "
            f"got {tuple(B.shape)}, {tuple(C.shape)}"
        )
    if B.dim() == u.dim():
        B, C = B.unsqueeze(1), C.unsqueeze(1)
    groups = B.shape[1]
    if groups < 1 or dim % groups != 0:
        raise ValueError(f"dim ({dim}) must be a multiple of B's groups ({groups})")
    _check_like("B", B, u, (batch, groups, dstate, *u.shape[2:]), u.dtype)
    _check_like("C", C, u, (batch, groups, dstate, *u.shape[2:]), u.dtype)
    rows = batch if ssm_state_indices is None else ssm_state.shape[0]
    _check_like("ssm_state", ssm_state, u, (rows, dim, dstate), torch.float32)
    if ssm_state_indices is not None:
        ssm_state_indices = _check_int32("ssm_state_indices", ssm_state_indices, u, (batch,))

    with torch.no_grad():
        unsqueeze = u.dim() == 2
        if unsqueeze:
            u, delta, B, C = (t.unsqueeze(-1) for t in (u, delta, B, C))
            z = None if z is None else z.unsqueeze(-1)
        out = torch.empty_like(u)
        native_scan_update(u, ssm_state, delta, A, B, C, D, z, delta_bias, bool(delta_softplus), ssm_state_indices, out)
        return out.squeeze(-1) if unsqueeze else out
