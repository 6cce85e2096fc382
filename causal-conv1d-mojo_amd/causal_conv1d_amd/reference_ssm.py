"""Plain PyTorch formulations of the scan, its decode step and the norm
(``ssm_scan_ref``, ``ssm_scan_update_ref``, ``add_norm_ref``), for callers that
want to compare results: the recurrence position by position, on any device, in fp32 or
in the inputs' dtype where that is wider. Autograd runs through them. The
package's kernels never call them.
"""

from __future__ import annotations

import torch
import torch.nn.functional as F


def _wide(t: torch.Tensor | None, dtype: torch.dtype) -> torch.Tensor | None:
    return None if t is None else t.to(dtype)


def _groups_of(B: torch.Tensor, dim: int) -> torch.Tensor:
    return B.repeat_interleave(dim // B.shape[1], dim=1)


def ssm_scan_ref(u, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=False, seq_idx=None,
                 cu_seqlens=None, initial_states=None, return_final_states=False):
    """Arguments and results of ``ssm_scan_fn``."""
    if cu_seqlens is not None:
        ends = cu_seqlens.tolist()
        outs, states, covered = [], [], 0
        for i, (a, b) in enumerate(zip(ends, ends[1:])):
            part = [None if t is None else t[..., a:b] for t in (u, delta, B, C, z)]
            o, s = ssm_scan_ref(part[0], part[1], A, part[2], part[3], D, part[4], delta_bias, delta_softplus,
                                initial_states=None if initial_states is None else initial_states[i:i + 1],
                                return_final_states=True)
            outs += [u.new_zeros(1, u.shape[1], a - covered), o]
            states.append(s)
            covered = b
        out = torch.cat([*outs, u.new_zeros(1, u.shape[1], u.shape[2] - covered)], -1)
        return (out, torch.cat(states)) if return_final_states else out
    wide = torch.promote_types(u.dtype, torch.float32)
    batch, dim, seqlen = u.shape
    if B.dim() == 3:
        B, C = B.unsqueeze(1), C.unsqueeze(1)
    live = None if seq_idx is None else (seq_idx >= 0)[:, None]
    x, dt, Bw, Cw, zw = (_wide(t, wide) for t in (u, delta, B, C, z))
    if live is not None:  # padding may hold anything
        x, dt, zw = (None if t is None else torch.where(live, t, torch.zeros_like(t)) for t in (x, dt, zw))
        Bw, Cw = (torch.where(live[:, None], t, torch.zeros_like(t)) for t in (Bw, Cw))
    if delta_bias is not None:
        dt = dt + delta_bias.to(wide)[:, None]
    if delta_softplus:
        dt = F.softplus(dt, threshold=40.0)
    if live is not None:
        dt = torch.where(live, dt, torch.zeros_like(dt))
    Bw, Cw, A = _groups_of(Bw, dim), _groups_of(Cw, dim), A.to(wide)
    h = _wide(initial_states, wide)
    if h is None:
        h = torch.zeros(batch, dim, A.shape[1], dtype=wide, device=u.device)
    ys = []
    for t in range(seqlen):
        if seq_idx is not None and t > 0:
            h = torch.where((seq_idx[:, t] != seq_idx[:, t - 1])[:, None, None], torch.zeros_like(h), h)
        h = torch.exp(dt[:, :, t, None] * A) * h + (dt[:, :, t] * x[:, :, t])[..., None] * Bw[:, :, :, t]
        ys.append((h * Cw[:, :, :, t]).sum(-1))
    y = torch.stack(ys, -1) if ys else torch.zeros_like(x)
    if D is not None:
        y = y + D.to(wide)[:, None] * x
    if z is not None:
        y = y * F.silu(zw)
    if live is not None:
        y = torch.where(live, y, torch.zeros_like(y))
    out = y.to(u.dtype)
    return (out, h) if return_final_states else out


def ssm_scan_update_ref(u, ssm_state, delta, A, B, C, D=None, z=None, delta_bias=None, delta_softplus=False,
                        ssm_state_indices=None):
    """Arguments and result of ``ssm_scan_update``; ``ssm_state`` is updated in place."""
    one = u.dim() == 2
    if one:
        u, delta, B, C = (t.unsqueeze(-1) for t in (u, delta, B, C))
        z = None if z is None else z.unsqueeze(-1)
    rows = torch.arange(u.shape[0], device=u.device) if ssm_state_indices is None else ssm_state_indices.long()
    live = (rows >= 0) & (rows < ssm_state.shape[0])
    out = torch.zeros_like(u)
    pick = lambda t: None if t is None else t[live]  # noqa: E731
    out[live], ssm_state[rows[live]] = ssm_scan_ref(
        pick(u), pick(delta), A, pick(B), pick(C), D, pick(z), delta_bias, delta_softplus,
        initial_states=ssm_state[rows[live]], return_final_states=True)
    return out.squeeze(-1) if one else out


def add_norm_ref(x, weight, bias=None, residual=None, eps=1e-5, rms=False, return_residual=False):
    """Arguments and results of ``add_norm_fn``."""
    wide = torch.promote_types(x.dtype, torch.float32)
    r = x.to(wide) if residual is None else x.to(wide) + residual.to(wide)
    off = r if rms else r - r.mean(-1, keepdim=True)
    y = off * torch.rsqrt((off * off).mean(-1, keepdim=True) + eps) * weight.to(wide)
    if bias is not None:
        y = y + bias.to(wide)
    y = y.to(x.dtype)
    if not return_residual:
        return y
    return y, x if residual is None else r.to(residual.dtype)
