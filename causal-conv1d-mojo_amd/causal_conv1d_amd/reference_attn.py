"""Plain PyTorch formulations of linear attention with a decay for each head, its
decode step, and the head norm with rotation (``linear_attn_ref``,
``linear_attn_update_ref``, ``head_norm_rotary_ref``), for callers that want to
compare results: the recurrence position by position, on any device, in fp32 or
in the inputs' dtype where that is wider. Autograd runs through them. The
package's kernels never call them.
"""

from __future__ import annotations

import torch


def linear_attn_ref(q, k, v, g, scale=None, cu_seqlens=None, initial_states=None, return_final_states=False):
    """Arguments and results of ``linear_attn_fn``."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    if cu_seqlens is not None:
        ends = cu_seqlens.tolist()
        outs, states, covered = [], [], 0
        for i, (a, b) in enumerate(zip(ends, ends[1:])):
            o, s = linear_attn_ref(*(t[:, a:b] for t in (q, k, v, g)), scale,
                                   initial_states=None if initial_states is None else initial_states[i:i + 1],
                                   return_final_states=True)
            outs += [v.new_zeros(1, a - covered, *v.shape[2:]), o]
            states.append(s)
            covered = b
        out = torch.cat([*outs, v.new_zeros(1, v.shape[1] - covered, *v.shape[2:])], 1)
        if not return_final_states:
            return out
        empty = torch.zeros(0, v.shape[2], q.shape[3], v.shape[3], dtype=torch.float32, device=v.device)
        return out, torch.cat(states) if states else empty
    wide = torch.promote_types(q.dtype, torch.float32)
    each = v.shape[2] // q.shape[2]
    qw, kw = (t.to(wide).repeat_interleave(each, 2) for t in (q, k))
    vw, decay = v.to(wide), torch.exp(g.to(wide))
    if initial_states is None:
        S = torch.zeros(v.shape[0], v.shape[2], q.shape[3], v.shape[3], dtype=wide, device=v.device)
    else:
        S = initial_states.to(wide)
    outs = []
    for t in range(v.shape[1]):
        S = decay[:, t, :, None, None] * S + kw[:, t, :, :, None] * vw[:, t, :, None, :]
        outs.append(scale * (qw[:, t, :, :, None] * S).sum(-2))
    out = (torch.stack(outs, 1) if outs else vw).to(v.dtype)
    return (out, S) if return_final_states else out


def linear_attn_update_ref(q, attn_state, k, v, g, scale=None, attn_state_indices=None):
    """Arguments and result of ``linear_attn_update``; ``attn_state`` is updated in place."""
    one = q.dim() == 3
    if one:
        q, k, v, g = (t.unsqueeze(1) for t in (q, k, v, g))
    rows = torch.arange(q.shape[0], device=q.device) if attn_state_indices is None else attn_state_indices.long()
    live = (rows >= 0) & (rows < attn_state.shape[0])
    out = torch.zeros(v.shape, dtype=v.dtype, device=v.device)
    out[live], attn_state[rows[live]] = linear_attn_ref(
        q[live], k[live], v[live], g[live], scale, initial_states=attn_state[rows[live]], return_final_states=True)
    return out.squeeze(1) if one else out


def head_norm_rotary_ref(q, k, q_weight=None, k_weight=None, inv_freq=None, positions=None, eps=1e-6,
                         interleaved=False, amplitude=1.0):
    """Arguments and results of ``head_norm_rotary_fn``."""
    if inv_freq is not None:
        if positions is None:
            positions = torch.arange(q.shape[1], device=q.device)
        angle = positions.double()[..., None] * inv_freq.double()

    def one(x, weight):
        wide = torch.promote_types(x.dtype, torch.float32)
        y = x.to(wide)
        if weight is not None:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + eps) * weight.to(wide)
        if inv_freq is None:
            return y.to(x.dtype)
        half = inv_freq.shape[0]
        cos, sin = ((f(angle) * amplitude).to(wide).unsqueeze(-2) for f in (torch.cos, torch.sin))
        turned, rest = y[..., :2 * half], y[..., 2 * half:]
        a, b = turned.unflatten(-1, (half, 2)).unbind(-1) if interleaved else turned.unflatten(-1, (2, half)).unbind(-2)
        pair = a * cos - b * sin, b * cos + a * sin
        turned = torch.stack(pair, -1 if interleaved else -2).flatten(-2)
        return torch.cat((turned, rest), -1).to(x.dtype)

    return one(q, q_weight), one(k, k_weight)
