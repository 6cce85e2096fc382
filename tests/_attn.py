"""Linear attention's and the rotation's definitions in float64, with the magnitude of every sum, for the tests of
``linear_attn_fn``, ``linear_attn_update`` and ``head_norm_rotary_fn``.

Tolerance of a result (written once, used by every comparison):

    |got - exact| <= u_T |exact| + (P_T + (64 + 4 sqrt(L)) 2**-24) S

u_T is the rounding of one value to the result's type (2**-8 bf16, 2**-11 fp16, 2**-24 fp32), S the same formula over
the absolute values of its terms, L the number of positions: each fp32 operation behind a term adds up to 2**-24 of it,
a few dozen of them at most, and the roundings of L positions of a recurrence or a sum add as independent ones do (four
standard deviations). P_T is what operands split into bf16 planes leave out where a 16-bit result follows: a value is
held in two planes to 2**-18 of it (twice half a step of 2**-8), a product leaves out the one pair of second planes, at
most 2**-18 as well, and a term goes through two such products of two operands each: 8 * 2**-18 = 2**-15 at most. In
fp32, and for the states, three planes hold a value to 2**-27 and pairs below 2**-26 are left out, a few 2**-24 in all,
within the 64 above.
"""

from __future__ import annotations

import math

import torch

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def close(got, exact, scale, length, name="", extra=0.0):
    """``extra``: what the definition itself is uncertain by."""
    e, g, s = exact.double().cpu(), got.detach().double().cpu(), scale.double().cpu()
    assert g.shape == e.shape, f"{name}: shape {tuple(g.shape)} != {tuple(e.shape)}"
    left = 0.0 if got.dtype == torch.float32 else 2.0**-15
    bound = UNIT[got.dtype] * e.abs() + (left + (64.0 + 4.0 * math.sqrt(length)) * 2.0**-24) * s + extra + 1e-30
    if got.dtype == torch.float16:
        bound = bound + 2.0**-25  # subnormal spacing
    bad = ~((g - e).abs() <= bound)
    if bad.any():
        at = bad.nonzero()[0].tolist()
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} beyond the bound; at {at}: "
                             f"{g[tuple(at)].item()} against {e[tuple(at)].item()}, bound {bound[tuple(at)].item()}, "
                             f"worst {((g - e).abs() / bound).nan_to_num(math.inf).max().item()} of it")


def attn64(q, k, v, g, scale, init=None, dout=None, dfinal=None, mag=False):
    """out, final and (with dout or dfinal) every gradient, in float64, position by position; ``mag``: the sums' magnitudes."""
    f = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    m = (lambda t: None if t is None else t.abs()) if mag else (lambda t: t)
    q, k, v, init, dout, dfinal = (m(f(t)) for t in (q, k, v, init, dout, dfinal))
    a = torch.exp(f(g))
    scale = abs(scale) if mag else scale
    B, L, K, dk = q.shape
    H, dv = v.shape[2:]
    q, k = (t.repeat_interleave(H // K, 2) for t in (q, k))
    S = torch.zeros(B, H, dk, dv, dtype=torch.float64) if init is None else init
    states, out = [S], torch.zeros_like(v)
    for t in range(L):
        S = a[:, t, :, None, None] * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        states.append(S)
        out[:, t] = scale * (q[:, t, :, :, None] * S).sum(2)
    got = {"out": out, "final": S}
    if dout is None and dfinal is None:
        return got
    dout = torch.zeros_like(v) if dout is None else dout
    G = torch.zeros_like(S) if dfinal is None else dfinal
    dq, dkey, dval, dg = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros(B, L, H, dtype=torch.float64)
    over = (G * S).sum((-1, -2))  # the magnitude of the sums that dg is formed by
    for t in reversed(range(L)):
        G = G + scale * q[:, t, :, :, None] * dout[:, t, :, None, :]
        dq[:, t] = scale * (states[t + 1] * dout[:, t, :, None, :]).sum(-1)
        dkey[:, t] = (G * v[:, t, :, None, :]).sum(-1)
        dval[:, t] = (G * k[:, t, :, :, None]).sum(-2)
        if mag:
            over = over + (q[:, t] * dq[:, t]).sum(-1) + (k[:, t] * dkey[:, t]).sum(-1)
            dg[:, t] = over
        else:
            dg[:, t] = a[:, t] * (G * states[t]).sum((-1, -2))
        G = a[:, t, :, None, None] * G
    each = (B, L, K, H // K, dk)
    got.update(dq=dq.reshape(each).sum(3), dk=dkey.reshape(each).sum(3), dv=dval, dg=dg, dinit=G)
    return got


def rotary64(q, k, wq=None, wk=None, freq=None, pos=None, eps=1e-6, interleaved=False, amplitude=1.0, dq=None, dk=None):
    """(values, magnitudes) of q, k and (with dq) the gradients."""
    f = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    q, k, wq, wk, freq, dq, dk = map(f, (q, k, wq, wk, freq, dq, dk))
    if freq is not None and freq.numel():
        pos = torch.arange(q.shape[1]).double() if pos is None else pos.double().cpu()
        angle = (pos[..., None] * freq).unsqueeze(-2)
        cos, sin = torch.cos(angle) * amplitude, torch.sin(angle) * amplitude

    def turn(x, back=False, mag=False):
        if freq is None or not freq.numel():
            return x
        h = freq.numel()
        part = x[..., :2 * h]
        a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else (part[..., :h], part[..., h:])
        s = -sin if back else sin
        if mag:
            pair = a * abs(amplitude) + b * abs(amplitude), b * abs(amplitude) + a * abs(amplitude)
        else:
            pair = a * cos - b * s, b * cos + a * s
        part = torch.stack(pair, -1).flatten(-2) if interleaved else torch.cat(pair, -1)
        return torch.cat((part, x[..., 2 * h:]), -1)

    val, mag = {}, {}
    for name, x, w, d in (("q", q, wq, dq), ("k", k, wk, dk)):
        rstd = 1.0 if w is None else 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
        ww = 1.0 if w is None else w
        val[name], mag[name] = turn(x * rstd * ww), turn((x * rstd * ww).abs(), mag=True)
        if d is None:
            continue
        e, em = turn(d, True), turn(d.abs(), mag=True)
        if w is None:
            val["d" + name], mag["d" + name] = e, em
            continue
        xh = x * rstd
        lead = tuple(range(x.dim() - 1))
        val["dw" + name], mag["dw" + name] = (e * xh).sum(lead), (em * xh.abs()).sum(lead)
        e, em = e * w, em * w.abs()
        val["d" + name] = rstd * (e - xh * (e * xh).mean(-1, keepdim=True))
        mag["d" + name] = rstd * (em + xh.abs() * (em * xh.abs()).mean(-1, keepdim=True))
    return val, mag
