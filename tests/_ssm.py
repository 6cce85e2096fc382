"""The scan's and the norm's definitions in float64, with the magnitude of every
sum, for the tests of ``ssm_scan_fn``, ``ssm_scan_update`` and ``add_norm_fn``.

Tolerance of a result (written once, used by every comparison):

    |got - exact| <= u_T |exact| + (64 + 4 sqrt(L)) 2**-24 S

u_T is the rounding of one value to the result's type (2**-8 bf16, 2**-11 fp16,
2**-24 fp32), S the same formula over the absolute values of its terms, and L
the number of positions: each fp32 operation behind a term adds up to 2**-24 of
it, a few dozen operations of one position at most, and the roundings of L
positions of a recurrence or a sum add as independent ones do (four standard
deviations). What multiplies a state goes through exp(dt A), whose argument's
rounding is damped by the decay itself (x exp(-x) <= 0.37).
"""

from __future__ import annotations

import math

import torch

UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}


def close(got, exact, scale, length, name=""):
    e = exact.double().cpu()
    g = got.detach().double().cpu()
    assert g.shape == e.shape, f"{name}: shape {tuple(g.shape)} != {tuple(e.shape)}"
    bound = UNIT[got.dtype] * e.abs() + (64.0 + 4.0 * math.sqrt(length)) * 2.0**-24 * scale.double().cpu() + 1e-30
    if got.dtype == torch.float16:
        bound = bound + 2.0**-25  # subnormal spacing
    bad = ~((g - e).abs() <= bound)
    if bad.any():
        at = bad.nonzero()[0].tolist()
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} beyond the bound; at {at}: "
                             f"{g[tuple(at)].item()} against {e[tuple(at)].item()}, bound {bound[tuple(at)].item()}")


def softplus64(x):
    return torch.where(x > 40, x, torch.log1p(torch.exp(x.clamp(max=40.0))))


def scan64(u, delta, A, B, C, D=None, z=None, bias=None, softplus=False, ids=None, init=None, dout=None, dfinal=None,
           mag=False):
    """out, final and (with dout) every gradient of one batch, in float64; with ``mag`` the sums' magnitudes."""
    f = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    m = (lambda t: t.abs()) if mag else (lambda t: t)
    u, delta, A, B, C, D, z, bias, init, dout, dfinal = map(f, (u, delta, A, B, C, D, z, bias, init, dout, dfinal))
    ids = None if ids is None else ids.cpu()
    if B.dim() == 3:
        B, C = B[:, None], C[:, None]
    nb, dim, L = u.shape
    N, G = A.shape[1], B.shape[1]
    live = torch.ones(nb, L, dtype=torch.bool) if ids is None else ids >= 0
    cut = torch.zeros(nb, L, dtype=torch.bool)
    if ids is not None:
        cut[:, 1:] = ids[:, 1:] != ids[:, :-1]
        cut[:, :1] = True
    w = lambda t: torch.where(live[:, None], t, torch.zeros_like(t))  # noqa: E731
    u, delta = w(u), w(delta)
    z, dout = (None if t is None else w(t) for t in (z, dout))
    B, C = (torch.where(live[:, None, None], t, torch.zeros_like(t)) for t in (B, C))
    raw = delta + (0.0 if bias is None else bias[:, None])
    dt = w(softplus64(raw) if softplus else raw)
    Bd, Cd = (m(t.repeat_interleave(dim // G, 1)) for t in (B, C))
    a = torch.exp(dt[:, :, None] * A[:, :, None])
    uu, dtm, Am = m(u), m(dt), m(A)
    h = torch.zeros(nb, dim, N, dtype=torch.float64) if init is None else m(init)
    first, hs, ys = h, [], []
    for t in range(L):
        h = torch.where(cut[:, t, None, None], torch.zeros_like(h), h)
        h = a[..., t] * h + (dtm[..., t] * uu[..., t])[..., None] * Bd[..., t]
        hs.append(h)
        ys.append((h * Cd[..., t]).sum(-1))
    y = torch.stack(ys, -1) if ys else torch.zeros_like(u)
    if D is not None:
        y = y + m(D)[:, None] * uu
    sg = None if z is None else torch.sigmoid(z)
    got = {"out": w(y if z is None else y * m(z * sg)), "final": h}
    if dout is None:
        return got
    do = m(dout)
    dy = do
    if z is not None:
        got["dz"] = w(do * y * (sg * (1 + m(z) * (1 - sg))))
        dy = do * m(z * sg)
    carry = torch.zeros(nb, dim, N, dtype=torch.float64) if dfinal is None else m(dfinal)
    du, ddt = torch.zeros_like(u), torch.zeros_like(u)
    dB, dC = torch.zeros_like(Bd), torch.zeros_like(Cd)
    dA = torch.zeros_like(A)
    for t in reversed(range(L)):
        g = carry + dy[..., t, None] * Cd[..., t]
        dC[..., t] = dy[..., t, None] * hs[t]
        dB[..., t] = g * (dtm[..., t] * uu[..., t])[..., None]
        along = (g * Bd[..., t]).sum(-1)
        prior = torch.where(cut[:, t, None, None], torch.zeros_like(h), hs[t - 1] if t else first)
        x = g * a[..., t] * prior
        dA += (x * dtm[..., t, None]).sum(0)
        ddt[..., t] = along * uu[..., t] + (x * Am).sum(-1)
        du[..., t] = along * dtm[..., t] + (0.0 if D is None else dy[..., t] * m(D))
        carry = torch.where(cut[:, t, None, None], torch.zeros_like(g), g * a[..., t])
    slope = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    ddelta = w(ddt * slope)
    got.update(du=w(du), ddelta=ddelta, dA=dA, dB=dB.unflatten(1, (G, -1)).sum(2), dC=dC.unflatten(1, (G, -1)).sum(2),
               dD=(dy * uu).sum((0, 2)), dbias=ddelta.sum((0, 2)), dinit=carry)
    return got


def norm64(x, weight, bias=None, residual=None, eps=1e-5, rms=False, dy=None, dsum=None):
    """(values, magnitudes) of out, sum and (with dy) the gradients, rows in the last axis but one."""
    f = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    x, weight, bias, residual, dy, dsum = map(f, (x, weight, bias, residual, dy, dsum))
    r = x if residual is None else x + residual
    rm = x.abs() if residual is None else x.abs() + residual.abs()
    mean = torch.zeros_like(r[:, :1]) if rms else r.mean(1, keepdim=True)
    var = ((r - mean) ** 2).mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt(var + eps)
    xh = (r - mean) * rstd
    xm = (rm + (0.0 if rms else rm.mean(1, keepdim=True))) * rstd
    b = 0.0 if bias is None else bias
    val = {"out": xh * weight + b, "sum": r}
    mag = {"out": xm * weight.abs() + (0.0 if bias is None else bias.abs()), "sum": rm}
    if dy is None:
        return val, mag
    d, dm = dy * weight, (dy * weight).abs()
    along, alongm = (d * xh).mean(1, keepdim=True), (dm * xm).mean(1, keepdim=True)
    level, levelm = (0.0, 0.0) if rms else (d.mean(1, keepdim=True), dm.mean(1, keepdim=True))
    val["dx"] = rstd * (d - level - xh * along) + (0.0 if dsum is None else dsum)
    mag["dx"] = rstd * (dm + levelm + xm * alongm) + (0.0 if dsum is None else dsum.abs())
    val["dw"], mag["dw"] = (dy * xh).sum(0), (dy.abs() * xm).sum(0)
    val["db"], mag["db"] = dy.sum(0), dy.abs().sum(0)
    return val, mag
