"""Performance cases of linear attention with a decay for each head, and of what runs on its queries and keys.

Each case is one pass of what a program does with the public entry points:

* ``attn``   -- ``linear_attn_fn`` over prompts, without gradients or (``train``) with its autograd backward;
* ``step``   -- ``linear_attn_update`` with new tokens;
* ``rotary`` -- ``head_norm_rotary_fn``, without gradients or (``train``) with its autograd backward.

``own`` false runs the operators in their plain form (elementary torch operations in 32 bits, in 64 for sums of
log decays, for angles and for the long sums behind their gradient, rounded once at the end), true calls the framework.

``extra`` of an attention: ``prompts`` sequences packed into one row with cu_seqlens, going on from their states and
returning the new ones; ``packed`` the same packing without states; ``states`` one sequence a row with states.
"""

from __future__ import annotations

import functools
import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CHUNK = 64                                        # positions the plain form takes at once
ATTN_LARGEST = 4 * 2048 * 40 * 128 * 128          # state elements touched by the largest listed attention
ATTN_VALUES = 4 * 2048 * 40 * 128                 # values of its v
STEP_LARGEST = 128 * 40 * 128 * 128               # state elements of the largest listed step
ROTARY_LARGEST = 4 * 2048 * (40 + 40) * 128       # values of the largest listed rotation


@functools.lru_cache(maxsize=None)
def _cc():
    """The package, imported once as a program imports it."""
    pkg = str(Path(__file__).resolve().parent.parent / "causal-conv1d-mojo_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import causal_conv1d_amd

    return causal_conv1d_amd


def _attn(name, dtype, batch, seqlen, heads, key_heads, dk, dv, train=False, extra="none", seqs=1):
    return {"name": name, "op": "attn", "dtype": dtype, "batch": batch, "seqlen": seqlen, "heads": heads,
            "key_heads": key_heads, "dk": dk, "dv": dv, "train": train, "extra": extra, "seqs": seqs}


def _step(name, dtype, batch, heads, key_heads, dk, dv, tokens=1, rows=0, padded=0):
    return {"name": name, "op": "step", "dtype": dtype, "batch": batch, "heads": heads, "key_heads": key_heads,
            "dk": dk, "dv": dv, "tokens": tokens, "rows": rows, "padded": padded}


def _rotary(name, dtype, batch, seqlen, heads, key_heads, dim, rotated, norm=True, interleaved=False, scaling="none",
            reach=0, train=False):
    return {"name": name, "op": "rotary", "dtype": dtype, "batch": batch, "seqlen": seqlen, "heads": heads,
            "key_heads": key_heads, "dim": dim, "rotated": rotated, "norm": norm, "interleaved": interleaved,
            "scaling": scaling, "reach": reach, "train": train}


def listed():
    return [
        # one user's short prompt of any length: latency
        _attn("attn short prompt", "fp16", 1, 131, 16, 16, 64, 64, extra="states"),
        # eight prompts packed into one row, going on from their states
        _attn("attn prompts", "bf16", 1, 8192, 32, 32, 128, 128, extra="prompts", seqs=8),
        # a small layer's training step
        _attn("attn train small", "bf16", 2, 512, 12, 12, 64, 64, train=True),
        # a large layer's training step: 5120 channels in 40 heads
        _attn("attn train", "bf16", 4, 2048, 40, 40, 128, 128, train=True),
        # packed documents of no round length, heads that share their queries and keys in groups
        _attn("attn train groups", "fp16", 1, 4 * 2041, 32, 8, 128, 64, train=True, extra="packed", seqs=13),
        # 32 bits, odd head sizes, handed on from chunk to chunk with the states' gradients
        _attn("attn train fp32", "fp32", 1, 2048, 16, 16, 80, 72, train=True, extra="states"),
        # one user's next token: nothing but latency
        _step("step one", "bf16", 1, 24, 24, 64, 64),
        # a serving batch whose sequences live at random rows of a state pool, some slots unused
        _step("step pool", "bf16", 128, 40, 40, 128, 128, rows=256, padded=6),
        # four tokens a call on shared queries and keys
        _step("step burst", "fp16", 31, 64, 8, 128, 64, tokens=4),
        # a serving batch's next tokens far into long contexts, frequencies scaled for them
        _rotary("rotary step", "bf16", 64, 1, 40, 8, 128, 128, scaling="ramp", reach=1000000),
        # a large layer's queries and keys in training
        _rotary("rotary train", "bf16", 4, 2048, 40, 40, 128, 128, train=True),
        # part of an odd head, interleaved pairs, in 32 bits
        _rotary("rotary train odd", "fp32", 1, 4099, 7, 1, 80, 36, interleaved=True, scaling="linear", train=True),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], even over its logarithm."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _heads(rng, most):
    """Heads, and key heads that divide them."""
    key = _spread(rng, 1, most)
    each = rng.choice((1, 1, 2, 4, 8))
    return (key * each, key) if key * each <= most else (key, key)


def _head_dim(rng):
    return rng.choice((64, 64, 128, 128, 32, 96, rng.randint(1, 128)))


def draw(rng):
    op = rng.choice(("attn", "attn", "step", "rotary"))
    dtype = rng.choice(("bf16", "bf16", "fp16", "fp32"))
    if op == "rotary":
        heads, key_heads = _heads(rng, 64)
        dim = rng.choice((64, 128, 128, 256, 80, 2 * rng.randint(1, 128), rng.randint(3, 256)))
        rotated = rng.choice((dim // 2 * 2, dim // 2 * 2, 2 * rng.randint(1, dim // 2), 0))
        batch, seqlen = _spread(rng, 1, 64), _spread(rng, 1, 8192)
        while batch * seqlen * (heads + key_heads) * dim > ROTARY_LARGEST:
            batch, seqlen = (batch + 1) // 2, seqlen if batch > 1 else (seqlen + 1) // 2
        c = _rotary("", dtype, batch, seqlen, heads, key_heads, dim, rotated, rotated == 0 or rng.random() < 0.7,
                    rng.random() < 0.4, rng.choice(("none", "linear", "ramp")),
                    rng.choice((0, _spread(rng, 1000, 1000000))), rng.random() < 0.6)
        del c["name"]
        return c
    heads, key_heads = _heads(rng, 80)
    dk, dv = _head_dim(rng), _head_dim(rng)
    if op == "step":
        batch, tokens = _spread(rng, 1, 512), rng.choice((1, 1, 1, rng.randint(2, 8)))
        while batch * heads * dk * dv > STEP_LARGEST:
            batch = (batch + 1) // 2
        rows, padded = 0, 0
        if rng.random() < 0.5:
            rows, padded = batch + _spread(rng, 1, 128), rng.choice((0, 0, batch // 8))
        c = _step("", dtype, batch, heads, key_heads, dk, dv, tokens, rows, padded)
    else:
        batch, seqlen = _spread(rng, 1, 16), _spread(rng, 4, 16384)
        if rng.random() < 0.5:
            seqlen = max(1, seqlen // 64) * 64
        train = rng.random() < 0.6
        while batch * seqlen * heads * dk * dv > ATTN_LARGEST or batch * seqlen * heads * max(dk, dv) > ATTN_VALUES:
            batch, seqlen = (batch + 1) // 2, seqlen if batch > 1 else (seqlen + 1) // 2
        extra = rng.choice(("none", "packed", "states", "prompts"))
        seqs = 1
        if extra in ("packed", "prompts"):
            batch, seqlen = 1, min(16384, batch * seqlen)
            seqs = max(1, min(seqlen // 4, rng.randint(1, 16)))
        c = _attn("", dtype, batch, seqlen, heads, key_heads, dk, dv, train, extra, seqs)
    del c["name"]
    return c


# ---------------------------------------------------------------- inputs


def _normal(gen, dtype, *shape):
    return torch.randn(*shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype)


def _decays(gen, dtype, heads, *lead):
    """Log decays of heads that remember from about one to about a thousand positions, moved by the inputs."""
    rate = torch.logspace(-3.0, 0.0, heads, device=DEVICE)
    x = torch.randn(*lead, heads, generator=gen, device=DEVICE) + 0.5
    return (-rate * torch.log1p(torch.exp(x))).to(dtype)


def _bounds(c, seed):
    """Boundaries 0 .. seqlen of seqs sequences of random lengths."""
    cpu = torch.Generator().manual_seed(seed)
    L, n = c["seqlen"], c["seqs"]
    inner = torch.randperm(L - 1, generator=cpu)[:n - 1].sort().values + 1 if n > 1 else \
        torch.empty(0, dtype=torch.int64)
    return torch.cat((torch.tensor([0]), inner, torch.tensor([L])))


def _chunks(bounds):
    """The plain form's plan: for each chunk the positions it holds (-1: none) and its sequence, and for each
    sequence its first and last chunk."""
    lengths = bounds[1:] - bounds[:-1]
    count = (lengths + CHUNK - 1) // CHUNK
    last = count.cumsum(0) - 1
    first = last - count + 1
    seq = torch.repeat_interleave(torch.arange(len(count)), count)
    at = (torch.arange(len(seq)) - first[seq])[:, None] * CHUNK + torch.arange(CHUNK)
    at = torch.where(at < lengths[seq][:, None], at + bounds[:-1][seq][:, None], -1)
    return {k: v.to(DEVICE) for k, v in (("at", at), ("seq", seq), ("first", first), ("last", last))}


def _prepare_attn(c, seed, gen):
    dtype = DTYPES[c["dtype"]]
    B, L, H, K, dk, dv = c["batch"], c["seqlen"], c["heads"], c["key_heads"], c["dk"], c["dv"]
    s = {"case": c, "q": _normal(gen, dtype, B, L, K, dk), "k": _normal(gen, dtype, B, L, K, dk),
         "v": _normal(gen, dtype, B, L, H, dv), "g": _decays(gen, dtype, H, B, L), "cu": None, "initial": None}
    packed = c["extra"] in ("packed", "prompts")
    bounds = _bounds(c, seed) if packed else torch.arange(B + 1) * L
    s["plan"], s["bounds"] = _chunks(bounds), bounds.tolist()
    if packed:
        s["cu"] = bounds.to(torch.int32).to(DEVICE)
    if c["extra"] in ("states", "prompts"):
        s["initial"] = _normal(gen, torch.float32, len(bounds) - 1, H, dk, dv)
    if c["train"]:
        s["dout"] = _normal(gen, dtype, B, L, H, dv)
        s["dfinal"] = _normal(gen, torch.float32, *s["initial"].shape) if s["initial"] is not None else None
        for name in ("q", "k", "v", "g", "initial"):
            if s[name] is not None:
                s[name].requires_grad_()
    return s


def _prepare_step(c, seed, gen):
    dtype = DTYPES[c["dtype"]]
    B, T, H, K, dk, dv = c["batch"], c["tokens"], c["heads"], c["key_heads"], c["dk"], c["dv"]
    lead = (B,) if T == 1 else (B, T)
    s = {"case": c, "q": _normal(gen, dtype, *lead, K, dk), "k": _normal(gen, dtype, *lead, K, dk),
         "v": _normal(gen, dtype, *lead, H, dv), "g": _decays(gen, dtype, H, *lead),
         "state": _normal(gen, torch.float32, c["rows"] or B, H, dk, dv), "indices": None}
    if c["rows"]:
        indices = torch.randperm(c["rows"], generator=torch.Generator().manual_seed(seed))[:B].to(torch.int32)
        if c["padded"]:
            indices[-c["padded"]:] = -1  # a captured batch size is filled up with unused slots
        s["indices"] = indices.to(DEVICE)
    return s


def _frequencies(c):
    """Frequencies base ** (-2 i / rotated), as they are, all stretched, or stretched where a turn is longer than
    the lengths that were trained on; and what the rotated values are multiplied with."""
    R = c["rotated"]
    f = 10000.0 ** (-torch.arange(0, R, 2, dtype=torch.float64) / max(R, 1))
    amplitude = 1.0
    if c["scaling"] == "linear":
        f = f / 4.0
    if c["scaling"] == "ramp":
        turns = 4096.0 * f / (2.0 * math.pi)  # over the trained length
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)
        f, amplitude = f * keep + f / 16.0 * (1.0 - keep), 0.1 * math.log(16.0) + 1.0
    return f.to(torch.float32).to(DEVICE), amplitude


def _prepare_rotary(c, gen):
    dtype = DTYPES[c["dtype"]]
    B, L, H, K, D = c["batch"], c["seqlen"], c["heads"], c["key_heads"], c["dim"]
    s = {"case": c, "q": _normal(gen, dtype, B, L, H, D), "k": _normal(gen, dtype, B, L, K, D), "wq": None, "wk": None,
         "freq": None, "amplitude": 1.0}
    if c["norm"]:
        s["wq"], s["wk"] = (1.0 + 0.1 * torch.randn(D, generator=gen, device=DEVICE) for _ in range(2))
    if c["rotated"]:
        s["freq"], s["amplitude"] = _frequencies(c)
    # every row goes on from a place of its own
    start = torch.randint(0, c["reach"] + 1, (B, 1), generator=gen, device=DEVICE)
    s["positions"] = start + torch.arange(L, device=DEVICE)
    if c["train"]:
        s["dq"], s["dk"] = _normal(gen, dtype, B, L, H, D), _normal(gen, dtype, B, L, K, D)
        for name in ("q", "k", "wq", "wk"):
            if s[name] is not None:
                s[name].requires_grad_()
    return s


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["op"] == "attn":
        return _prepare_attn(case, seed, gen)
    if case["op"] == "step":
        return _prepare_step(case, seed, gen)
    return _prepare_rotary(case, gen)


# ---------------------------------------------------------------- the framework's calls


def _own_attn(c, s):
    states = s["initial"] is not None

    def call():
        return _cc().linear_attn_fn(s["q"], s["k"], s["v"], s["g"], cu_seqlens=s["cu"], initial_states=s["initial"],
                                    return_final_states=states)

    if not c["train"]:
        with torch.no_grad():
            r = call()
        return {"out": r[0], "final": r[1]} if states else {"out": r}
    r = call()
    wanted = [name for name in ("q", "k", "v", "g", "initial") if s[name] is not None]
    grads = torch.autograd.grad(r, [s[name] for name in wanted], (s["dout"], s["dfinal"]) if states else s["dout"])
    got = {"out": r[0], "final": r[1]} if states else {"out": r}
    got.update({"d" + name: g for name, g in zip(wanted, grads)})
    return got


def _own_step(c, s):
    out = _cc().linear_attn_update(s["q"], s["state"], s["k"], s["v"], s["g"], attn_state_indices=s["indices"])
    return {"out": out, "state": s["state"]}


def _own_rotary(c, s):
    def call():
        return _cc().head_norm_rotary_fn(s["q"], s["k"], s["wq"], s["wk"], inv_freq=s["freq"],
                                         positions=s["positions"], eps=1e-6, interleaved=c["interleaved"],
                                         amplitude=s["amplitude"])

    if not c["train"]:
        with torch.no_grad():
            q, k = call()
        return {"q": q, "k": k}
    q, k = call()
    wanted = [name for name in ("q", "k", "wq", "wk") if s[name] is not None]
    grads = torch.autograd.grad((q, k), [s[name] for name in wanted], (s["dq"], s["dk"]))
    return {"q": q, "k": k, **{"d" + name: g for name, g in zip(wanted, grads)}}


# ---------------------------------------------------------------- the plain forms


def _take(t, plan):
    """(batch, seqlen, heads, ..) as (chunks, heads, CHUNK, ..), 0 where a chunk holds no position."""
    at = plan["at"]
    rows = t.flatten(0, 1)[at.clamp(min=0)]
    rows = torch.where((at >= 0).reshape(*at.shape, *([1] * (rows.dim() - 2))), rows, 0.0)
    return rows.transpose(1, 2)


def _put(t, plan, shape):
    """_take's inverse, to a (batch, seqlen, heads, ..) tensor."""
    live = plan["at"] >= 0
    rows = torch.empty(shape[0] * shape[1], *shape[2:], dtype=t.dtype, device=t.device)
    rows[plan["at"][live]] = t.transpose(1, 2)[live]
    return rows.reshape(shape)


def _mul(a, b):
    return torch.matmul(a.contiguous(), b.contiguous())


def _turned(t):
    return t.transpose(-1, -2).contiguous()


def _plain_attn(c, s):
    dtype, plan = s["q"].dtype, s["plan"]
    H, K, dk, dv = c["heads"], c["key_heads"], c["dk"], c["dv"]
    scale = dk ** -0.5
    q, k, v = (_take(s[name].detach().float(), plan) for name in ("q", "k", "v"))
    q, k = (t.repeat_interleave(H // K, 1) for t in (q * scale, k))
    seq, N = plan["seq"], plan["at"].shape[0]
    g = _take(s["g"].detach().double()[..., None], plan)[..., 0]
    cum = g.cumsum(-1)
    reach = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=DEVICE).tril()
    rel = torch.exp(torch.where(reach, cum[..., :, None] - cum[..., None, :], -math.inf)).float()
    into, left, whole = torch.exp(cum).float(), torch.exp(cum[..., -1:] - cum).float(), torch.exp(cum[..., -1]).float()
    # what a chunk's state gets from the chunks before it in its sequence
    total = cum[..., -1].t().cumsum(1)
    before = torch.nn.functional.pad(total, (1, 0))[:, :-1]
    earlier = (seq[:, None] == seq) & (torch.arange(N, device=DEVICE)[:, None] > torch.arange(N, device=DEVICE))
    pass_on = torch.exp(torch.where(earlier, before[:, :, None] - total[:, None, :], -math.inf)).float()
    local = _mul(_turned(k * left[..., None]), v)
    flat = local.transpose(0, 1).reshape(H, N, dk * dv)
    state = _mul(pass_on, flat).reshape(H, N, dk, dv).transpose(0, 1)
    if s["initial"] is not None:
        from_first = torch.exp(before - before[:, plan["first"]][:, seq]).float().t()
        state = state + from_first[..., None, None] * s["initial"].detach()[seq]
    A = _mul(q, _turned(k)) * rel
    out = _mul(A, v) + into[..., None] * _mul(q, state)
    got = {"out": _put(out, plan, s["v"].shape).to(dtype)}
    end = whole[..., None, None] * state + local
    if s["initial"] is not None:
        got["final"] = end[plan["last"]]
    if not c["train"]:
        return got
    dout = _take(s["dout"].float(), plan)
    grad = _mul(_turned(q * into[..., None]), dout)
    flat = grad.transpose(0, 1).reshape(H, N, dk * dv)
    after = _mul(_turned(pass_on), flat).reshape(H, N, dk, dv).transpose(0, 1)
    if s["dfinal"] is not None:
        to_last = torch.exp(total[:, plan["last"]][:, seq] - total).float().t()
        after = after + to_last[..., None, None] * s["dfinal"][seq]
    dA = _mul(dout, _turned(v))
    dq_state = into[..., None] * _mul(dout, _turned(state))
    dk_state = left[..., None] * _mul(v, _turned(after))
    dq = _mul(dA * rel, k) + dq_state
    dkey = _mul(_turned(dA * rel), q) + dk_state
    dval = _mul(_turned(A), dout) + left[..., None] * _mul(k, after)
    # a decay's gradient: all that is carried over its position
    p = A.double() * dA.double()
    rows, cols = (q.double() * dq_state.double()).sum(-1), (k.double() * dk_state.double()).sum(-1)
    over = (p.sum(-1) - p.sum(-2)).flip(-1).cumsum(-1).flip(-1)
    dg = whole.double()[..., None] * (after.double() * state.double()).sum((-1, -2))[..., None] + over
    dg = dg + rows.flip(-1).cumsum(-1).flip(-1) + cols.cumsum(-1) - cols
    each = (N, K, H // K, CHUNK, dk)
    got["dq"] = _put(scale * dq.reshape(each).sum(2), plan, s["q"].shape).to(dtype)
    got["dk"] = _put(dkey.reshape(each).sum(2), plan, s["k"].shape).to(dtype)
    got["dv"] = _put(dval, plan, s["v"].shape).to(dtype)
    got["dg"] = _put(dg, plan, s["g"].shape).to(dtype)
    if s["initial"] is not None:
        first = plan["first"]
        got["dinitial"] = grad[first] + whole[first][..., None, None] * after[first]
    return got


def _plain_step(c, s):
    dtype, H, K, T = s["q"].dtype, c["heads"], c["key_heads"], c["tokens"]
    one = (lambda t: t[:, None]) if T == 1 else (lambda t: t)
    q, k, v = (one(s[name]).float().transpose(1, 2) for name in ("q", "k", "v"))
    g = one(s["g"]).double()
    q, k = (t.repeat_interleave(H // K, 1) for t in (q * c["dk"] ** -0.5, k))
    cum = g.cumsum(1).transpose(1, 2)
    reach = torch.ones(T, T, dtype=torch.bool, device=DEVICE).tril()
    rel = torch.exp(torch.where(reach, cum[..., :, None] - cum[..., None, :], -math.inf)).float()
    into, left = torch.exp(cum).float()[..., None], torch.exp(cum[..., -1:] - cum).float()[..., None]
    live = None
    state = s["state"]
    if s["indices"] is not None:
        live = s["indices"] >= 0
        state = state[s["indices"].clamp(min=0).long()]
    out = _mul(_mul(q, _turned(k)) * rel, v) + into * _mul(q, state)
    new = into[..., -1:, :] * state + _mul(_turned(k * left), v)
    if live is None:
        s["state"].copy_(new)
    else:
        out = torch.where(live[:, None, None, None], out, 0.0)
        s["state"][s["indices"][live].long()] = new[live]
    return {"out": out.transpose(1, 2).reshape(s["v"].shape).to(dtype), "state": s["state"]}


def _turn(c, x, cos, sin):
    """Pairs of the first rotated values turned by (cos, sin); the rest as it is."""
    R = c["rotated"]
    if not R:
        return x
    if c["interleaved"]:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., R:]), -1)


def _plain_rotary(c, s):
    dtype, got = s["q"].dtype, {}
    cos = sin = None
    if c["rotated"]:
        angle = s["positions"][..., None, None].double() * s["freq"].double()
        cos, sin = ((f(angle) * s["amplitude"]).float() for f in (torch.cos, torch.sin))

    def one(name):
        x, w = s[name].detach().float(), s["w" + name]
        rstd = torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) if w is not None else None
        xh = x if w is None else x * rstd
        got[name] = _turn(c, xh if w is None else xh * w.detach(), cos, sin).to(dtype)
        if not c["train"]:
            return
        d = _turn(c, s["d" + name].float(), cos, None if sin is None else -sin)
        if w is not None:
            got["dw" + name] = (d * xh).sum((0, 1, 2))
            d = d * w.detach()
            d = rstd * (d - xh * (d * xh).mean(-1, keepdim=True))
        got["d" + name] = d.to(dtype)

    one("q")
    one("k")
    return got


def run(state):
    c = state["case"]
    if own:
        return {"attn": _own_attn, "step": _own_step, "rotary": _own_rotary}[c["op"]](c, state)
    with torch.no_grad():
        return {"attn": _plain_attn, "step": _plain_step, "rotary": _plain_rotary}[c["op"]](c, state)


# ---------------------------------------------------------------- bytes and operations


def work(case):
    c = case
    size = 4 if c["dtype"] == "fp32" else 2
    H, K = c["heads"], c["key_heads"]
    if c["op"] == "rotary":
        tokens = c["batch"] * c["seqlen"]
        n = tokens * (H + K) * c["dim"]
        params = 8 * c["dim"] * (1 if c["norm"] else 0)
        moved, flops = 2 * n * size + params + 8 * tokens, 7 * n
        if c["train"]:  # the gradients of the results in, those of the inputs and the weights out
            moved, flops = moved + 2 * n * size + params, flops + 12 * n
        return {"bytes": moved, "flops": flops}
    dk, dv = c["dk"], c["dv"]
    if c["op"] == "step":
        T, live = c["tokens"], c["batch"] - c["padded"]
        moved = c["batch"] * T * (2 * K * dk + 2 * H * dv + H) * size + 8 * live * H * dk * dv
        moved += 4 * c["batch"] if c["rows"] else 0
        # of a state element and token: the decay (1), its step (2), the output (2)
        return {"bytes": moved, "flops": 5 * live * T * H * dk * dv}
    tokens = c["batch"] * c["seqlen"]
    keys, values, decays = tokens * K * dk * size, tokens * H * dv * size, tokens * H * size
    seqs = c["seqs"] if c["extra"] in ("packed", "prompts") else c["batch"]
    states = 4 * seqs * H * dk * dv if c["extra"] in ("states", "prompts") else 0
    moved, flops = 2 * keys + 2 * values + decays + 2 * states, 5 * tokens * H * dk * dv
    if c["train"]:  # dout in; the gradients of q, k, v, g and the states out
        moved += 2 * keys + 2 * values + decays + 2 * states
        # of a state element: the step of its gradient (3), the sums for q, k and v (6)
        flops += 9 * tokens * H * dk * dv
    return {"bytes": moved, "flops": flops}


# ---------------------------------------------------------------- 64 bits


def _exact_head(q, k, v, g, first, dout, dfinal):
    """One sequence of one head without chunks: every pair of positions. (out, final), and the gradients."""
    L = q.shape[0]
    cum = torch.cumsum(g, 0)
    M = (cum[:, None] - cum[None, :]).masked_fill_(torch.ones(L, L, dtype=torch.bool, device=DEVICE).triu_(1), -math.inf)
    M.exp_()
    A = (q @ k.t()).mul_(M)
    e, w = torch.exp(cum)[:, None], torch.exp(cum[-1] - cum)[:, None]
    got = [A @ v + e * (q @ first), torch.exp(cum[-1]) * first + (w * k).t() @ v]
    if dout is None:
        return got
    dA = dout @ v.t()
    r, b = e * (dout @ first.t()), w * (v @ dfinal.t())
    got.append(A.t() @ dout + w * (k @ dfinal))  # dv
    p = A.mul_(dA)
    # a decay's gradient: the pairs on its two sides, what enters before it and what leaves after it
    over = torch.cumsum((p.sum(1) - p.sum(0)).flip(0), 0).flip(0)
    dA.mul_(M)
    out_of, in_to = (q * r).sum(1), (k * b).sum(1)
    dg = over + torch.cumsum(out_of.flip(0), 0).flip(0) + torch.cumsum(in_to, 0) - in_to
    dg = dg + torch.exp(cum[-1]) * (first * dfinal).sum()
    got += [dA @ k + r, dA.t() @ q + b, dg, (e * q).t() @ dout + torch.exp(cum[-1]) * dfinal]
    return got


def _exact_attn(c, s):
    """Sequence by sequence and head by head."""
    H, K, dk, dv = c["heads"], c["key_heads"], c["dk"], c["dv"]
    d = {n: s[n].detach().double().flatten(0, 1) for n in ("q", "k", "v", "g")}
    scale = dk ** -0.5
    zero = torch.zeros(dk, dv, dtype=torch.float64, device=DEVICE)
    train = c["train"]
    dout = s["dout"].double().flatten(0, 1) if train else None
    out, dval, dg = torch.empty_like(d["v"]), torch.empty_like(d["v"]), torch.empty_like(d["g"])
    dq, dkey = torch.zeros_like(d["q"]), torch.zeros_like(d["k"])
    ends = s["bounds"]
    final = torch.empty(len(ends) - 1, H, dk, dv, dtype=torch.float64, device=DEVICE)
    dinitial = torch.empty_like(final)
    for i, (a, b) in enumerate(zip(ends, ends[1:])):
        for h in range(H):
            j = h // (H // K)
            first = zero if s["initial"] is None else s["initial"].detach()[i, h].double()
            dfinal = s["dfinal"][i, h].double() if train and s["dfinal"] is not None else zero
            r = _exact_head(d["q"][a:b, j] * scale, d["k"][a:b, j], d["v"][a:b, h], d["g"][a:b, h], first,
                            dout[a:b, h] if train else None, dfinal)
            out[a:b, h], final[i, h] = r[0], r[1]
            if train:
                dval[a:b, h], dg[a:b, h], dinitial[i, h] = r[2], r[5], r[6]
                dq[a:b, j] += r[3] * scale
                dkey[a:b, j] += r[4]
    states = s["initial"] is not None
    got = {"out": out.reshape(s["v"].shape)}
    if states:
        got["final"] = final
    if train:
        got.update(dq=dq.reshape(s["q"].shape), dk=dkey.reshape(s["k"].shape), dv=dval.reshape(s["v"].shape),
                   dg=dg.reshape(s["g"].shape))
        if states:
            got["dinitial"] = dinitial
    return got


def _exact_step(c, s):
    """Token by token, from the recurrence."""
    H, K, T = c["heads"], c["key_heads"], c["tokens"]
    of = torch.arange(H, device=DEVICE) // (H // K)
    lines = torch.arange(c["batch"], device=DEVICE) if s["indices"] is None else s["indices"].long()
    live = (lines >= 0).nonzero()[:, 0]
    state = s["state"].double()
    S = state[lines[live]]
    out = torch.zeros(s["v"].shape, dtype=torch.float64, device=DEVICE)
    for t in range(T):
        q, k, v, g = (s[n][live].double() if T == 1 else s[n][live, t].double() for n in ("q", "k", "v", "g"))
        S = torch.exp(g)[..., None, None] * S + k[:, of][..., :, None] * v[..., None, :]
        y = (q[:, of][..., :, None] * S).sum(2) * c["dk"] ** -0.5
        if T == 1:
            out[live] = y
        else:
            out[live, t] = y
    state[lines[live]] = S
    return {"out": out, "state": state}


def _exact_rotary(c, s):
    """Pairs as complex numbers."""
    R, got = c["rotated"], {}
    turn = None
    if R:
        angle = s["positions"].double()[..., None] * s["freq"].double()
        turn = torch.polar(torch.full_like(angle, s["amplitude"]), angle)[:, :, None]

    def turned(x, by):
        if by is None:
            return x
        pairs = x[..., :R].unflatten(-1, (R // 2, 2) if c["interleaved"] else (2, R // 2))
        at = -1 if c["interleaved"] else -2
        z = torch.complex(pairs.select(at, 0).contiguous(), pairs.select(at, 1).contiguous()) * by
        return torch.cat((torch.stack((z.real, z.imag), at).flatten(-2), x[..., R:]), -1)

    for name in ("q", "k"):
        x, w = s[name].detach().double(), s["w" + name]
        norm = 1.0 if w is None else 1.0 / torch.sqrt(torch.sum(x ** 2, -1, keepdim=True) / c["dim"] + 1e-6)
        weight = 1.0 if w is None else w.detach().double()
        got[name] = turned(x * norm * weight, turn)
        if c["train"]:
            d = turned(s["d" + name].double(), None if turn is None else turn.conj())
            if w is None:
                got["d" + name] = d
                continue
            got["dw" + name] = torch.sum(d * x * norm, (0, 1, 2))
            d = d * weight
            got["d" + name] = norm * d - x * norm ** 3 * torch.sum(d * x, -1, keepdim=True) / c["dim"]
    return got


def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "step": _exact_step, "rotary": _exact_rotary}[case["op"]](case, s)
