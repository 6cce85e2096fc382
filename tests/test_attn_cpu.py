"""Linear attention, its decode step and the rotation without a GPU: plain formulations against the definitions and
against differences, refusals of the entry points, and the C ABI."""

from __future__ import annotations

import ctypes
import math
import subprocess
from pathlib import Path

import pytest
import torch

import causal_conv1d_amd as cc
from _attn import attn64, rotary64
from causal_conv1d_amd import _lib

ROOT = Path(__file__).resolve().parent.parent
F64 = torch.float64


def _attn(B=2, L=9, H=4, K=2, dk=5, dv=3, seqs=None):
    r = lambda *s: torch.randn(*s, dtype=F64)  # noqa: E731
    return {"q": r(B, L, K, dk), "k": r(B, L, K, dk), "v": r(B, L, H, dv), "g": -r(B, L, H).abs(),
            "initial_states": r(B if seqs is None else seqs, H, dk, dv)}


def test_plain_form_is_the_definition():
    p = _attn()
    out, final = cc.linear_attn_ref(**p, return_final_states=True)
    e = attn64(p["q"], p["k"], p["v"], p["g"], 5**-0.5, p["initial_states"])
    torch.testing.assert_close(out, e["out"])
    torch.testing.assert_close(final, e["final"])


def test_definition_gradients_are_the_plain_forms_and_differences():
    p = _attn(1, 5)
    leaves = {n: t.requires_grad_() for n, t in p.items()}
    f = lambda *a: cc.linear_attn_ref(*a[:4], initial_states=a[4], return_final_states=True)  # noqa: E731
    r = f(*leaves.values())
    d = [torch.randn_like(t) for t in r]
    e = attn64(*list(p.values())[:4], 5**-0.5, p["initial_states"], *d)
    for n, g in zip(("dq", "dk", "dv", "dg", "dinit"), torch.autograd.grad(r, list(leaves.values()), d)):
        torch.testing.assert_close(e[n], g)
    assert torch.autograd.gradcheck(f, tuple(leaves.values()))


def test_plain_form_packed():
    p = _attn(1, 12, seqs=3)
    out, final = cc.linear_attn_ref(**p, cu_seqlens=torch.tensor([1, 4, 4, 10]), return_final_states=True)
    for i, (a, b) in enumerate(((1, 4), (4, 4), (4, 10))):
        e = attn64(*(p[n][:, a:b] for n in ("q", "k", "v", "g")), 5**-0.5, p["initial_states"][i:i + 1])
        torch.testing.assert_close(out[:, a:b], e["out"])
        torch.testing.assert_close(final[i:i + 1], e["final"])
    assert (out[:, 0] == 0).all() and (out[:, 10:] == 0).all()


def test_plain_update_is_the_plain_form():
    p = _attn(3, 4)
    state = torch.randn(5, 4, 5, 3, dtype=F64)
    before, rows = state.clone(), torch.tensor([4, -1, 0], dtype=torch.int32)
    out = cc.linear_attn_update_ref(p["q"], state, p["k"], p["v"], p["g"], attn_state_indices=rows)
    live = [0, 2]
    e, final = cc.linear_attn_ref(*(p[n][live] for n in ("q", "k", "v", "g")), initial_states=before[[4, 0]],
                                  return_final_states=True)
    torch.testing.assert_close(out[live], e)
    torch.testing.assert_close(state[[4, 0]], final)
    assert (out[1] == 0).all() and torch.equal(state[1:4], before[1:4])


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
def test_plain_rotation_is_the_definition(norm, interleaved):
    q, k = torch.randn(2, 6, 3, 10, dtype=F64), torch.randn(2, 6, 1, 10, dtype=F64)
    wq, wk = (torch.rand(10, dtype=F64) + 0.5 if norm else None for _ in range(2))
    freq, pos = torch.tensor([1.0, 0.1, 0.013, 0.5], dtype=torch.float32), torch.randint(0, 9999, (2, 6))
    leaves = [t.requires_grad_() for t in (q, k, wq, wk) if t is not None]
    r = cc.head_norm_rotary_ref(q, k, wq, wk, freq, pos, 1e-3, interleaved, 1.5)
    d = [torch.randn_like(t) for t in r]
    e, _ = rotary64(q, k, wq, wk, freq, pos, 1e-3, interleaved, 1.5, *d)
    torch.testing.assert_close(r[0], e["q"])
    torch.testing.assert_close(r[1], e["k"])
    for n, g in zip(("dq", "dk", "dwq", "dwk"), torch.autograd.grad(r, leaves, d)):
        torch.testing.assert_close(e[n], g)


def test_frequencies():
    f, a = cc.rotary_frequencies(64)
    assert f.dtype == torch.float32 and f.shape == (32,) and a == 1.0 and f[0] == 1.0
    torch.testing.assert_close(f[-1].item(), 10000.0 ** (-62 / 64))
    g, a = cc.rotary_frequencies(64, scaling="linear", factor=4.0)
    torch.testing.assert_close(g, f / 4)
    g, a = cc.rotary_frequencies(64, scaling="base", factor=8.0)
    assert g[0] == 1.0 and a == 1.0
    torch.testing.assert_close(g[-1], f[-1] / 8)
    g, a = cc.rotary_frequencies(64, scaling="ramp", factor=16.0, trained_length=4096)
    turns = 4096 * f.double() / (2 * math.pi)
    assert torch.equal(g[turns > 32], f[turns > 32]) and a == pytest.approx(0.1 * math.log(16) + 1)
    torch.testing.assert_close(g[turns < 1], f[turns < 1] / 16)
    assert ((g <= f) & (g >= f / 16 * (1 - 1e-6))).all()


@pytest.mark.parametrize("kw", [{"rotated": 3}, {"rotated": 0}, {"factor": 0.5}, {"scaling": "other"}, {"base": 0.0},
                                {"scaling": "ramp", "fast_turns": 1.0}])
def test_frequency_refusals(kw):
    with pytest.raises(ValueError):
        cc.rotary_frequencies(**{"rotated": 64, **kw})


# ---------------------------------------------------------------- refusals


def _z(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def _call():
    return {"q": _z(2, 6, 2, 8), "k": _z(2, 6, 2, 8), "v": _z(2, 6, 4, 16), "g": _z(2, 6, 4)}


@pytest.mark.parametrize("error,match,kw", [
    (NotImplementedError, "unsupported dtype", {"q": _z(2, 6, 2, 8, dtype=F64)}),
    (ValueError, "expected q of shape", {"q": _z(2, 6, 2)}),
    (ValueError, "expected q, k and v", {"v": _z(2, 6, 4)}),
    (ValueError, "k shape", {"k": _z(2, 6, 1, 8)}),
    (ValueError, "v shape", {"v": _z(2, 5, 4, 16)}),
    (ValueError, "g shape", {"g": _z(2, 6, 2)}),
    (NotImplementedError, "g.dtype", {"g": _z(2, 6, 4, dtype=torch.float32)}),
    (NotImplementedError, "k.dtype", {"k": _z(2, 6, 2, 8, dtype=torch.float16)}),
    (ValueError, "must be a multiple", {"v": _z(2, 6, 3, 16)}),
    (ValueError, "must be a multiple", {"q": _z(2, 6, 0, 8), "k": _z(2, 6, 0, 8)}),
    (NotImplementedError, "head size must be in", {"q": _z(2, 6, 2, 129), "k": _z(2, 6, 2, 129)}),
    (NotImplementedError, "head size must be in", {"v": _z(2, 6, 4, 0)}),
    (ValueError, "cu_seqlens needs batch == 1", {"cu_seqlens": torch.zeros(2, dtype=torch.int32)}),
    (ValueError, "initial_states shape", {"initial_states": torch.zeros(2, 4, 16, 8)}),
    (NotImplementedError, "initial_states.dtype", {"initial_states": _z(2, 4, 8, 16)}),
    (NotImplementedError, "ROCm", {}),
])
def test_attn_refusals(error, match, kw):
    with pytest.raises(error, match=match):
        cc.linear_attn_fn(**{**_call(), **kw})


@pytest.mark.parametrize("match,cu", [("cu_seqlens shape", torch.zeros(1, dtype=torch.int32)),
                                      ("cu_seqlens shape", torch.zeros(2, 2, dtype=torch.int32)),
                                      ("cu_seqlens.dtype must be int32", torch.zeros(2, dtype=torch.int64))])
def test_cu_seqlens_refusals(match, cu):
    with pytest.raises(ValueError, match=match):
        cc.linear_attn_fn(**{n: t[:1] for n, t in _call().items()}, cu_seqlens=cu)


@pytest.mark.parametrize("error,match,kw", [
    (ValueError, "expected q", {"q": _z(2, 8)}),
    (ValueError, "expected q", {"attn_state": torch.zeros(2, 4, 8)}),
    (ValueError, "attn_state shape", {"attn_state": torch.zeros(3, 4, 8, 16)}),
    (NotImplementedError, "attn_state.dtype", {"attn_state": _z(2, 4, 8, 16)}),
    (ValueError, "attn_state_indices shape", {"attn_state_indices": torch.zeros(3, dtype=torch.int32)}),
    (ValueError, "attn_state_indices.dtype must be int32", {"attn_state_indices": torch.zeros(2, dtype=torch.int64)}),
    (NotImplementedError, "ROCm", {}),
])
def test_update_refusals(error, match, kw):
    p = {n: t[:, 0] for n, t in _call().items()}
    p["attn_state"] = torch.zeros(2, 4, 8, 16)
    with pytest.raises(error, match=match):
        cc.linear_attn_update(**{**p, **kw})


@pytest.mark.parametrize("error,match,kw", [
    (NotImplementedError, "unsupported dtype", {"q": _z(2, 6, 4, 8, dtype=F64)}),
    (ValueError, "expected q", {"q": _z(2, 8)}),
    (ValueError, "expected q", {"k": _z(2, 5, 2, 8)}),
    (ValueError, "expected q", {"k": _z(2, 6, 2, 10)}),
    (NotImplementedError, "must match q", {"k": _z(2, 6, 2, 8, dtype=torch.float16)}),
    (NotImplementedError, "dim must be in", {"q": _z(2, 6, 4, 257), "k": _z(2, 6, 2, 257)}),
    (ValueError, "q_weight shape", {"q_weight": torch.ones(7)}),
    (NotImplementedError, "k_weight.dtype", {"k_weight": _z(8)}),
    (ValueError, "inv_freq shape", {"inv_freq": torch.ones(5)}),
    (NotImplementedError, "inv_freq.dtype", {"inv_freq": _z(4)}),
    (ValueError, "positions shape", {"positions": torch.zeros(6, dtype=torch.int64)}),
    (ValueError, "positions.dtype", {"positions": torch.zeros(2, 6)}),
    (ValueError, "single tokens need positions", {"q": _z(2, 4, 8), "k": _z(2, 2, 8), "inv_freq": torch.ones(4)}),
    (NotImplementedError, "ROCm", {}),
])
def test_rotary_refusals(error, match, kw):
    with pytest.raises(error, match=match):
        cc.head_norm_rotary_fn(**{"q": _z(2, 6, 4, 8), "k": _z(2, 6, 2, 8), **kw})


# ---------------------------------------------------------------- the C ABI

STRUCTS = {"cc1d_attn_params": _lib.AttnParams, "cc1d_attn_bwd_params": _lib.AttnBwdParams,
           "cc1d_attn_update_params": _lib.AttnUpdateParams, "cc1d_rotary_params": _lib.RotaryParams,
           "cc1d_rotary_bwd_params": _lib.RotaryBwdParams}


def test_struct_layout_matches_header(tmp_path):
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "cc1d.h"', "int main(void) {"]
    for cname, st in STRUCTS.items():
        lines.append(f'printf("{cname} sizeof %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in st._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join([*lines, "return 0; }"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c11", f"-I{ROOT / 'include'}", str(src), "-o", str(exe)], check=True)
    for ln in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        s, f, v = ln.split()
        assert int(v) == (ctypes.sizeof(STRUCTS[s]) if f == "sizeof" else getattr(STRUCTS[s], f).offset), (s, f)


def _fill(p, sizes, kw):
    for k, v in {**sizes, **kw}.items():
        setattr(p, k, v)
    return p


ATTN = {"batch": 1, "seqlen": 16, "heads": 4, "key_heads": 2, "dk": 8, "dv": 8, "dtype": 1, "scale": 1.0}


@pytest.mark.parametrize("code,kw", [
    (2, {"dtype": 3}), (14, {"dk": 0}), (14, {"dk": 129}), (14, {"dv": 129}), (4, {"seqlen": -1}), (13, {"key_heads": 3}),
    (13, {"key_heads": 0}), (4, {"cu_seqlens": 16, "batch": 2, "num_seqs": 1}), (4, {"cu_seqlens": 16, "num_seqs": 0}),
    (4, {"batch": 1 << 22}), (4, {"heads": 1 << 22}), (4, {"seqlen": 1 << 31}), (4, {"batch": 1 << 16, "heads": 1 << 10}),
    (1, {}), (0, {"batch": 0}), (0, {"heads": 0}), (0, {"seqlen": 0}),
])
def test_attn_codes(code, kw):
    lib = _lib.load()
    assert lib.cc1d_attn_fwd(None, None) == 1 and lib.cc1d_attn_bwd(None, None) == 1
    p = _fill(_lib.AttnParams(), ATTN, kw)
    assert lib.cc1d_attn_fwd(ctypes.byref(p), None) == code
    assert lib.cc1d_strerror(code).decode() != "unknown status"
    assert (lib.cc1d_attn_workspace_floats(ctypes.byref(p)) < 0) == (code not in (0, 1))
    b = _lib.AttnBwdParams()
    b.fwd = p
    assert (lib.cc1d_attn_bwd_workspace_floats(ctypes.byref(b)) < 0) == (code not in (0, 1))
    if code not in (0, 1):
        assert lib.cc1d_attn_bwd(ctypes.byref(b), None) == code


def test_attn_needs_its_workspace():
    lib = _lib.load()
    p = _fill(_lib.AttnParams(), ATTN, {"seqlen": 4096, **{n: 16 for n in ("q", "k", "v", "g", "out")}})
    n = lib.cc1d_attn_workspace_floats(ctypes.byref(p))
    assert n > 0
    p.workspace, p.workspace_floats = 16, n - 1
    assert lib.cc1d_attn_fwd(ctypes.byref(p), None) == 8
    p.workspace, p.workspace_floats = None, n
    assert lib.cc1d_attn_fwd(ctypes.byref(p), None) == 1
    b = _lib.AttnBwdParams()
    b.fwd = p
    for name in ("dout", "dq", "dk", "dv", "dg"):
        setattr(b, name, 16)
    n = lib.cc1d_attn_bwd_workspace_floats(ctypes.byref(b))
    b.workspace, b.workspace_floats = 16, n - 1
    assert lib.cc1d_attn_bwd(ctypes.byref(b), None) == 8
    b.workspace, b.workspace_floats = None, n
    assert lib.cc1d_attn_bwd(ctypes.byref(b), None) == 1


UPDATE = {"batch": 2, "tokens": 1, "heads": 4, "key_heads": 2, "dk": 8, "dv": 8, "state_rows": 2, "dtype": 1, "scale": 1.0}


@pytest.mark.parametrize("code,kw", [
    (2, {"dtype": -1}), (14, {"dk": 129}), (14, {"dv": 0}), (4, {"tokens": -1}), (13, {"key_heads": 3}), (4, {"state_rows": 1}),
    (4, {"batch": 1 << 23, "state_rows": 1 << 23}), (1, {}), (0, {"batch": 0}), (0, {"heads": 0}), (0, {"tokens": 0}),
])
def test_update_codes(code, kw):
    lib = _lib.load()
    assert lib.cc1d_attn_update(None, None) == 1
    p = _fill(_lib.AttnUpdateParams(), UPDATE, kw)
    assert lib.cc1d_attn_update(ctypes.byref(p), None) == code


ROTARY = {"batch": 1, "seqlen": 4, "q_heads": 4, "k_heads": 2, "dim": 64, "rotated": 64, "dtype": 1, "inv_freq": 16,
          "positions_bytes": 8}


@pytest.mark.parametrize("code,kw", [
    (2, {"dtype": 3}), (14, {"dim": 0}), (14, {"dim": 257}), (15, {"rotated": 3}), (15, {"rotated": 66}), (15, {"rotated": -2}),
    (4, {"q_heads": -1}), (4, {"batch": 1 << 24}), (2, {"positions": 16, "positions_bytes": 2}), (1, {"inv_freq": None}), (1, {}),
    (0, {"batch": 0}), (0, {"seqlen": 0, "inv_freq": None}), (0, {"q_heads": 0, "k_heads": 0}),
])
def test_rotary_codes(code, kw):
    lib = _lib.load()
    assert lib.cc1d_rotary_fwd(None, None) == 1 and lib.cc1d_rotary_bwd(None, None) == 1
    p = _fill(_lib.RotaryParams(), ROTARY, kw)
    assert lib.cc1d_rotary_fwd(ctypes.byref(p), None) == code
    b = _lib.RotaryBwdParams()
    b.fwd = p
    b.fwd.q_weight = 16
    if code not in (0, 1):
        assert lib.cc1d_rotary_bwd(ctypes.byref(b), None) == code
        assert lib.cc1d_rotary_bwd_workspace_floats(ctypes.byref(b)) < 0
    else:
        assert lib.cc1d_rotary_bwd(ctypes.byref(b), None) == 1  # the weight's gradient is missing


def test_messages():
    lib = _lib.load()
    for code in (13, 14, 15):
        assert lib.cc1d_strerror(code).decode() != "unknown status"
