"""The scan, its decode step and the norm without a GPU: the float64 formulas that
the GPU tests compare with (against autograd and against differences), the plain
torch formulations, argument checks, the C ABI's refusals and struct layouts."""

from __future__ import annotations

import ctypes
import re
import subprocess
from pathlib import Path

import pytest
import torch

import causal_conv1d_amd as cc
from _ssm import norm64, scan64
from causal_conv1d_amd import _lib
from causal_conv1d_amd._scan import scan_tile_floats

ROOT = Path(__file__).resolve().parent.parent


def _inputs(B=2, D=4, L=9, N=3, G=2, dtype=torch.float64):
    r = lambda *s: torch.randn(*s, dtype=torch.float64).to(dtype)  # noqa: E731
    return dict(u=r(B, D, L), delta=0.5 * r(B, D, L), A=-torch.rand(D, N, dtype=torch.float64) * 2, B=r(B, G, N, L),
                C=r(B, G, N, L), D=r(D).double(), z=r(B, D, L), delta_bias=0.3 * r(D).double())


# ---------------------------------------------------------------- the formulas


@pytest.mark.parametrize("gate,softplus,extra", [(True, True, "states"), (False, True, "ids"), (True, False, "ids"),
                                                 (False, False, "none")])
def test_scan_formulas_are_the_gradients_of_the_recurrence(gate, softplus, extra):
    p = _inputs()
    if not gate:
        p["z"] = None
    ids = torch.tensor([[0, 0, 0, 1, 1, -1, -1, 2, 2], [-1, 4, 4, 4, 3, 4, 4, 4, -2]], dtype=torch.int32)
    ids = ids if extra == "ids" else None
    init = torch.randn(2, 4, 3, dtype=torch.float64) if extra == "states" else None
    leaves = {k: v.requires_grad_() for k, v in {**p, "init": init}.items() if v is not None}
    out, fin = cc.ssm_scan_ref(**p, delta_softplus=softplus, seq_idx=ids, initial_states=init, return_final_states=True)
    dout, dfin = torch.randn_like(out), torch.randn_like(fin) if extra == "states" else None
    grads = torch.autograd.grad((out, fin) if dfin is not None else out, list(leaves.values()),
                                (dout, dfin) if dfin is not None else dout)
    e = scan64(p["u"], p["delta"], p["A"], p["B"], p["C"], p["D"], p["z"], p["delta_bias"], softplus, ids, init, dout,
               dfin)
    names = {"u": "du", "delta": "ddelta", "A": "dA", "B": "dB", "C": "dC", "D": "dD", "z": "dz",
             "delta_bias": "dbias", "init": "dinit"}
    torch.testing.assert_close(e["out"], out.detach(), rtol=1e-12, atol=1e-12)
    for k, g in zip(leaves, grads):
        torch.testing.assert_close(e[names[k]], g, rtol=1e-10, atol=1e-11, msg=lambda s, k=k: f"{k}: {s}")


def test_scan_formulas_agree_with_differences():
    p = _inputs(B=1, D=2, L=6, N=2, G=1)
    init, dfin = torch.randn(1, 2, 2, dtype=torch.float64), torch.randn(1, 2, 2, dtype=torch.float64)
    dout = torch.randn(1, 2, 6, dtype=torch.float64)

    def loss(**kw):
        q = {**p, "init": init, **kw}
        e = scan64(q["u"], q["delta"], q["A"], q["B"], q["C"], q["D"], q["z"], q["delta_bias"], True, None, q["init"])
        return ((e["out"] * dout).sum() + (e["final"] * dfin).sum()).item()

    e = scan64(p["u"], p["delta"], p["A"], p["B"], p["C"], p["D"], p["z"], p["delta_bias"], True, None, init, dout, dfin)
    for k, g in (("u", "du"), ("delta", "ddelta"), ("A", "dA"), ("B", "dB"), ("C", "dC"), ("D", "dD"), ("z", "dz"),
                 ("delta_bias", "dbias"), ("init", "dinit")):
        base = {**p, "init": init}[k]
        for i in range(base.numel()):
            step = torch.zeros_like(base).view(-1)
            step[i] = 1e-5
            d = (loss(**{k: base + step.view_as(base)}) - loss(**{k: base - step.view_as(base)})) / 2e-5
            assert abs(d - e[g].reshape(-1)[i].item()) < 1e-7 * (1 + abs(d)), (k, i)  # O(step^2) and 1e-16 / step


@pytest.mark.parametrize("rms", [False, True])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_formulas_are_the_gradients(rms, residual):
    x, w, b = torch.randn(3, 7).double(), torch.randn(7).double(), torch.randn(7).double()
    r = torch.randn(3, 7).double() if residual else None
    leaves = [t.requires_grad_() for t in (x, w, b, r) if t is not None]
    got = cc.add_norm_ref(x, w, b, r, 1e-5, rms, return_residual=residual)
    dy, ds = torch.randn(3, 7).double(), torch.randn(3, 7).double() if residual else None
    grads = torch.autograd.grad(got, leaves, (dy, ds) if residual else dy)
    e, _ = norm64(x, w, b, r, 1e-5, rms, dy, ds)
    for g, k in zip(grads, ("dx", "dw", "db", "dx")):
        torch.testing.assert_close(e[k], g, rtol=1e-11, atol=1e-11)
    base = x.detach().clone()
    for i in range(0, 21, 4):  # differences
        step = torch.zeros(21, dtype=torch.float64)
        step[i] = 1e-5
        f = lambda s: (lambda v: (v["out"] * dy).sum() + (0 if ds is None else (v["sum"] * ds).sum()))(  # noqa: E731
            norm64(base + s * step.view(3, 7), w, b, r, 1e-5, rms)[0]).item()
        d = (f(1) - f(-1)) / 2e-5
        assert abs(d - e["dx"].reshape(-1)[i].item()) < 1e-7 * (1 + abs(d))


def test_a_planted_mistake_is_seen():
    """The comparison's bound is tight enough to see a decay taken one position late."""
    from _ssm import close

    p = _inputs(dtype=torch.float32)
    e = scan64(*(p[k] for k in ("u", "delta", "A", "B", "C")), softplus=True)
    s = scan64(*(p[k] for k in ("u", "delta", "A", "B", "C")), softplus=True, mag=True)
    wrong = scan64(p["u"], torch.roll(p["delta"], 1, -1), *(p[k] for k in ("A", "B", "C")), softplus=True)
    close(e["out"].float(), e["out"], s["out"], 9)
    with pytest.raises(AssertionError, match="beyond the bound"):
        close(wrong["out"].float(), e["out"], s["out"], 9)


def test_references_agree_with_each_other():
    p = _inputs(B=1, L=11)
    cu = torch.tensor([0, 4, 4, 9], dtype=torch.int32)
    init = torch.randn(3, 4, 3, dtype=torch.float64)
    out, fin = cc.ssm_scan_ref(**p, delta_softplus=True, cu_seqlens=cu, initial_states=init, return_final_states=True)
    assert (out[..., 9:] == 0).all() and torch.equal(fin[1], init[1])
    state = torch.cat([init, init])
    for t in range(4):
        step = {k: (v[..., t] if k in ("u", "delta", "z", "B", "C") else v) for k, v in p.items()}
        got = cc.ssm_scan_update_ref(step.pop("u"), state, **step, delta_softplus=True,
                                     ssm_state_indices=torch.tensor([3], dtype=torch.int32))
        torch.testing.assert_close(got, out[..., t])
    torch.testing.assert_close(state[3], fin[0])
    assert torch.equal(state[:3], init) and torch.equal(state[4:], init[1:])


def test_softplus_polynomial_is_as_close_as_it_says():
    """The kernels' atanh(s) / s, with the coefficients and the bound read from the source."""
    src = (ROOT / "causal-conv1d-mojo_amd" / "csrc" / "cc1d_scan_device.hpp").read_text()
    said = float(re.search(r"Chebyshev points \(([\d.e-]+) off at most\)", src).group(1))
    body = src[src.index("float softplus(float raw)"):src.index("float sigmoid(float x)")]
    first = re.search(r"p = __builtin_fmaf\(s2, ([\d.]+)f, ([\d.]+)f\)", body).groups()
    coefficients = [float(torch.tensor(float(c))) for c in (*first, *re.findall(r"fmaf\(s2, p, ([\d.]+)f\)", body))]
    assert len(coefficients) == 5
    s = torch.linspace(1e-6, 1 / 3, 200001, dtype=torch.float64)
    p = torch.zeros_like(s)
    for c in coefficients:
        p = p * s * s + c
    off = (p - torch.atanh(s) / s).abs().max().item()
    assert said / 2 < off <= said


# ---------------------------------------------------------------- refusals


def _bf16(**kw):
    p = {k: (v.bfloat16() if k in ("u", "delta", "z", "B", "C") else v.float()) for k, v in _inputs().items()}
    p.update(kw)
    return p


@pytest.mark.parametrize("error,match,kw", [
    (NotImplementedError, "unsupported dtype", {"u": torch.zeros(2, 4, 9, dtype=torch.float64)}),
    (ValueError, "expected u of shape", {"u": torch.zeros(4, 9)}),
    (NotImplementedError, "delta.dtype", {"delta": torch.zeros(2, 4, 9)}),
    (ValueError, "delta shape", {"delta": torch.zeros(2, 4, 8).bfloat16()}),
    (ValueError, "z shape", {"z": torch.zeros(2, 3, 9).bfloat16()}),
    (ValueError, "A shape", {"A": torch.zeros(5, 3)}),
    (ValueError, "A shape", {"A": torch.zeros(4)}),
    (NotImplementedError, "A.dtype", {"A": torch.zeros(4, 3).bfloat16()}),
    (NotImplementedError, "dstate must be in", {"A": torch.zeros(4, 257)}),
    (NotImplementedError, "dstate must be in", {"A": torch.zeros(4, 0)}),
    (ValueError, "expected B and C", {"B": torch.zeros(2, 3, 9).bfloat16()}),
    (ValueError, "B shape", {"B": torch.zeros(2, 2, 4, 9).bfloat16()}),
    (NotImplementedError, "C.dtype", {"C": torch.zeros(2, 2, 3, 9)}),
    (ValueError, "multiple of B's groups", {"B": torch.zeros(2, 3, 3, 9).bfloat16(), "C": torch.zeros(2, 3, 3, 9).bfloat16()}),
    (ValueError, "D shape", {"D": torch.zeros(3)}),
    (NotImplementedError, "delta_bias.dtype", {"delta_bias": torch.zeros(4).bfloat16()}),
    (ValueError, "seq_idx shape", {"seq_idx": torch.zeros(2, 8, dtype=torch.int32)}),
    (ValueError, "seq_idx.dtype must be int32", {"seq_idx": torch.zeros(2, 9, dtype=torch.int64)}),
    (ValueError, "mutually exclusive", {"seq_idx": torch.zeros(2, 9, dtype=torch.int32), "return_final_states": True}),
    (ValueError, "mutually exclusive", {"seq_idx": torch.zeros(2, 9, dtype=torch.int32),
                                        "cu_seqlens": torch.zeros(2, dtype=torch.int32)}),
    (ValueError, "batch == 1", {"cu_seqlens": torch.tensor([0, 9], dtype=torch.int32)}),
    (ValueError, "initial_states shape", {"initial_states": torch.zeros(2, 4, 4)}),
    (NotImplementedError, "initial_states.dtype", {"initial_states": torch.zeros(2, 4, 3).bfloat16()}),
    (NotImplementedError, "ROCm", {}),
])
def test_scan_refusals(error, match, kw):
    with pytest.raises(error, match=match):
        cc.ssm_scan_fn(**_bf16(**kw), delta_softplus=True)


def test_scan_refuses_odd_cu_seqlens():
    p = {k: v[:1] if k in ("u", "delta", "z", "B", "C") else v for k, v in _bf16().items()}
    for cu, match in ((torch.zeros(1, dtype=torch.int32), "cu_seqlens shape"),
                      (torch.zeros(2, 2, dtype=torch.int32), "cu_seqlens shape"),
                      (torch.tensor([0, 9]), "cu_seqlens.dtype must be int32")):
        with pytest.raises(ValueError, match=match):
            cc.ssm_scan_fn(**p, cu_seqlens=cu)


@pytest.mark.parametrize("error,match,kw", [
    (ValueError, "expected u", {"u": torch.zeros(2).bfloat16()}),
    (ValueError, "delta shape", {"delta": torch.zeros(2, 5).bfloat16()}),
    (ValueError, "ssm_state shape", {"ssm_state": torch.zeros(3, 4, 3)}),
    (NotImplementedError, "ssm_state.dtype", {"ssm_state": torch.zeros(2, 4, 3).bfloat16()}),
    (ValueError, "expected B and C", {"B": torch.zeros(2, 2, 3, 1).bfloat16()}),
    (ValueError, "B shape", {"B": torch.zeros(2, 2, 4).bfloat16()}),
    (ValueError, "ssm_state_indices shape", {"ssm_state_indices": torch.zeros(3, dtype=torch.int32)}),
    (ValueError, "ssm_state_indices.dtype must be int32", {"ssm_state_indices": torch.zeros(2, dtype=torch.int64)}),
    (NotImplementedError, "ROCm", {}),
])
def test_update_refusals(error, match, kw):
    p = {k: v[..., 0] if k in ("u", "delta", "z", "B", "C") else v for k, v in _bf16().items()}
    p["ssm_state"] = torch.zeros(2, 4, 3)
    p.update(kw)
    with pytest.raises(error, match=match):
        cc.ssm_scan_update(p.pop("u"), p.pop("ssm_state"), **p)


@pytest.mark.parametrize("error,match,kw", [
    (NotImplementedError, "unsupported dtype", {"x": torch.zeros(2, 8, dtype=torch.float64)}),
    (ValueError, "weight shape", {"weight": torch.ones(7)}),
    (NotImplementedError, "bias.dtype", {"bias": torch.ones(8).bfloat16()}),
    (ValueError, "residual shape", {"residual": torch.zeros(3, 8).bfloat16()}),
    (NotImplementedError, "residual.dtype", {"residual": torch.zeros(2, 8).half()}),
    (NotImplementedError, "dim must be in", {"x": torch.zeros(2, 0).bfloat16(), "weight": torch.ones(0)}),
    (NotImplementedError, "dim must be in", {"x": torch.zeros(1, 32769).bfloat16(), "weight": torch.ones(32769)}),
    (NotImplementedError, "ROCm", {}),
])
def test_norm_refusals(error, match, kw):
    p = {"x": torch.zeros(2, 8).bfloat16(), "weight": torch.ones(8)}
    p.update(kw)
    with pytest.raises(error, match=match):
        cc.add_norm_fn(**p)


# ---------------------------------------------------------------- the C ABI

STRUCTS = {"cc1d_scan_params": _lib.ScanParams, "cc1d_scan_bwd_params": _lib.ScanBwdParams,
           "cc1d_scan_update_params": _lib.ScanUpdateParams, "cc1d_norm_params": _lib.NormParams,
           "cc1d_norm_bwd_params": _lib.NormBwdParams}


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


def _scan(**kw):
    p = _lib.ScanParams()
    p.batch, p.dim, p.seqlen, p.dstate, p.groups, p.dtype = 1, 8, 16, 4, 1, 1
    for k, v in kw.items():
        setattr(p, k, v)
    return p


@pytest.mark.parametrize("code,kw", [
    (2, {"dtype": 3}), (10, {"dstate": 0}), (10, {"dstate": 257}), (4, {"seqlen": -1}), (11, {"groups": 3}),
    (11, {"groups": 0}), (5, {"seq_idx": 16, "initial_states": 16}), (5, {"seq_idx": 16, "final_states": 16}),
    (5, {"seq_idx": 16, "cu_seqlens": 16}), (4, {"cu_seqlens": 16, "batch": 2, "num_seqs": 1}),
    (4, {"cu_seqlens": 16, "num_seqs": 0}), (4, {"batch": 1 << 20, "dim": 1 << 20}), (4, {"seqlen": 1 << 31}),
    (1, {}), (0, {"batch": 0}), (0, {"dim": 0}), (0, {"seqlen": 0}),
])
def test_scan_codes(code, kw):
    lib = _lib.load()
    assert lib.cc1d_scan_fwd(None, None) == 1
    p = _scan(**kw)
    assert lib.cc1d_scan_fwd(ctypes.byref(p), None) == code
    assert lib.cc1d_strerror(code).decode() != "unknown status"
    assert (lib.cc1d_scan_tile_floats(ctypes.byref(p)) < 0) == (code not in (0, 1))
    b = _lib.ScanBwdParams()
    b.fwd = p
    assert (lib.cc1d_scan_bwd_workspace_floats(ctypes.byref(b)) < 0) == (code not in (0, 1))
    if code not in (0, 1):
        assert lib.cc1d_scan_bwd(ctypes.byref(b), None) == code


@pytest.mark.parametrize("kw", [{"batch": 1 << 16, "dim": 4096},  # rows of 16 positions: 32 channels a block of 512 threads
                                {"num_seqs": 1 << 14, "cu_seqlens": 16, "dim": 4096, "seqlen": 512},
                                {"batch": 1 << 14, "dim": 4096, "seqlen": 100}], ids=["short", "packed", "rows"])
def test_scans_of_more_threads_than_a_launch_has_are_refused(kw):
    """A launch counts its threads in 32 bits: what has more is refused as a shape, before anything runs."""
    lib = _lib.load()
    p = _scan(u=16, delta=16, A=16, B=16, C=16, out=16, tile_states=16, **kw)
    assert lib.cc1d_scan_fwd(ctypes.byref(p), None) == 4


def test_scan_bwd_of_more_threads_than_a_launch_has_is_refused():
    lib = _lib.load()
    b = _lib.ScanBwdParams()
    for k in ("dout", "du", "ddelta", "dA", "dB", "dC", "workspace"):
        setattr(b, k, 16)
    b.workspace_floats = 1 << 62
    b.fwd = _scan(u=16, delta=16, A=16, B=16, C=16, tile_states=16, dim=1 << 25, dstate=256, seqlen=4)
    assert lib.cc1d_scan_bwd(ctypes.byref(b), None) == 4  # a thread per channel and state of dA


def test_scan_update_of_more_threads_than_a_launch_has_is_refused():
    p = _lib.ScanUpdateParams()
    p.batch, p.dim, p.seqlen, p.dstate, p.groups, p.state_rows, p.dtype = 1 << 18, 4096, 1, 16, 1, 1 << 18, 1
    for k in ("u", "delta", "A", "B", "C", "ssm_state", "out"):
        setattr(p, k, 16)
    assert _lib.load().cc1d_scan_update(ctypes.byref(p), None) == 4


def test_messages_fit_the_scan_and_the_norm():
    """The codes that the convolution's entry points also give name what these lack."""
    lib = _lib.load()
    assert "cu_seqlens" in lib.cc1d_strerror(5).decode()
    workspace = lib.cc1d_strerror(8).decode()
    assert "cc1d_bwd" not in workspace and "_workspace_floats()" in workspace


@pytest.mark.parametrize("batch,dim,seqlen,dstate,groups", [
    (4, 5120, 2048, 16, 1), (4, 5120, 2048, 17, 1), (4, 5120, 2048, 64, 1), (4, 5120, 2048, 128, 1), (8, 8192, 4096, 128, 1),
    (1, 5120, 16384, 128, 1), (512, 1024, 300, 256, 1), (4096, 4096, 64, 64, 1), (65536, 64, 64, 256, 1),
    (64, 4096, 8192, 16, 8), (1, 8192, 1 << 20, 256, 1), (1, 2048, 2048, 64, 8)])
def test_scan_bwd_workspace_does_not_grow_with_everything(batch, dim, seqlen, dstate, groups):
    """The shares of dB and dC are those of a part of the call: 2**30 floats at most (of these sizes)."""
    b = _lib.ScanBwdParams()
    b.fwd = _scan(batch=batch, dim=dim, seqlen=seqlen, dstate=dstate, groups=groups)
    params = batch * dim * (2 * dstate + 2)
    shares = _lib.load().cc1d_scan_bwd_workspace_floats(ctypes.byref(b)) - params
    assert 2 * groups * dstate <= shares <= 1 << 30


def test_scan_bwd_needs_its_workspace():
    b = _lib.ScanBwdParams()
    b.fwd = _scan(u=16, delta=16, A=16, B=16, C=16, tile_states=16)
    for k in ("dout", "du", "ddelta", "dA", "dB", "dC", "workspace"):
        setattr(b, k, 16)
    lib = _lib.load()
    b.workspace_floats = lib.cc1d_scan_bwd_workspace_floats(ctypes.byref(b)) - 1
    assert lib.cc1d_scan_bwd(ctypes.byref(b), None) == 8
    b.fwd.z = 16  # without a dz
    assert lib.cc1d_scan_bwd(ctypes.byref(b), None) == 1


def test_scan_bwd_without_channels_still_has_dB_and_dC():
    """No channel adds to dB and dC: they are zeros to be written, not buffers to be left as they are."""
    b = _lib.ScanBwdParams()
    b.fwd = _scan(dim=0)
    lib = _lib.load()
    assert lib.cc1d_scan_bwd_workspace_floats(ctypes.byref(b)) == 0
    assert lib.cc1d_scan_bwd(ctypes.byref(b), None) == 1  # nowhere to write them
    b.dB = 16
    assert lib.cc1d_scan_bwd(ctypes.byref(b), None) == 1
    for kw in ({"seqlen": 0}, {"batch": 0}):  # no values of B either
        b.fwd = _scan(dim=0, **kw)
        assert lib.cc1d_scan_bwd(ctypes.byref(b), None) == 0


@pytest.mark.parametrize("code,kw", [(2, {"dtype": 3}), (10, {"dstate": 257}), (11, {"groups": 3}),
                                     (4, {"state_rows": 0}), (1, {}), (0, {"batch": 0}), (0, {"seqlen": 0})])
def test_scan_update_codes(code, kw):
    p = _lib.ScanUpdateParams()
    p.batch, p.dim, p.seqlen, p.dstate, p.groups, p.state_rows, p.dtype = 1, 8, 1, 4, 1, 1, 1
    for k, v in kw.items():
        setattr(p, k, v)
    lib = _lib.load()
    assert lib.cc1d_scan_update(ctypes.byref(p), None) == code
    assert lib.cc1d_scan_update(None, None) == 1


@pytest.mark.parametrize("code,kw", [(2, {"dtype": 3}), (2, {"dtype": 2, "residual_dtype": 1}), (12, {"dim": 0}),
                                     (12, {"dim": 32769}), (4, {"rows": -1}), (1, {}), (0, {"rows": 0})])
def test_norm_codes(code, kw):
    p = _lib.NormParams()
    p.rows, p.dim, p.dtype, p.residual_dtype = 2, 8, 1, 1
    for k, v in kw.items():
        setattr(p, k, v)
    lib = _lib.load()
    assert lib.cc1d_norm_fwd(ctypes.byref(p), None) == code
    b = _lib.NormBwdParams()
    b.fwd = p
    assert (lib.cc1d_norm_bwd_workspace_floats(ctypes.byref(b)) < 0) == (code not in (0, 1))
    assert lib.cc1d_norm_bwd(ctypes.byref(b), None) == (code if code not in (0, 1) else 1)


@pytest.mark.parametrize("L", [0, 1, 100, 255, 256, 257, 511, 512, 513, 4096, 5000])
@pytest.mark.parametrize("N", [1, 16, 40])
def test_tile_states_size_is_the_librarys(L, N):
    lib = _lib.load()
    A = torch.empty(8, N)
    for batch, seqs in ((1, 0), (3, 0), (1, 1), (1, 7)):
        u = torch.empty(batch, 8, L, dtype=torch.bfloat16, device="meta")
        cu = torch.empty(seqs + 1, dtype=torch.int32) if seqs else None
        p = _scan(batch=batch, seqlen=L, dstate=N, num_seqs=seqs, cu_seqlens=16 if seqs else None)
        assert scan_tile_floats(u, A, cu) == lib.cc1d_scan_tile_floats(ctypes.byref(p))


def test_native_host_path_leaves_cpu_tensors_and_odd_arguments_to_python():
    from causal_conv1d_amd import _host

    ext = _host.load()
    p = _bf16()
    args = [p[k] for k in ("u", "delta", "A", "B", "C", "D", "z", "delta_bias")]
    assert ext.ssm_scan(*args, True, None, None, None, False) is NotImplemented
    assert ext.ssm_scan(None, *args[1:], 1, None, None, None, "x") is NotImplemented
    assert ext.ssm_scan_update(args[0], torch.zeros(2, 4, 3), *args[1:], True, None) is NotImplemented
    assert ext.add_norm(torch.zeros(2, 8), torch.ones(8), None, None, 1e-5, False, False) is NotImplemented
    for f, n in ((ext.ssm_scan, 13), (ext.ssm_scan_update, 11), (ext.add_norm, 7), (ext.bind_ssm, 8)):
        with pytest.raises(RuntimeError, match=f"takes {n}"):
            f(None)
