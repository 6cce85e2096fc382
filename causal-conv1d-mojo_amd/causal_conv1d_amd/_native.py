"""Tensor-level wrappers over the C ABI: fill a params struct, launch on the
current HIP stream of the tensors' device.

These replace the reference's ``native_fwd`` / ``native_bwd_full`` /
``native_update`` tuple builders (``fwd/__init__.py:11-60``,
``bwd_full/__init__.py:11-73``, ``update/__init__.py:11-60``). There is one
path only: a ROCm device tensor goes to the HIP kernels; anything else
raises NotImplementedError.
"""

from __future__ import annotations

import ctypes

import torch

from causal_conv1d_amd import _lib
from causal_conv1d_amd._dtype import _DTYPE_CODE


def _require_device(x: torch.Tensor) -> None:
    if x.device.type != "cuda" or torch.version.hip is None:
        raise NotImplementedError(
            f"causal_conv1d_amd runs on ROCm GPUs (MI355X / gfx950) only; got a tensor on {x.device}"
        )


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(x: torch.Tensor) -> int:
    return torch.cuda.current_stream(x.device).cuda_stream


def _set3(arr, t: torch.Tensor | None) -> None:
    if t is not None:
        s = t.stride()
        arr[0], arr[1], arr[2] = s[0], s[1], s[2]


def _set2(arr, t: torch.Tensor | None) -> None:
    if t is not None:
        s = t.stride()
        arr[0], arr[1] = s[0], s[1]


def native_fwd(x, weight, bias, seq_idx, initial_states, out, apply_silu, final_states_out=None) -> None:
    _require_device(x)
    lib = _lib.load()
    p = _lib.FwdParams()
    p.x, p.weight, p.bias = x.data_ptr(), weight.data_ptr(), _ptr(bias)
    p.seq_idx, p.initial_states = _ptr(seq_idx), _ptr(initial_states)
    p.out, p.final_states_out = out.data_ptr(), _ptr(final_states_out)
    p.batch, p.dim, p.seqlen = x.shape
    p.width = weight.shape[1]
    _set3(p.x_stride, x)
    _set2(p.weight_stride, weight)
    p.bias_stride = bias.stride(0) if bias is not None else 0
    _set2(p.seq_idx_stride, seq_idx)
    _set3(p.initial_states_stride, initial_states)
    _set3(p.out_stride, out)
    _set3(p.final_states_stride, final_states_out)
    p.dtype = _DTYPE_CODE[x.dtype]
    p.apply_silu = int(bool(apply_silu))
    _lib.check(lib.cc1d_fwd(ctypes.byref(p), _stream(x)))


def _bwd_params(x, weight, bias, dout, seq_idx, initial_states, dx, dinitial_states, apply_silu, dfinal_states):
    p = _lib.BwdParams()
    p.x, p.weight, p.bias, p.dout = x.data_ptr(), weight.data_ptr(), _ptr(bias), dout.data_ptr()
    p.seq_idx, p.initial_states, p.dfinal_states = _ptr(seq_idx), _ptr(initial_states), _ptr(dfinal_states)
    p.dx = dx.data_ptr()
    p.dinitial_states = _ptr(dinitial_states)
    p.batch, p.dim, p.seqlen = x.shape
    p.width = weight.shape[1]
    _set3(p.x_stride, x)
    _set2(p.weight_stride, weight)
    p.bias_stride = bias.stride(0) if bias is not None else 0
    _set3(p.dout_stride, dout)
    _set2(p.seq_idx_stride, seq_idx)
    _set3(p.initial_states_stride, initial_states)
    _set3(p.dfinal_states_stride, dfinal_states)
    _set3(p.dx_stride, dx)
    _set3(p.dinitial_states_stride, dinitial_states)
    p.dtype = _DTYPE_CODE[x.dtype]
    p.apply_silu = int(bool(apply_silu))
    return p


def native_bwd(x, weight, bias, dout, seq_idx, initial_states, dx, dweight_acc, dbias_acc, dinitial_states,
               apply_silu, dfinal_states=None) -> None:
    """cc1d_bwd: adds the fp32 weight/bias-gradient sums into dweight_acc / dbias_acc."""
    _require_device(x)
    lib = _lib.load()
    p = _bwd_params(x, weight, bias, dout, seq_idx, initial_states, dx, dinitial_states, apply_silu, dfinal_states)
    p.dweight_acc, p.dbias_acc = dweight_acc.data_ptr(), _ptr(dbias_acc)
    _set2(p.dweight_acc_stride, dweight_acc)
    p.dbias_acc_stride = dbias_acc.stride(0) if dbias_acc is not None else 0
    _lib.check(lib.cc1d_bwd(ctypes.byref(p), _stream(x)))


def native_bwd_typed(x, weight, bias, dout, seq_idx, initial_states, dx, dweight, dbias, dinitial_states,
                     apply_silu, dfinal_states=None) -> None:
    """cc1d_bwd_typed: writes dweight / dbias in their dtype from a per-call fp32 workspace."""
    _require_device(x)
    lib = _lib.load()
    p = _bwd_params(x, weight, bias, dout, seq_idx, initial_states, dx, dinitial_states, apply_silu, dfinal_states)
    n = lib.cc1d_bwd_workspace_floats(ctypes.byref(p))
    if n < 0:
        _lib.check(lib.cc1d_bwd_typed(ctypes.byref(p), None, _stream(x)))
    ws = torch.empty(max(n, 1), dtype=torch.float32, device=x.device)
    g = _lib.BwdGrads()
    g.dweight, g.dbias, g.workspace = dweight.data_ptr(), _ptr(dbias), ws.data_ptr()
    _set2(g.dweight_stride, dweight)
    g.dbias_stride = dbias.stride(0) if dbias is not None else 0
    g.workspace_floats = ws.numel()
    _lib.check(lib.cc1d_bwd_typed(ctypes.byref(p), ctypes.byref(g), _stream(x)))


def native_bwd_typed_noalloc(x, weight, bias, dout, seq_idx, initial_states, dx, dweight, dbias, dinitial_states,
                             apply_silu, dfinal_states=None) -> None:
    """cc1d_bwd_typed_noalloc: as native_bwd_typed, with the library's static device scratch
    as the workspace (no allocation at all; calls that overlap on one GPU race)."""
    _require_device(x)
    lib = _lib.load()
    p = _bwd_params(x, weight, bias, dout, seq_idx, initial_states, dx, dinitial_states, apply_silu, dfinal_states)
    g = _lib.BwdGrads()
    g.dweight, g.dbias = dweight.data_ptr(), _ptr(dbias)
    _set2(g.dweight_stride, dweight)
    g.dbias_stride = dbias.stride(0) if dbias is not None else 0
    _lib.check(lib.cc1d_bwd_typed_noalloc(ctypes.byref(p), ctypes.byref(g), _stream(x)))


def native_update(x, weight, bias, conv_state, conv_state_indices, cache_seqlens, out, apply_silu) -> None:
    _require_device(x)
    lib = _lib.load()
    p = _lib.UpdateParams()
    p.x, p.weight, p.bias = x.data_ptr(), weight.data_ptr(), _ptr(bias)
    p.conv_state = conv_state.data_ptr()
    p.conv_state_indices, p.cache_seqlens = _ptr(conv_state_indices), _ptr(cache_seqlens)
    p.out = out.data_ptr()
    p.batch, p.dim, p.seqlen = x.shape
    p.width = weight.shape[1]
    p.state_len = conv_state.shape[2]
    p.state_rows = conv_state.shape[0]
    _set3(p.x_stride, x)
    _set2(p.weight_stride, weight)
    p.bias_stride = bias.stride(0) if bias is not None else 0
    _set3(p.conv_state_stride, conv_state)
    _set3(p.out_stride, out)
    p.dtype = _DTYPE_CODE[x.dtype]
    p.apply_silu = int(bool(apply_silu))
    _lib.check(lib.cc1d_update(ctypes.byref(p), _stream(x)))


def native_varlen_states(x, cu_seqlens, states) -> None:
    _require_device(x)
    lib = _lib.load()
    p = _lib.VarlenParams()
    p.x, p.cu_seqlens, p.states = x.data_ptr(), cu_seqlens.data_ptr(), states.data_ptr()
    p.total_tokens, p.dim = x.shape
    p.batch, _, p.state_len = states.shape
    _set2(p.x_stride, x)
    _set3(p.states_stride, states)
    # a bit-for-bit copy: any element type, by its size
    p.dtype = _DTYPE_CODE.get(x.dtype, 0)
    p.elem_bytes = x.element_size()
    _lib.check(lib.cc1d_varlen_states(ctypes.byref(p), _stream(x)))


def _set4(arr, t: torch.Tensor) -> None:
    arr[0], arr[1], arr[2], arr[3] = t.stride()


def _stride0(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.stride(0)


def _scan_params(u, delta, A, B, C, D, z, delta_bias, seq_idx, cu_seqlens, delta_softplus):
    p = _lib.ScanParams()
    p.u, p.delta, p.z, p.A = u.data_ptr(), delta.data_ptr(), _ptr(z), A.data_ptr()
    p.B, p.C, p.D, p.delta_bias = B.data_ptr(), C.data_ptr(), _ptr(D), _ptr(delta_bias)
    p.seq_idx, p.cu_seqlens = _ptr(seq_idx), _ptr(cu_seqlens)
    p.batch, p.dim, p.seqlen = u.shape
    p.dstate, p.groups = A.shape[1], B.shape[1]
    p.num_seqs = 0 if cu_seqlens is None else cu_seqlens.shape[0] - 1
    _set3(p.u_stride, u)
    _set3(p.delta_stride, delta)
    _set3(p.z_stride, z)
    _set2(p.A_stride, A)
    _set4(p.B_stride, B)
    _set4(p.C_stride, C)
    p.D_stride, p.delta_bias_stride = _stride0(D), _stride0(delta_bias)
    _set2(p.seq_idx_stride, seq_idx)
    p.dtype = _DTYPE_CODE[u.dtype]
    p.delta_softplus = int(delta_softplus)
    return p


def native_scan_fwd(u, delta, A, B, C, D, z, delta_bias, seq_idx, cu_seqlens, initial_states, delta_softplus, out,
                    final_states, tile_states) -> None:
    _require_device(u)
    lib = _lib.load()
    p = _scan_params(u, delta, A, B, C, D, z, delta_bias, seq_idx, cu_seqlens, delta_softplus)
    p.initial_states, p.final_states, p.tile_states = _ptr(initial_states), _ptr(final_states), _ptr(tile_states)
    p.out = out.data_ptr()
    _set3(p.initial_states_stride, initial_states)
    _set3(p.out_stride, out)
    _set3(p.final_states_stride, final_states)
    _lib.check(lib.cc1d_scan_fwd(ctypes.byref(p), _stream(u)))


def native_scan_bwd(u, delta, A, B, C, D, z, delta_bias, seq_idx, cu_seqlens, tile_states, dout, dfinal_states,
                    delta_softplus, du, ddelta, dA, dB, dC, dD, dz, ddelta_bias, dinitial_states) -> None:
    _require_device(u)
    lib = _lib.load()
    b = _lib.ScanBwdParams()
    b.fwd = _scan_params(u, delta, A, B, C, D, z, delta_bias, seq_idx, cu_seqlens, delta_softplus)
    b.fwd.tile_states = tile_states.data_ptr()
    b.dout, b.dfinal_states = dout.data_ptr(), _ptr(dfinal_states)
    b.du, b.ddelta, b.dz = du.data_ptr(), ddelta.data_ptr(), _ptr(dz)
    b.dA, b.dB, b.dC, b.dD = dA.data_ptr(), dB.data_ptr(), dC.data_ptr(), _ptr(dD)
    b.ddelta_bias, b.dinitial_states = _ptr(ddelta_bias), _ptr(dinitial_states)
    _set3(b.dout_stride, dout)
    _set3(b.dfinal_states_stride, dfinal_states)
    _set3(b.du_stride, du)
    _set3(b.ddelta_stride, ddelta)
    _set3(b.dz_stride, dz)
    n = max(0, lib.cc1d_scan_bwd_workspace_floats(ctypes.byref(b)))
    ws = torch.empty(max(n, 1), dtype=torch.float32, device=u.device)
    b.workspace, b.workspace_floats = ws.data_ptr(), ws.numel()
    _lib.check(lib.cc1d_scan_bwd(ctypes.byref(b), _stream(u)))


def native_scan_update(u, ssm_state, delta, A, B, C, D, z, delta_bias, delta_softplus, ssm_state_indices, out) -> None:
    _require_device(u)
    lib = _lib.load()
    p = _lib.ScanUpdateParams()
    p.u, p.delta, p.z, p.A = u.data_ptr(), delta.data_ptr(), _ptr(z), A.data_ptr()
    p.B, p.C, p.D, p.delta_bias = B.data_ptr(), C.data_ptr(), _ptr(D), _ptr(delta_bias)
    p.ssm_state, p.ssm_state_indices, p.out = ssm_state.data_ptr(), _ptr(ssm_state_indices), out.data_ptr()
    p.batch, p.dim, p.seqlen = u.shape
    p.dstate, p.groups, p.state_rows = A.shape[1], B.shape[1], ssm_state.shape[0]
    _set3(p.u_stride, u)
    _set3(p.delta_stride, delta)
    _set3(p.z_stride, z)
    _set2(p.A_stride, A)
    _set4(p.B_stride, B)
    _set4(p.C_stride, C)
    p.D_stride, p.delta_bias_stride = _stride0(D), _stride0(delta_bias)
    _set3(p.ssm_state_stride, ssm_state)
    _set3(p.out_stride, out)
    p.dtype = _DTYPE_CODE[u.dtype]
    p.delta_softplus = int(delta_softplus)
    _lib.check(lib.cc1d_scan_update(ctypes.byref(p), _stream(u)))


def _norm_params(x, weight, residual, rms):
    like = x if x is not None else residual
    p = _lib.NormParams()
    p.x, p.residual, p.weight = _ptr(x), _ptr(residual), weight.data_ptr()
    p.rows, p.dim = like.shape
    p.x_stride, p.residual_stride, p.weight_stride = _stride0(x), _stride0(residual), weight.stride(0)
    p.rms = int(rms)
    return p


def native_norm_fwd(x, weight, bias, residual, eps, rms, y, sum, stats) -> None:
    _require_device(x)
    lib = _lib.load()
    p = _norm_params(x, weight, residual, rms)
    p.bias, p.bias_stride = _ptr(bias), _stride0(bias)
    p.y, p.sum, p.stats = y.data_ptr(), _ptr(sum), _ptr(stats)
    p.y_stride, p.sum_stride = y.stride(0), _stride0(sum)
    p.eps, p.dtype = eps, _DTYPE_CODE[x.dtype]
    p.residual_dtype = p.dtype if residual is None else _DTYPE_CODE[residual.dtype]
    _lib.check(lib.cc1d_norm_fwd(ctypes.byref(p), _stream(x)))


def native_norm_bwd(x, weight, residual, stats, rms, dy, dsum, dx, dresidual, dweight, dbias) -> None:
    _require_device(dy)
    lib = _lib.load()
    b = _lib.NormBwdParams()
    b.fwd = _norm_params(x, weight, residual, rms)
    b.fwd.stats = stats.data_ptr()
    b.fwd.dtype = _DTYPE_CODE[dy.dtype]
    b.fwd.residual_dtype = b.fwd.dtype if residual is None else _DTYPE_CODE[residual.dtype]
    b.dy, b.dsum, b.dx, b.dresidual = dy.data_ptr(), _ptr(dsum), dx.data_ptr(), _ptr(dresidual)
    b.dweight, b.dbias = dweight.data_ptr(), _ptr(dbias)
    b.dy_stride, b.dsum_stride = dy.stride(0), _stride0(dsum)
    b.dx_stride, b.dresidual_stride = dx.stride(0), _stride0(dresidual)
    n = max(0, lib.cc1d_norm_bwd_workspace_floats(ctypes.byref(b)))
    ws = torch.empty(max(n, 1), dtype=torch.float32, device=dy.device)
    b.workspace, b.workspace_floats = ws.data_ptr(), ws.numel()
    _lib.check(lib.cc1d_norm_bwd(ctypes.byref(b), _stream(dy)))
