"""ctypes binding of ``libcc1d_amd.so`` (the C ABI in ``include/cc1d.h``).

The structures below mirror ``cc1d_fwd_params`` / ``cc1d_bwd_params`` /
``cc1d_bwd_grads`` / ``cc1d_update_params`` / ``cc1d_varlen_params`` and the
params of the scan, the norm, linear attention and the rotation field for field. The library
is loaded on first use; a missing or stale build raises instead of falling
back to anything else.
"""

from __future__ import annotations

import ctypes
import os
import sys
from pathlib import Path

_LIB_PATH = Path(__file__).resolve().parent / "_lib" / "libcc1d_amd.so"
ABI_VERSION = 3
# fp32 elements of the static device scratch of cc1d_bwd_typed_noalloc (CC1D_NOALLOC_WORKSPACE_FLOATS)
NOALLOC_WORKSPACE_FLOATS = 1 << 21

_i64 = ctypes.c_int64
_i32 = ctypes.c_int32
_vp = ctypes.c_void_p
_i64x2 = _i64 * 2
_i64x3 = _i64 * 3


class FwdParams(ctypes.Structure):
    _fields_ = [
        ("x", _vp), ("weight", _vp), ("bias", _vp), ("seq_idx", _vp), ("initial_states", _vp),
        ("out", _vp), ("final_states_out", _vp),
        ("batch", _i64), ("dim", _i64), ("seqlen", _i64), ("width", _i64),
        ("x_stride", _i64x3), ("weight_stride", _i64x2), ("bias_stride", _i64),
        ("seq_idx_stride", _i64x2), ("initial_states_stride", _i64x3), ("out_stride", _i64x3),
        ("final_states_stride", _i64x3),
        ("dtype", _i32), ("apply_silu", _i32),
    ]


class BwdParams(ctypes.Structure):
    _fields_ = [
        ("x", _vp), ("weight", _vp), ("bias", _vp), ("dout", _vp), ("seq_idx", _vp),
        ("initial_states", _vp), ("dfinal_states", _vp),
        ("dx", _vp), ("dweight_acc", _vp), ("dbias_acc", _vp), ("dinitial_states", _vp),
        ("batch", _i64), ("dim", _i64), ("seqlen", _i64), ("width", _i64),
        ("x_stride", _i64x3), ("weight_stride", _i64x2), ("bias_stride", _i64), ("dout_stride", _i64x3),
        ("seq_idx_stride", _i64x2), ("initial_states_stride", _i64x3), ("dfinal_states_stride", _i64x3),
        ("dx_stride", _i64x3), ("dweight_acc_stride", _i64x2), ("dbias_acc_stride", _i64),
        ("dinitial_states_stride", _i64x3),
        ("dtype", _i32), ("apply_silu", _i32),
    ]


class BwdGrads(ctypes.Structure):
    _fields_ = [
        ("dweight", _vp), ("dbias", _vp), ("workspace", _vp),
        ("dweight_stride", _i64x2), ("dbias_stride", _i64), ("workspace_floats", _i64),
    ]


class UpdateParams(ctypes.Structure):
    _fields_ = [
        ("x", _vp), ("weight", _vp), ("bias", _vp), ("conv_state", _vp), ("conv_state_indices", _vp),
        ("cache_seqlens", _vp), ("out", _vp),
        ("batch", _i64), ("dim", _i64), ("seqlen", _i64), ("width", _i64), ("state_len", _i64),
        ("state_rows", _i64),
        ("x_stride", _i64x3), ("weight_stride", _i64x2), ("bias_stride", _i64),
        ("conv_state_stride", _i64x3), ("out_stride", _i64x3),
        ("dtype", _i32), ("apply_silu", _i32),
    ]


class VarlenParams(ctypes.Structure):
    _fields_ = [
        ("x", _vp), ("cu_seqlens", _vp), ("states", _vp),
        ("total_tokens", _i64), ("dim", _i64), ("batch", _i64), ("state_len", _i64),
        ("x_stride", _i64x2), ("states_stride", _i64x3),
        ("dtype", _i32), ("elem_bytes", _i32),
    ]


_i64x4 = _i64 * 4


class ScanParams(ctypes.Structure):
    _fields_ = [
        ("u", _vp), ("delta", _vp), ("z", _vp), ("A", _vp), ("B", _vp), ("C", _vp), ("D", _vp),
        ("delta_bias", _vp), ("seq_idx", _vp), ("cu_seqlens", _vp), ("initial_states", _vp),
        ("out", _vp), ("final_states", _vp), ("tile_states", _vp),
        ("batch", _i64), ("dim", _i64), ("seqlen", _i64), ("dstate", _i64), ("groups", _i64), ("num_seqs", _i64),
        ("u_stride", _i64x3), ("delta_stride", _i64x3), ("z_stride", _i64x3), ("A_stride", _i64x2),
        ("B_stride", _i64x4), ("C_stride", _i64x4), ("D_stride", _i64), ("delta_bias_stride", _i64),
        ("seq_idx_stride", _i64x2), ("initial_states_stride", _i64x3), ("out_stride", _i64x3),
        ("final_states_stride", _i64x3),
        ("dtype", _i32), ("delta_softplus", _i32),
    ]


class ScanBwdParams(ctypes.Structure):
    _fields_ = [
        ("fwd", ScanParams), ("dout", _vp), ("dfinal_states", _vp), ("du", _vp), ("ddelta", _vp), ("dz", _vp),
        ("dA", _vp), ("dB", _vp), ("dC", _vp), ("dD", _vp), ("ddelta_bias", _vp), ("dinitial_states", _vp),
        ("workspace", _vp), ("workspace_floats", _i64),
        ("dout_stride", _i64x3), ("dfinal_states_stride", _i64x3), ("du_stride", _i64x3),
        ("ddelta_stride", _i64x3), ("dz_stride", _i64x3),
    ]


class ScanUpdateParams(ctypes.Structure):
    _fields_ = [
        ("u", _vp), ("delta", _vp), ("z", _vp), ("A", _vp), ("B", _vp), ("C", _vp), ("D", _vp),
        ("delta_bias", _vp), ("ssm_state", _vp), ("ssm_state_indices", _vp), ("out", _vp),
        ("batch", _i64), ("dim", _i64), ("seqlen", _i64), ("dstate", _i64), ("groups", _i64), ("state_rows", _i64),
        ("u_stride", _i64x3), ("delta_stride", _i64x3), ("z_stride", _i64x3), ("A_stride", _i64x2),
        ("B_stride", _i64x4), ("C_stride", _i64x4), ("D_stride", _i64), ("delta_bias_stride", _i64),
        ("ssm_state_stride", _i64x3), ("out_stride", _i64x3),
        ("dtype", _i32), ("delta_softplus", _i32),
    ]


class NormParams(ctypes.Structure):
    _fields_ = [
        ("x", _vp), ("residual", _vp), ("weight", _vp), ("bias", _vp), ("y", _vp), ("sum", _vp), ("stats", _vp),
        ("rows", _i64), ("dim", _i64),
        ("x_stride", _i64), ("residual_stride", _i64), ("weight_stride", _i64), ("bias_stride", _i64),
        ("y_stride", _i64), ("sum_stride", _i64),
        ("eps", ctypes.c_double), ("dtype", _i32), ("residual_dtype", _i32), ("rms", _i32),
    ]


class NormBwdParams(ctypes.Structure):
    _fields_ = [
        ("fwd", NormParams), ("dy", _vp), ("dsum", _vp), ("dx", _vp), ("dresidual", _vp), ("dweight", _vp),
        ("dbias", _vp), ("workspace", _vp), ("workspace_floats", _i64),
        ("dy_stride", _i64), ("dsum_stride", _i64), ("dx_stride", _i64), ("dresidual_stride", _i64),
    ]


class AttnParams(ctypes.Structure):
    _fields_ = [
        ("q", _vp), ("k", _vp), ("v", _vp), ("g", _vp), ("cu_seqlens", _vp), ("initial_states", _vp),
        ("out", _vp), ("final_states", _vp), ("workspace", _vp), ("workspace_floats", _i64),
        ("batch", _i64), ("seqlen", _i64), ("heads", _i64), ("key_heads", _i64), ("dk", _i64), ("dv", _i64),
        ("num_seqs", _i64),
        ("q_stride", _i64x4), ("k_stride", _i64x4), ("v_stride", _i64x4), ("g_stride", _i64x3),
        ("initial_states_stride", _i64x4),
        ("scale", ctypes.c_double), ("dtype", _i32),
    ]


class AttnBwdParams(ctypes.Structure):
    _fields_ = [
        ("fwd", AttnParams), ("dout", _vp), ("dfinal_states", _vp), ("dq", _vp), ("dk", _vp), ("dv", _vp),
        ("dg", _vp), ("dinitial_states", _vp), ("workspace", _vp), ("workspace_floats", _i64),
        ("dout_stride", _i64x4), ("dfinal_states_stride", _i64x4),
    ]


class AttnUpdateParams(ctypes.Structure):
    _fields_ = [
        ("q", _vp), ("k", _vp), ("v", _vp), ("g", _vp), ("attn_state", _vp), ("attn_state_indices", _vp), ("out", _vp),
        ("batch", _i64), ("tokens", _i64), ("heads", _i64), ("key_heads", _i64), ("dk", _i64), ("dv", _i64),
        ("state_rows", _i64),
        ("q_stride", _i64x4), ("k_stride", _i64x4), ("v_stride", _i64x4), ("g_stride", _i64x3),
        ("attn_state_stride", _i64x4),
        ("scale", ctypes.c_double), ("dtype", _i32),
    ]


class RotaryParams(ctypes.Structure):
    _fields_ = [
        ("q", _vp), ("k", _vp), ("q_weight", _vp), ("k_weight", _vp), ("inv_freq", _vp), ("positions", _vp),
        ("q_out", _vp), ("k_out", _vp),
        ("batch", _i64), ("seqlen", _i64), ("q_heads", _i64), ("k_heads", _i64), ("dim", _i64), ("rotated", _i64),
        ("q_stride", _i64x4), ("k_stride", _i64x4), ("positions_stride", _i64x2),
        ("eps", ctypes.c_double), ("amplitude", ctypes.c_double),
        ("dtype", _i32), ("positions_bytes", _i32), ("interleaved", _i32),
    ]


class RotaryBwdParams(ctypes.Structure):
    _fields_ = [
        ("fwd", RotaryParams), ("dq_out", _vp), ("dk_out", _vp), ("dq", _vp), ("dk", _vp), ("dq_weight", _vp),
        ("dk_weight", _vp), ("workspace", _vp), ("workspace_floats", _i64),
        ("dq_out_stride", _i64x4), ("dk_out_stride", _i64x4),
    ]


EXPORTED_SYMBOLS = (
    "cc1d_abi_version",
    "cc1d_strerror",
    "cc1d_fwd",
    "cc1d_bwd",
    "cc1d_bwd_workspace_floats",
    "cc1d_bwd_typed",
    "cc1d_bwd_typed_noalloc",
    "cc1d_update",
    "cc1d_varlen_states",
    "cc1d_scan_fwd",
    "cc1d_scan_tile_floats",
    "cc1d_scan_bwd",
    "cc1d_scan_bwd_workspace_floats",
    "cc1d_scan_update",
    "cc1d_norm_fwd",
    "cc1d_norm_bwd",
    "cc1d_norm_bwd_workspace_floats",
    "cc1d_attn_fwd",
    "cc1d_attn_workspace_floats",
    "cc1d_attn_bwd",
    "cc1d_attn_bwd_workspace_floats",
    "cc1d_attn_update",
    "cc1d_rotary_fwd",
    "cc1d_rotary_bwd",
    "cc1d_rotary_bwd_workspace_floats",
)

_lib = None


def library_path() -> Path:
    """The in-tree library; CC1D_AMD_LIB may name another build of it (announced on
    stderr when the library is loaded, so a stray variable cannot go unnoticed)."""
    return Path(os.environ.get("CC1D_AMD_LIB", _LIB_PATH))


def load():
    """Load and type the shared library (cached). Raises if it is missing."""
    global _lib
    if _lib is not None:
        return _lib
    path = library_path()
    if not path.exists():
        raise RuntimeError(
            f"causal_conv1d_amd: native library {path} is not built; "
            "run `python causal-conv1d-mojo_amd/csrc/build.py`"
        )
    if path.resolve() != _LIB_PATH.resolve():
        print(f"causal_conv1d_amd: loading {path} (CC1D_AMD_LIB), not the in-tree {_LIB_PATH}",
              file=sys.stderr, flush=True)
    lib = ctypes.CDLL(str(path))
    lib.cc1d_abi_version.restype = ctypes.c_int
    lib.cc1d_abi_version.argtypes = []
    lib.cc1d_strerror.restype = ctypes.c_char_p
    lib.cc1d_strerror.argtypes = [ctypes.c_int]
    for name, st in (("cc1d_fwd", FwdParams), ("cc1d_bwd", BwdParams), ("cc1d_update", UpdateParams),
                     ("cc1d_varlen_states", VarlenParams), ("cc1d_scan_fwd", ScanParams),
                     ("cc1d_scan_bwd", ScanBwdParams), ("cc1d_scan_update", ScanUpdateParams),
                     ("cc1d_norm_fwd", NormParams), ("cc1d_norm_bwd", NormBwdParams),
                     ("cc1d_attn_fwd", AttnParams), ("cc1d_attn_bwd", AttnBwdParams),
                     ("cc1d_attn_update", AttnUpdateParams), ("cc1d_rotary_fwd", RotaryParams),
                     ("cc1d_rotary_bwd", RotaryBwdParams)):
        fn = getattr(lib, name)
        fn.restype = ctypes.c_int
        fn.argtypes = [ctypes.POINTER(st), _vp]
    for name, st in (("cc1d_bwd_workspace_floats", BwdParams), ("cc1d_scan_tile_floats", ScanParams),
                     ("cc1d_scan_bwd_workspace_floats", ScanBwdParams),
                     ("cc1d_norm_bwd_workspace_floats", NormBwdParams),
                     ("cc1d_attn_workspace_floats", AttnParams),
                     ("cc1d_attn_bwd_workspace_floats", AttnBwdParams),
                     ("cc1d_rotary_bwd_workspace_floats", RotaryBwdParams)):
        fn = getattr(lib, name)
        fn.restype = ctypes.c_int64
        fn.argtypes = [ctypes.POINTER(st)]
    for name in ("cc1d_bwd_typed", "cc1d_bwd_typed_noalloc"):
        fn = getattr(lib, name)
        fn.restype = ctypes.c_int
        fn.argtypes = [ctypes.POINTER(BwdParams), ctypes.POINTER(BwdGrads), _vp]
    got = lib.cc1d_abi_version()
    if got != ABI_VERSION:
        raise RuntimeError(f"causal_conv1d_amd: ABI version mismatch (library {got}, bindings {ABI_VERSION})")
    _lib = lib
    return lib


def check(status: int) -> None:
    if status != 0:
        msg = load().cc1d_strerror(status).decode()
        raise RuntimeError(f"causal_conv1d_amd native call failed: {msg} (status {status})")
