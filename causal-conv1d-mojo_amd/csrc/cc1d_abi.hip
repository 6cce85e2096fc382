// cc1d_abi.hip -- extern "C" entry points declared in include/cc1d.h.
//
// Validates the plain-pointer arguments, handles zero-size problems, and
// forwards to the kernel launchers on the caller's stream. No allocation, no
// synchronisation, no exceptions across the boundary.
#include "cc1d_internal.hpp"

using namespace cc1d;

namespace {

constexpr int64_t kMaxBlocks = (int64_t)1 << 31;

bool valid_dtype(int32_t d) { return d == CC1D_DTYPE_FP16 || d == CC1D_DTYPE_BF16 || d == CC1D_DTYPE_FP32; }
bool valid_width(int64_t w) { return w >= 2 && w <= 9; }
int esize(int32_t d) { return d == CC1D_DTYPE_FP32 ? 4 : 2; }

// Every launcher uses at most one thread per element of the largest tensor
// it touches; refuse problems whose grids would not fit.
bool grid_fits(int64_t threads) { return threads / 256 + 1 < kMaxBlocks; }

// Shared by cc1d_bwd_typed and cc1d_bwd_typed_noalloc (which ignores the workspace).
int bwd_typed_entry(const cc1d_bwd_params* p, const cc1d_bwd_grads* g, void* stream, bool noalloc) {
    if (p == nullptr || g == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!valid_dtype(p->dtype)) return CC1D_ERR_DTYPE;
    if (!valid_width(p->width)) return CC1D_ERR_WIDTH;
    if (p->batch < 0 || p->dim < 0 || p->seqlen < 0) return CC1D_ERR_SHAPE;
    if (p->seq_idx != nullptr &&
        (p->initial_states != nullptr || p->dfinal_states != nullptr || p->dinitial_states != nullptr))
        return CC1D_ERR_EXCLUSIVE;
    if (p->initial_states != nullptr && p->dinitial_states == nullptr) return CC1D_ERR_NULL_POINTER;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (p->dim == 0) return CC1D_OK;
    if (g->dweight == nullptr) return CC1D_ERR_NULL_POINTER;
    if (p->batch == 0 || p->seqlen == 0) {
        // no positions: the gradients are sums over no terms
        const int64_t ws[3] = {0, g->dweight_stride[0], g->dweight_stride[1]};
        int st = launch_zero3(g->dweight, esize(p->dtype), 1, p->dim, p->width, ws, s);
        if (st == CC1D_OK && g->dbias != nullptr) {
            const int64_t bs[3] = {0, g->dbias_stride, 0};
            st = launch_zero3(g->dbias, esize(p->dtype), 1, p->dim, 1, bs, s);
        }
        if (st == CC1D_OK && p->dinitial_states != nullptr && p->batch > 0)
            st = launch_zero3(p->dinitial_states, esize(p->dtype), p->batch, p->dim, p->width - 1,
                              p->dinitial_states_stride, s);
        return st;
    }
    if (!grid_fits(p->batch * p->dim * p->seqlen)) return CC1D_ERR_SHAPE;
    if (p->x == nullptr || p->weight == nullptr || p->dout == nullptr || p->dx == nullptr)
        return CC1D_ERR_NULL_POINTER;
    // (a NULL workspace is refused by the launcher when the call needs one)
    if (noalloc) return launch_bwd_typed_noalloc(*p, *g, s);
    return launch_bwd_typed(*p, *g, s);
}

// Sizes and options of a scan, before its pointers.
int check_scan(const cc1d_scan_params& p) {
    if (!valid_dtype(p.dtype)) return CC1D_ERR_DTYPE;
    if (p.dstate < 1 || p.dstate > CC1D_MAX_DSTATE) return CC1D_ERR_DSTATE;
    if (p.batch < 0 || p.dim < 0 || p.seqlen < 0) return CC1D_ERR_SHAPE;
    if (p.groups < 1 || p.dim % p.groups != 0) return CC1D_ERR_GROUPS;
    if (p.seq_idx != nullptr &&
        (p.initial_states != nullptr || p.final_states != nullptr || p.cu_seqlens != nullptr))
        return CC1D_ERR_EXCLUSIVE;
    if (p.cu_seqlens != nullptr && (p.batch != 1 || p.num_seqs < 0 || (p.num_seqs == 0 && p.seqlen > 0)))
        return CC1D_ERR_SHAPE;
    const int64_t seqs = p.cu_seqlens != nullptr ? p.num_seqs : p.batch;
    // a block per sequence and channel at most, a thread per value of dB and dC, 32-bit positions (launches check
    // their threads, which depend on the kernel)
    const double blocks = (double)seqs * (double)p.dim;
    const double values = (double)p.batch * (double)p.groups * (double)p.dstate * (double)p.seqlen;
    if (blocks >= (double)kMaxBlocks || values / 256 + 1 >= (double)kMaxBlocks || p.seqlen >= ((int64_t)1 << 31) - 4096)
        return CC1D_ERR_SHAPE;
    return CC1D_OK;
}

bool scan_empty(const cc1d_scan_params& p) {
    return p.dim == 0 || (p.cu_seqlens != nullptr ? p.num_seqs == 0 : p.batch == 0);
}

int check_norm(const cc1d_norm_params& p) {
    if (!valid_dtype(p.dtype) || (p.residual_dtype != p.dtype && p.residual_dtype != CC1D_DTYPE_FP32))
        return CC1D_ERR_DTYPE;
    if (p.rows < 0 || p.rows >= kMaxBlocks) return CC1D_ERR_SHAPE;
    if (p.dim < 1 || p.dim > CC1D_MAX_NORM_DIM) return CC1D_ERR_NORM_DIM;
    return CC1D_OK;
}

}  // namespace

extern "C" {

int cc1d_abi_version(void) { return CC1D_ABI_VERSION; }

const char* cc1d_strerror(int status) {
    switch (status) {
    case CC1D_OK: return "ok";
    case CC1D_ERR_NULL_POINTER: return "a required pointer is NULL";
    case CC1D_ERR_DTYPE: return "unsupported dtype code (expected 0=fp16, 1=bf16, 2=fp32) or element size";
    case CC1D_ERR_WIDTH: return "width must be in 2..9";
    case CC1D_ERR_SHAPE: return "invalid or too large shape";
    case CC1D_ERR_EXCLUSIVE: return "seq_idx is mutually exclusive with initial_states and final_states (in a scan also with cu_seqlens)";
    case CC1D_ERR_STATE_LEN: return "conv_state length must be >= width - 1";
    case CC1D_ERR_LAUNCH: return "kernel launch failed";
    case CC1D_ERR_WORKSPACE: return "workspace smaller than the entry point's *_workspace_floats()";
    case CC1D_ERR_SCRATCH_LIMIT:
        return "problem needs more workspace than the static scratch of cc1d_bwd_typed_noalloc "
               "(CC1D_NOALLOC_WORKSPACE_FLOATS floats)";
    case CC1D_ERR_DSTATE: return "dstate must be in 1..256";
    case CC1D_ERR_GROUPS: return "dim must be a multiple of groups";
    case CC1D_ERR_NORM_DIM: return "norm dim must be in 1..32768";
    default: return "unknown status";
    }
}

int cc1d_fwd(const cc1d_fwd_params* p, void* stream) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!valid_dtype(p->dtype)) return CC1D_ERR_DTYPE;
    if (!valid_width(p->width)) return CC1D_ERR_WIDTH;
    if (p->batch < 0 || p->dim < 0 || p->seqlen < 0) return CC1D_ERR_SHAPE;
    if (p->seq_idx != nullptr && (p->initial_states != nullptr || p->final_states_out != nullptr))
        return CC1D_ERR_EXCLUSIVE;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (p->batch == 0 || p->dim == 0) return CC1D_OK;
    if (!grid_fits(p->batch * p->dim * (p->seqlen > 0 ? p->seqlen : 1))) return CC1D_ERR_SHAPE;
    if (p->seqlen == 0) {
        if (p->final_states_out == nullptr) return CC1D_OK;
        return launch_zero3(p->final_states_out, esize(p->dtype), p->batch, p->dim, p->width - 1,
                            p->final_states_stride, s);
    }
    if (p->x == nullptr || p->weight == nullptr || p->out == nullptr) return CC1D_ERR_NULL_POINTER;
    return launch_fwd(*p, s);
}

int cc1d_bwd(const cc1d_bwd_params* p, void* stream) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!valid_dtype(p->dtype)) return CC1D_ERR_DTYPE;
    if (!valid_width(p->width)) return CC1D_ERR_WIDTH;
    if (p->batch < 0 || p->dim < 0 || p->seqlen < 0) return CC1D_ERR_SHAPE;
    if (p->seq_idx != nullptr &&
        (p->initial_states != nullptr || p->dfinal_states != nullptr || p->dinitial_states != nullptr))
        return CC1D_ERR_EXCLUSIVE;
    if (p->initial_states != nullptr && p->dinitial_states == nullptr) return CC1D_ERR_NULL_POINTER;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    if (p->batch == 0 || p->dim == 0) return CC1D_OK;
    if (!grid_fits(p->batch * p->dim * (p->seqlen > 0 ? p->seqlen : 1))) return CC1D_ERR_SHAPE;
    if (p->seqlen == 0) {
        // no positions: dx is empty, the accumulators receive nothing and
        // dinitial_states (a sum over no terms) is zero
        if (p->dinitial_states == nullptr) return CC1D_OK;
        return launch_zero3(p->dinitial_states, esize(p->dtype), p->batch, p->dim, p->width - 1,
                            p->dinitial_states_stride, s);
    }
    if (p->x == nullptr || p->weight == nullptr || p->dout == nullptr || p->dx == nullptr ||
        p->dweight_acc == nullptr)
        return CC1D_ERR_NULL_POINTER;
    return launch_bwd(*p, s);
}

int64_t cc1d_bwd_workspace_floats(const cc1d_bwd_params* p) {
    if (p == nullptr || !valid_dtype(p->dtype) || !valid_width(p->width)) return -1;
    if (p->batch <= 0 || p->dim <= 0 || p->seqlen <= 0) return 0;
    return bwd_workspace_floats(*p);
}

int cc1d_bwd_typed(const cc1d_bwd_params* p, const cc1d_bwd_grads* g, void* stream) {
    return bwd_typed_entry(p, g, stream, false);
}

int cc1d_bwd_typed_noalloc(const cc1d_bwd_params* p, const cc1d_bwd_grads* g, void* stream) {
    return bwd_typed_entry(p, g, stream, true);
}

int cc1d_update(const cc1d_update_params* p, void* stream) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!valid_dtype(p->dtype)) return CC1D_ERR_DTYPE;
    if (!valid_width(p->width)) return CC1D_ERR_WIDTH;
    if (p->batch < 0 || p->dim < 0 || p->seqlen < 0 || p->state_len < 0 || p->state_rows < 0)
        return CC1D_ERR_SHAPE;
    if (p->state_len < p->width - 1) return CC1D_ERR_STATE_LEN;
    if (p->conv_state_indices == nullptr && p->state_rows < p->batch) return CC1D_ERR_SHAPE;
    if (p->batch == 0 || p->dim == 0 || p->seqlen == 0) return CC1D_OK;
    if (!grid_fits(p->batch * p->dim)) return CC1D_ERR_SHAPE;
    if (p->x == nullptr || p->weight == nullptr || p->conv_state == nullptr || p->out == nullptr)
        return CC1D_ERR_NULL_POINTER;
    return launch_update(*p, static_cast<hipStream_t>(stream));
}

int cc1d_varlen_states(const cc1d_varlen_params* p, void* stream) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    if (p->elem_bytes == 0 ? !valid_dtype(p->dtype)
                           : (p->elem_bytes != 1 && p->elem_bytes != 2 && p->elem_bytes != 4 && p->elem_bytes != 8 &&
                              p->elem_bytes != 16))
        return CC1D_ERR_DTYPE;
    if (p->total_tokens < 0 || p->dim < 0 || p->batch < 0 || p->state_len < 0) return CC1D_ERR_SHAPE;
    if (p->batch == 0 || p->dim == 0 || p->state_len == 0) return CC1D_OK;
    if (!grid_fits(p->batch * p->dim * p->state_len)) return CC1D_ERR_SHAPE;
    if (p->cu_seqlens == nullptr || p->states == nullptr || (p->x == nullptr && p->total_tokens > 0))
        return CC1D_ERR_NULL_POINTER;
    return launch_varlen_states(*p, static_cast<hipStream_t>(stream));
}

int cc1d_scan_fwd(const cc1d_scan_params* p, void* stream) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    const int st = check_scan(*p);
    if (st != CC1D_OK) return st;
    if (scan_empty(*p)) return CC1D_OK;
    // without positions only the states are read and written
    if (p->seqlen == 0 && p->final_states == nullptr) return CC1D_OK;
    if (p->A == nullptr) return CC1D_ERR_NULL_POINTER;
    if (p->seqlen > 0 && (p->u == nullptr || p->delta == nullptr || p->B == nullptr || p->C == nullptr || p->out == nullptr))
        return CC1D_ERR_NULL_POINTER;
    return launch_scan_fwd(*p, static_cast<hipStream_t>(stream));
}

int64_t cc1d_scan_tile_floats(const cc1d_scan_params* p) {
    if (p == nullptr || check_scan(*p) != CC1D_OK) return -1;
    return scan_empty(*p) ? 0 : scan_tile_floats(*p);
}

int cc1d_scan_bwd(const cc1d_scan_bwd_params* b, void* stream) {
    if (b == nullptr) return CC1D_ERR_NULL_POINTER;
    const cc1d_scan_params& p = b->fwd;
    const int st = check_scan(p);
    if (st != CC1D_OK) return st;
    if (p.seq_idx != nullptr && (b->dfinal_states != nullptr || b->dinitial_states != nullptr)) return CC1D_ERR_EXCLUSIVE;
    if (p.dim == 0) {  // no channel adds to dB and dC
        const int64_t rows = p.batch * p.groups, strides[3] = {p.dstate * p.seqlen, p.seqlen, 1};
        if (rows * p.seqlen > 0 && (b->dB == nullptr || b->dC == nullptr)) return CC1D_ERR_NULL_POINTER;
        const hipStream_t s = static_cast<hipStream_t>(stream);
        const int zeroed = launch_zero3(b->dB, esize(p.dtype), rows, p.dstate, p.seqlen, strides, s);
        return zeroed != CC1D_OK ? zeroed : launch_zero3(b->dC, esize(p.dtype), rows, p.dstate, p.seqlen, strides, s);
    }
    if (b->dA == nullptr || p.A == nullptr) return CC1D_ERR_NULL_POINTER;
    if (p.batch * p.seqlen > 0 &&
        (p.u == nullptr || p.delta == nullptr || p.B == nullptr || p.C == nullptr || p.tile_states == nullptr ||
         b->dout == nullptr || b->du == nullptr || b->ddelta == nullptr || b->dB == nullptr || b->dC == nullptr ||
         (p.z != nullptr && b->dz == nullptr)))
        return CC1D_ERR_NULL_POINTER;
    const int64_t need = scan_empty(p) ? 0 : scan_bwd_workspace_floats(*b);
    if (b->workspace_floats < need) return CC1D_ERR_WORKSPACE;
    if (need > 0 && b->workspace == nullptr) return CC1D_ERR_NULL_POINTER;
    return launch_scan_bwd(*b, static_cast<hipStream_t>(stream));
}

int64_t cc1d_scan_bwd_workspace_floats(const cc1d_scan_bwd_params* b) {
    if (b == nullptr || check_scan(b->fwd) != CC1D_OK) return -1;
    return scan_empty(b->fwd) ? 0 : scan_bwd_workspace_floats(*b);
}

int cc1d_scan_update(const cc1d_scan_update_params* p, void* stream) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    if (!valid_dtype(p->dtype)) return CC1D_ERR_DTYPE;
    if (p->dstate < 1 || p->dstate > CC1D_MAX_DSTATE) return CC1D_ERR_DSTATE;
    if (p->batch < 0 || p->dim < 0 || p->seqlen < 0 || p->state_rows < 0) return CC1D_ERR_SHAPE;
    if (p->groups < 1 || p->dim % p->groups != 0) return CC1D_ERR_GROUPS;
    if (p->ssm_state_indices == nullptr && p->state_rows < p->batch) return CC1D_ERR_SHAPE;
    if (p->batch == 0 || p->dim == 0 || p->seqlen == 0) return CC1D_OK;
    if ((double)p->batch * (double)p->dim >= (double)kMaxBlocks) return CC1D_ERR_SHAPE;  // a block per channel at most
    if (p->u == nullptr || p->delta == nullptr || p->A == nullptr || p->B == nullptr || p->C == nullptr ||
        p->out == nullptr || (p->ssm_state == nullptr && p->state_rows > 0))
        return CC1D_ERR_NULL_POINTER;
    return launch_scan_update(*p, static_cast<hipStream_t>(stream));
}

int cc1d_norm_fwd(const cc1d_norm_params* p, void* stream) {
    if (p == nullptr) return CC1D_ERR_NULL_POINTER;
    const int st = check_norm(*p);
    if (st != CC1D_OK) return st;
    if (p->rows == 0) return CC1D_OK;
    if (p->x == nullptr || p->weight == nullptr || p->y == nullptr) return CC1D_ERR_NULL_POINTER;
    return launch_norm_fwd(*p, static_cast<hipStream_t>(stream));
}

int cc1d_norm_bwd(const cc1d_norm_bwd_params* b, void* stream) {
    if (b == nullptr) return CC1D_ERR_NULL_POINTER;
    const cc1d_norm_params& p = b->fwd;
    const int st = check_norm(p);
    if (st != CC1D_OK) return st;
    if (b->dweight == nullptr || p.weight == nullptr) return CC1D_ERR_NULL_POINTER;
    if (p.rows > 0 && ((p.x == nullptr && p.residual == nullptr) || p.stats == nullptr || b->dy == nullptr ||
                       b->dx == nullptr || b->workspace == nullptr))
        return CC1D_ERR_NULL_POINTER;
    if (b->workspace_floats < norm_bwd_workspace_floats(*b)) return CC1D_ERR_WORKSPACE;
    return launch_norm_bwd(*b, static_cast<hipStream_t>(stream));
}

int64_t cc1d_norm_bwd_workspace_floats(const cc1d_norm_bwd_params* b) {
    if (b == nullptr || check_norm(b->fwd) != CC1D_OK) return -1;
    return norm_bwd_workspace_floats(*b);
}

}  // extern "C"
