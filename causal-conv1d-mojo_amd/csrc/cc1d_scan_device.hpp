// cc1d_scan_device.hpp -- shared by the kernels of the selective state space scan.
//
// The recurrence h[t] = a[t] h[t-1] + b[t] (a = exp(dt A), b = dt u B) is a
// prefix over pairs (a, b) under (a2, b2) o (a1, b1) = (a2 a1, a2 b1 + b2). A
// wavefront takes one channel's tile of 64 K positions, K consecutive ones per
// lane: each lane runs its K steps from 0, the lanes' pairs are combined over
// the wavefront, and each lane runs its steps again from the state that
// reaches it. The decay over a lane's steps is one exponential, exp(A sum dt).
#pragma once

#include "cc1d_internal.hpp"

namespace cc1d {

// dt = softplus(raw) = max(raw, 0) + log1p(e), e = exp(-|raw|), with
// log1p(e) = 2 atanh(s), s = e / (2 + e) <= 1/3: the odd series up to s^15,
// whose first omitted term is 9^-8 / 17 of the result. Steps are small
// numbers (1e-3 and below), so the relative error counts, and log2(1 + e)
// would lose it. The exponent's rounding (|raw| log2(e) may reach 20) is
// taken back with the product's remainder.
__device__ __forceinline__ float exp_neg(float x) {  // exp(-x), x >= 0
    const float q = -kLog2e * x;
    const float lo = __builtin_fmaf(-kLog2e, x, -q) - 1.9259629911e-8f * x;  // log2(e) - float(log2(e))
    const float e = __builtin_amdgcn_exp2f(q);
    return __builtin_fmaf(e * lo, kLn2, e);
}
__device__ __forceinline__ float softplus(float raw) {
    const float e = exp_neg(fminf(__builtin_fabsf(raw), 80.0f));
    const float s = e * __builtin_amdgcn_rcpf(2.0f + e);
    const float q = s * s;
    float p = __builtin_fmaf(q, 1.0f / 15.0f, 1.0f / 13.0f);
    p = __builtin_fmaf(q, p, 1.0f / 11.0f);
    p = __builtin_fmaf(q, p, 1.0f / 9.0f);
    p = __builtin_fmaf(q, p, 1.0f / 7.0f);
    p = __builtin_fmaf(q, p, 1.0f / 5.0f);
    p = __builtin_fmaf(q, p, 1.0f / 3.0f);
    p = __builtin_fmaf(q, p, 1.0f);
    const float r = __builtin_fmaf(2.0f * s, p, fmaxf(raw, 0.0f));
    return raw != raw ? raw : r;  // min and max drop a NaN
}
__device__ __forceinline__ float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __expf(-x)); }

// A sequence of the scan: positions start .. start + len - 1 of batch row
// `row`; its tiles' states are kept at slots slot, slot + 1, ...
struct ScanSpan {
    int64_t row, start, len, slot;
};

__device__ __forceinline__ int64_t clamp_pos(int64_t v, int64_t n) { return v < 0 ? 0 : (v > n ? n : v); }

// Sequence s. With cu_seqlens sequences have any length, so slot is a bound:
// the sequences before s fill at most start / tile + s tiles.
__device__ __forceinline__ ScanSpan scan_span(const cc1d_scan_params& p, int64_t s, int64_t tile) {
    if (p.cu_seqlens == nullptr) return {s, 0, p.seqlen, s * ((p.seqlen + tile - 1) / tile)};
    const int64_t start = clamp_pos(ld_uniform(p.cu_seqlens + s), p.seqlen);
    const int64_t end = clamp_pos(ld_uniform(p.cu_seqlens + s + 1), p.seqlen);
    return {0, start, end > start ? end - start : 0, start / tile + s};
}

inline int64_t scan_sequences(const cc1d_scan_params& p) { return p.cu_seqlens != nullptr ? p.num_seqs : p.batch; }
inline int64_t scan_slots(const cc1d_scan_params& p, int64_t tile) {
    return p.cu_seqlens != nullptr ? p.seqlen / tile + p.num_seqs : p.batch * ceil_div(p.seqlen, tile);
}

}  // namespace cc1d
