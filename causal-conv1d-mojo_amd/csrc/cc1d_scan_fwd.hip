// cc1d_scan_fwd.hip -- forward of the selective state space scan.
#include "cc1d_scan_device.hpp"

namespace cc1d {
namespace {

constexpr int K = 4;          // positions per lane
constexpr int TILE = 64 * K;  // positions per wavefront and step

// The positions of batch row 0 that no sequence covers: before the first and after the last.
template <typename T> __device__ void zero_uncovered(const cc1d_scan_params& p, int64_t s, int64_t d, const ScanSpan& q) {
    T* out = static_cast<T*>(p.out) + d * p.out_stride[1];
    if (s == 0)
        for (int64_t t = threadIdx.x; t < q.start; t += 64) out[t * p.out_stride[2]] = T{};
    if (s == p.num_seqs - 1)
        for (int64_t t = q.start + q.len + threadIdx.x; t < p.seqlen; t += 64) out[t * p.out_stride[2]] = T{};
}

// One wavefront per (sequence, channel), every layout.
template <typename T> __global__ void __launch_bounds__(64) scan_fwd_kernel(const cc1d_scan_params p) {
    __shared__ float carry[CC1D_MAX_DSTATE];
    const int lane = threadIdx.x;
    const int64_t s = blockIdx.x / p.dim, d = blockIdx.x % p.dim;
    const ScanSpan q = scan_span(p, s, TILE);
    if (p.cu_seqlens != nullptr) zero_uncovered<T>(p, s, d, q);
    const T* u = static_cast<const T*>(p.u) + q.row * p.u_stride[0] + d * p.u_stride[1];
    const T* delta = static_cast<const T*>(p.delta) + q.row * p.delta_stride[0] + d * p.delta_stride[1];
    const T* z = p.z ? static_cast<const T*>(p.z) + q.row * p.z_stride[0] + d * p.z_stride[1] : nullptr;
    T* out = static_cast<T*>(p.out) + q.row * p.out_stride[0] + d * p.out_stride[1];
    const int64_t g = d / (p.dim / p.groups);
    const T* Bp = static_cast<const T*>(p.B) + q.row * p.B_stride[0] + g * p.B_stride[1];
    const T* Cp = static_cast<const T*>(p.C) + q.row * p.C_stride[0] + g * p.C_stride[1];
    const int32_t* ids = p.seq_idx ? p.seq_idx + q.row * p.seq_idx_stride[0] : nullptr;
    const float bias = p.delta_bias ? p.delta_bias[d * p.delta_bias_stride] : 0.0f;
    const float skip = p.D ? p.D[d * p.D_stride] : 0.0f;
    const int N = (int)p.dstate;
    for (int n = lane; n < N; n += 64)
        carry[n] = p.initial_states ? p.initial_states[s * p.initial_states_stride[0] + d * p.initial_states_stride[1] +
                                                       n * p.initial_states_stride[2]]
                                    : 0.0f;
    __syncthreads();
    for (int64_t t0 = 0, slot = q.slot; t0 < q.len; t0 += TILE, ++slot) {
        if (p.tile_states)
            for (int n = lane; n < N; n += 64) p.tile_states[(slot * p.dim + d) * N + n] = carry[n];
        const int64_t tl = t0 + lane * K;
        float uu[K], dt[K], du[K], y[K];
        bool live[K], cut[K];  // the position takes part; h starts at 0 there
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int64_t t = q.start + tl + j;
            live[j] = tl + j < q.len;
            cut[j] = false;
            if (live[j] && ids) {
                const int32_t id = ids[t * p.seq_idx_stride[1]];
                cut[j] = t == 0 || ids[(t - 1) * p.seq_idx_stride[1]] != id;
                live[j] = id >= 0;
            }
            uu[j] = live[j] ? to_f32(u[t * p.u_stride[2]]) : 0.0f;
            const float raw = live[j] ? to_f32(delta[t * p.delta_stride[2]]) + bias : 0.0f;
            dt[j] = live[j] ? (p.delta_softplus ? softplus(raw) : raw) : 0.0f;
            du[j] = dt[j] * uu[j];
            y[j] = skip * uu[j];
        }
        for (int n = 0; n < N; ++n) {
            const float A2 = p.A[d * p.A_stride[0] + n * p.A_stride[1]] * kLog2e;
            float a[K], b[K], c[K], P = 1.0f, H = 0.0f;
            bool met = false;  // the lane's span has a start
#pragma unroll
            for (int j = 0; j < K; ++j) {
                const int64_t t = q.start + tl + j;
                a[j] = __builtin_amdgcn_exp2f(dt[j] * A2);
                b[j] = live[j] ? du[j] * to_f32(Bp[n * p.B_stride[2] + t * p.B_stride[3]]) : 0.0f;
                c[j] = live[j] ? to_f32(Cp[n * p.C_stride[2] + t * p.C_stride[3]]) : 0.0f;
                H = cut[j] ? b[j] : __builtin_fmaf(a[j], H, b[j]);
                P *= a[j];
                met |= cut[j];
            }
            const float before = carry[n];
            if (lane == 0 && !met) H = __builtin_fmaf(P, before, H);
            int reach = met;
            for (int w = 1; w < 64; w *= 2) {
                const float Hw = __shfl_up(H, w), Pw = __shfl_up(P, w);
                const int rw = __shfl_up(reach, w);
                if (lane >= w && !reach) {
                    H = __builtin_fmaf(P, Hw, H);
                    P *= Pw;
                    reach |= rw;
                }
            }
            float h = __shfl_up(H, 1);
            if (lane == 0) h = before;
            __syncthreads();
            if (lane == 63) carry[n] = H;
#pragma unroll
            for (int j = 0; j < K; ++j) {
                h = cut[j] ? b[j] : __builtin_fmaf(a[j], h, b[j]);
                if (live[j]) y[j] = __builtin_fmaf(c[j], h, y[j]);
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < K; ++j) {
            if (tl + j >= q.len) break;
            const int64_t t = q.start + tl + j;
            float v = y[j];
            if (z && live[j]) v *= silu(to_f32(z[t * p.z_stride[2]]));
            out[t * p.out_stride[2]] = from_f32<T>(live[j] ? v : 0.0f);
        }
    }
    if (p.final_states)
        for (int n = lane; n < N; n += 64)
            p.final_states[s * p.final_states_stride[0] + d * p.final_states_stride[1] + n * p.final_states_stride[2]] =
                carry[n];
}

}  // namespace

int64_t scan_tile_floats(const cc1d_scan_params& p) { return scan_slots(p, TILE) * p.dim * p.dstate; }

int launch_scan_fwd(const cc1d_scan_params& p, hipStream_t stream) {
    return with_dtype(p.dtype, [&](auto t) {
        const dim3 grid((unsigned)(scan_sequences(p) * p.dim));
        return launch(scan_fwd_kernel<decltype(t)>, grid, dim3(64), stream, p);
    });
}

}  // namespace cc1d
