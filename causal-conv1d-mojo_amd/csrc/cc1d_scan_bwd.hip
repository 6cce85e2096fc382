// cc1d_scan_bwd.hip -- backward of the selective state space scan.
//
// With g[t] = dL/dh[t], and dy = dout (times silu(z) when gated):
//   g[t] = C[t] dy[t] + a[t+1] g[t+1],  w[t] = g[t] a[t] h[t-1]
//   du = D dy + dt sum_n g B        ddt = u sum_n g B + sum_n A w
//   dA = sum_t dt w                 dB[t] = sum_d g dt u,  dC[t] = sum_d dy h
#include "cc1d_scan_device.hpp"

namespace cc1d {
namespace {

constexpr int K = 4;
constexpr int TILE = 64 * K;

struct ScanBwdArgs {
    cc1d_scan_bwd_params p;
    float *pB, *pC;  // (batch, dim, dstate, seqlen): each channel's terms of dB and dC
    float *pA;       // (sequences, dim, dstate)
    float *pD, *pbias;  // (sequences, dim)
};

template <typename T> __device__ void zero_uncovered(const ScanBwdArgs& a, int64_t d, int64_t from, int64_t to) {
    const cc1d_scan_bwd_params& p = a.p;
    for (int64_t t = from + threadIdx.x; t < to; t += 64) {
        static_cast<T*>(p.du)[d * p.du_stride[1] + t * p.du_stride[2]] = T{};
        static_cast<T*>(p.ddelta)[d * p.ddelta_stride[1] + t * p.ddelta_stride[2]] = T{};
        if (p.dz) static_cast<T*>(p.dz)[d * p.dz_stride[1] + t * p.dz_stride[2]] = T{};
        for (int64_t n = 0; n < p.fwd.dstate; ++n) {
            a.pB[(d * p.fwd.dstate + n) * p.fwd.seqlen + t] = 0.0f;
            a.pC[(d * p.fwd.dstate + n) * p.fwd.seqlen + t] = 0.0f;
        }
    }
}

// One wavefront per (sequence, channel), every layout.
template <typename T> __global__ void __launch_bounds__(64) scan_bwd_kernel(const ScanBwdArgs arg) {
    __shared__ float carry[CC1D_MAX_DSTATE];  // a g of the position after the tile
    __shared__ float dA[CC1D_MAX_DSTATE];
    const cc1d_scan_bwd_params& b = arg.p;
    const cc1d_scan_params& p = b.fwd;
    const int lane = threadIdx.x;
    const int64_t s = blockIdx.x / p.dim, d = blockIdx.x % p.dim;
    const ScanSpan q = scan_span(p, s, TILE);
    if (p.cu_seqlens != nullptr) {
        if (s == 0) zero_uncovered<T>(arg, d, 0, q.start);
        if (s == p.num_seqs - 1) zero_uncovered<T>(arg, d, q.start + q.len, p.seqlen);
    }
    const T* u = static_cast<const T*>(p.u) + q.row * p.u_stride[0] + d * p.u_stride[1];
    const T* delta = static_cast<const T*>(p.delta) + q.row * p.delta_stride[0] + d * p.delta_stride[1];
    const T* z = p.z ? static_cast<const T*>(p.z) + q.row * p.z_stride[0] + d * p.z_stride[1] : nullptr;
    const T* dout = static_cast<const T*>(b.dout) + q.row * b.dout_stride[0] + d * b.dout_stride[1];
    T* du_out = static_cast<T*>(b.du) + q.row * b.du_stride[0] + d * b.du_stride[1];
    T* dd_out = static_cast<T*>(b.ddelta) + q.row * b.ddelta_stride[0] + d * b.ddelta_stride[1];
    T* dz_out = z ? static_cast<T*>(b.dz) + q.row * b.dz_stride[0] + d * b.dz_stride[1] : nullptr;
    const int64_t grp = d / (p.dim / p.groups);
    const T* Bp = static_cast<const T*>(p.B) + q.row * p.B_stride[0] + grp * p.B_stride[1];
    const T* Cp = static_cast<const T*>(p.C) + q.row * p.C_stride[0] + grp * p.C_stride[1];
    const int32_t* ids = p.seq_idx ? p.seq_idx + q.row * p.seq_idx_stride[0] : nullptr;
    const float bias = p.delta_bias ? p.delta_bias[d * p.delta_bias_stride] : 0.0f;
    const float skip = p.D ? p.D[d * p.D_stride] : 0.0f;
    const int N = (int)p.dstate;
    for (int n = lane; n < N; n += 64) {
        carry[n] = b.dfinal_states ? b.dfinal_states[s * b.dfinal_states_stride[0] + d * b.dfinal_states_stride[1] +
                                                     n * b.dfinal_states_stride[2]]
                                   : 0.0f;
        dA[n] = 0.0f;
    }
    float dD = 0.0f, dbias = 0.0f;
    __syncthreads();
    const int64_t tiles = (q.len + TILE - 1) / TILE;
    for (int64_t i = tiles - 1; i >= 0; --i) {
        const int64_t tl = i * TILE + lane * K;
        float uu[K], raw[K], dt[K], dy[K], y[K], along[K], wsum[K], zz[K], dd[K];
        bool live[K], cut[K];
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
            raw[j] = live[j] ? to_f32(delta[t * p.delta_stride[2]]) + bias : 0.0f;
            dt[j] = live[j] ? (p.delta_softplus ? softplus(raw[j]) : raw[j]) : 0.0f;
            zz[j] = live[j] && z ? to_f32(z[t * p.z_stride[2]]) : 0.0f;
            dd[j] = live[j] ? to_f32(dout[t * b.dout_stride[2]]) : 0.0f;
            dy[j] = z ? dd[j] * silu(zz[j]) : dd[j];
            y[j] = skip * uu[j];
            along[j] = wsum[j] = 0.0f;
        }
        for (int n = 0; n < N; ++n) {
            const float A = p.A[d * p.A_stride[0] + n * p.A_stride[1]];
            const float A2 = A * kLog2e;
            float a[K], Bn[K], h[K], P = 1.0f, H = 0.0f;
            bool met = false;
#pragma unroll
            for (int j = 0; j < K; ++j) {
                const int64_t t = q.start + tl + j;
                a[j] = __builtin_amdgcn_exp2f(dt[j] * A2);
                Bn[j] = live[j] ? to_f32(Bp[n * p.B_stride[2] + t * p.B_stride[3]]) : 0.0f;
                const float bj = live[j] ? dt[j] * uu[j] * Bn[j] : 0.0f;
                H = cut[j] ? bj : __builtin_fmaf(a[j], H, bj);
                P *= a[j];
                met |= cut[j];
            }
            const float own = P;
            const float before = p.tile_states[((q.slot + i) * p.dim + d) * N + n];
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
            float hp = __shfl_up(H, 1);
            if (lane == 0) hp = before;
            const float entered = hp;
#pragma unroll
            for (int j = 0; j < K; ++j) {
                const float bj = live[j] ? dt[j] * uu[j] * Bn[j] : 0.0f;
                h[j] = hp = cut[j] ? bj : __builtin_fmaf(a[j], hp, bj);
            }
            // the same over the lanes from the end: Q = a g of the lane's first position
            float c[K], Q = 0.0f;
            P = own;
#pragma unroll
            for (int j = K - 1; j >= 0; --j) {
                const int64_t t = q.start + tl + j;
                const float Cn = live[j] ? to_f32(Cp[n * p.C_stride[2] + t * p.C_stride[3]]) : 0.0f;
                if (live[j]) y[j] = __builtin_fmaf(Cn, h[j], y[j]);
                c[j] = Cn * dy[j];
                Q = cut[j] ? 0.0f : a[j] * (c[j] + Q);
                if (tl + j < q.len) {
                    const int64_t at = ((q.row * p.dim + d) * N + n) * p.seqlen + t;
                    arg.pC[at] = live[j] ? dy[j] * h[j] : 0.0f;
                }
            }
            const float after = carry[n];
            if (lane == 63 && !met) Q = __builtin_fmaf(P, after, Q);
            reach = met;
            for (int w = 1; w < 64; w *= 2) {
                const float Qw = __shfl_down(Q, w), Pw = __shfl_down(P, w);
                const int rw = __shfl_down(reach, w);
                if (lane + w < 64 && !reach) {
                    Q = __builtin_fmaf(P, Qw, Q);
                    P *= Pw;
                    reach |= rw;
                }
            }
            float x = __shfl_down(Q, 1);
            if (lane == 63) x = after;
            __syncthreads();
            if (lane == 0) carry[n] = Q;
            float dAn = 0.0f;
#pragma unroll
            for (int j = K - 1; j >= 0; --j) {
                const float gj = c[j] + x;
                x = cut[j] ? 0.0f : a[j] * gj;
                const float prior = j > 0 ? h[j > 0 ? j - 1 : 0] : entered;
                const float w = cut[j] ? 0.0f : x * prior;
                if (live[j]) {
                    along[j] = __builtin_fmaf(gj, Bn[j], along[j]);
                    wsum[j] = __builtin_fmaf(A, w, wsum[j]);
                    dAn = __builtin_fmaf(dt[j], w, dAn);
                }
                if (tl + j < q.len) {
                    const int64_t at = ((q.row * p.dim + d) * N + n) * p.seqlen + q.start + tl + j;
                    arg.pB[at] = live[j] ? gj * dt[j] * uu[j] : 0.0f;
                }
            }
            dAn = wave_sum(dAn);
            if (lane == 0) dA[n] += dAn;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < K; ++j) {
            if (tl + j >= q.len) break;
            const int64_t t = q.start + tl + j;
            float ddt = __builtin_fmaf(uu[j], along[j], wsum[j]);
            if (p.delta_softplus) ddt *= sigmoid(raw[j]);
            du_out[t * b.du_stride[2]] = from_f32<T>(live[j] ? __builtin_fmaf(skip, dy[j], dt[j] * along[j]) : 0.0f);
            dd_out[t * b.ddelta_stride[2]] = from_f32<T>(live[j] ? ddt : 0.0f);
            if (z) dz_out[t * b.dz_stride[2]] = from_f32<T>(live[j] ? dd[j] * y[j] * silu_grad(zz[j]) : 0.0f);
            if (live[j]) {
                dD = __builtin_fmaf(dy[j], uu[j], dD);
                dbias += ddt;
            }
        }
    }
    dD = wave_sum(dD);
    dbias = wave_sum(dbias);
    if (lane == 0) {
        arg.pD[s * p.dim + d] = dD;
        arg.pbias[s * p.dim + d] = dbias;
    }
    for (int n = lane; n < N; n += 64) {
        arg.pA[(s * p.dim + d) * N + n] = dA[n];
        if (b.dinitial_states) b.dinitial_states[(s * p.dim + d) * N + n] = carry[n];
    }
}

// dB and dC: one thread per element, the channels of its group in order.
template <typename T> __global__ void __launch_bounds__(256) scan_bwd_reduce_bc(const ScanBwdArgs arg, int64_t items) {
    const cc1d_scan_params& p = arg.p.fwd;
    const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (idx >= items) return;
    const int64_t t = idx % p.seqlen, n = idx / p.seqlen % p.dstate, g = idx / (p.seqlen * p.dstate) % p.groups,
                  row = idx / (p.seqlen * p.dstate * p.groups), per = p.dim / p.groups;
    float sB = 0.0f, sC = 0.0f;
    for (int64_t d = g * per; d < (g + 1) * per; ++d) {
        const int64_t at = ((row * p.dim + d) * p.dstate + n) * p.seqlen + t;
        sB += arg.pB[at];
        sC += arg.pC[at];
    }
    static_cast<T*>(arg.p.dB)[idx] = from_f32<T>(sB);
    static_cast<T*>(arg.p.dC)[idx] = from_f32<T>(sC);
}

// dA, dD and ddelta_bias: one thread per channel and state, and two more per channel; the sequences in order.
__global__ void __launch_bounds__(256) scan_bwd_reduce_params(const ScanBwdArgs arg, int64_t seqs) {
    const cc1d_scan_params& p = arg.p.fwd;
    const int64_t nA = p.dim * p.dstate;
    int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const float* from = arg.pA;
    float* to = arg.p.dA;
    int64_t step = nA;
    if (i >= nA) {
        i -= nA;
        step = p.dim;
        from = arg.pD;
        to = arg.p.dD;
        if (i >= p.dim) {
            i -= p.dim;
            from = arg.pbias;
            to = arg.p.ddelta_bias;
            if (i >= p.dim) return;
        }
        if (to == nullptr) return;
    }
    float sum = 0.0f;
    for (int64_t s = 0; s < seqs; ++s) sum += from[s * step + i];
    to[i] = sum;
}

}  // namespace

int64_t scan_bwd_workspace_floats(const cc1d_scan_bwd_params& b) {
    const cc1d_scan_params& p = b.fwd;
    return 2 * p.batch * p.dim * p.dstate * p.seqlen + scan_sequences(p) * p.dim * (p.dstate + 2);
}

int launch_scan_bwd(const cc1d_scan_bwd_params& b, hipStream_t stream) {
    const cc1d_scan_params& p = b.fwd;
    const int64_t seqs = scan_sequences(p);
    ScanBwdArgs a{b, nullptr, nullptr, nullptr, nullptr, nullptr};
    a.pB = b.workspace;
    a.pC = a.pB + p.batch * p.dim * p.dstate * p.seqlen;
    a.pA = a.pC + p.batch * p.dim * p.dstate * p.seqlen;
    a.pD = a.pA + seqs * p.dim * p.dstate;
    a.pbias = a.pD + seqs * p.dim;
    const int64_t nbc = p.batch * p.groups * p.dstate * p.seqlen;
    return with_dtype(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        int st = CC1D_OK;
        if (seqs > 0) st = launch(scan_bwd_kernel<T>, dim3((unsigned)(seqs * p.dim)), dim3(64), stream, a);
        if (st == CC1D_OK && nbc > 0)
            st = launch(scan_bwd_reduce_bc<T>, dim3((unsigned)ceil_div(nbc, 256)), dim3(256), stream, a, nbc);
        if (st == CC1D_OK)
            st = launch(scan_bwd_reduce_params, dim3((unsigned)ceil_div(p.dim * (p.dstate + 2), 256)), dim3(256), stream,
                        a, seqs);
        return st;
    });
}

}  // namespace cc1d
