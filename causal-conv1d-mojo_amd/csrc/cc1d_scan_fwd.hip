// cc1d_scan_fwd.hip -- forward of the selective state space scan.
#include "cc1d_scan_device.hpp"

namespace cc1d {
namespace {

// A block: 8 wavefronts and `chans` channels (1, 2, 4, 8, or 16 with two per
// wavefront) of one group and sequence. With fewer than 8 channels the
// wavefronts of a channel take its states in turns and add their outputs.
struct ScanFwdArgs {
    cc1d_scan_params p;
    int64_t group_blocks;  // blocks per group
    int split;             // wavefronts per channel
};

// Positions of batch row 0 that no sequence covers: before the first and after the last.
template <typename T>
__device__ void zero_uncovered(const cc1d_scan_params& p, int64_t s, int64_t d, const ScanSpan& q) {
    const int lane = threadIdx.x & 63;
    T* out = static_cast<T*>(p.out) + d * p.out_stride[1];
    if (s == 0)
        for (int64_t t = lane; t < q.start; t += 64) out[t * p.out_stride[2]] = T{};
    if (s == p.num_seqs - 1)
        for (int64_t t = q.start + q.len + lane; t < p.seqlen; t += 64) out[t * p.out_stride[2]] = T{};
}

// What one channel's tile holds in registers.
template <int K> struct Channel {
    float dt[K], du[K], y[K], step_sum;
};

// One state of CHW channels: see cc1d_scan_device.hpp.
template <int K, int CHW, bool CUT>
__device__ __forceinline__ void scan_state(Channel<K> (&ch)[CHW], const float* A2, float* const* carry, int n,
                                           const float (&B)[K], const float (&C)[K], const Cuts<K>& cuts, int lane) {
    float a[CHW][K], H[CHW], P[CHW], first[CHW];
#pragma unroll
    for (int c = 0; c < CHW; ++c) {
        const float before = carry[c][n];
#pragma unroll
        for (int j = 0; j < K; ++j) a[c][j] = __builtin_amdgcn_exp2f(ch[c].dt[j] * A2[c]);
        P[c] = __builtin_amdgcn_exp2f(ch[c].step_sum * A2[c]);
        float h = ch[c].du[0] * B[0];
#pragma unroll
        for (int j = 1; j < K; ++j) {
            const float b = ch[c].du[j] * B[j];
            h = CUT && cuts.at[j] ? b : __builtin_fmaf(a[c][j], h, b);
        }
        first[c] = lane == 0 ? before : 0.0f;
        const float entered = __builtin_fmaf(P[c], first[c], h);
        H[c] = CUT && (cuts.met || lane != 0) ? h : entered;
    }
    if constexpr (CUT) {
#pragma unroll
        for (int c = 0; c < CHW; ++c) wave_prefix_cut(H[c], P[c], cuts.absorb);
    } else if constexpr (CHW == 2) {
        wave_prefix2(H[0], P[0], H[1], P[1]);
    } else {
        wave_prefix(H[0], P[0]);
    }
#pragma unroll
    for (int c = 0; c < CHW; ++c) {
        float h = dpp_keep<kDppWaveShr1, 0xf>(first[c], H[c]);
        if (lane == 63) carry[c][n] = H[c];
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const float b = ch[c].du[j] * B[j];
            h = CUT && cuts.at[j] ? b : __builtin_fmaf(a[c][j], h, b);
            ch[c].y[j] = __builtin_fmaf(C[j], h, ch[c].y[j]);
        }
    }
}

// UNIT: the time strides of u, delta, z and out are 1; TIME: those of B and C (and the rows hold K positions).
template <typename T, int K, int CHW, int NCAP, bool SEQ, bool UNIT, bool TIME>
__global__ void __launch_bounds__(512, UNIT && TIME ? 4 : 2) scan_fwd_rows(const ScanFwdArgs arg) {
    constexpr int TILE = 64 * K;
    __shared__ __attribute__((aligned(16))) float BC[2 * kStates * TILE];
    __shared__ float carries[8 * CHW * NCAP];
    const cc1d_scan_params& p = arg.p;
    const int lane = threadIdx.x & 63, wave = (int)uniform32(threadIdx.x >> 6);
    const int split = arg.split, part = wave % split;
    const int64_t per = p.dim / p.groups;
    const int64_t blk = blockIdx.x % arg.group_blocks, g = blockIdx.x / arg.group_blocks % p.groups,
                  s = blockIdx.x / arg.group_blocks / p.groups;
    const ScanSpan q = scan_span(p, s, TILE);
    const int64_t in_group = (blk * (8 / split) + wave / split) * CHW;  // the wavefront's first channel
    const int channels = (int)(per - in_group < CHW ? (per - in_group < 0 ? 0 : per - in_group) : CHW);
    const int N = (int)p.dstate;
    const int begin = (int)q.start, end = (int)(q.start + q.len), size = (int)p.seqlen;

    // A missing channel repeats the group's last one, and stores nothing.
    float* carry[CHW];
    float bias[CHW], skip[CHW];
    const T *pu[CHW], *pd[CHW], *pz[CHW];
    T* po[CHW];
    const float* pA[CHW];
    float* tiles[CHW];
    const int64_t us = UNIT ? 1 : p.u_stride[2], ds = UNIT ? 1 : p.delta_stride[2], zs = UNIT ? 1 : p.z_stride[2],
                  os = UNIT ? 1 : p.out_stride[2];
#pragma unroll
    for (int c = 0; c < CHW; ++c) {
        const int64_t d = g * per + (in_group + c < per ? in_group + c : per - 1);
        carry[c] = carries + (wave / split * CHW + c) * NCAP;
        bias[c] = p.delta_bias ? ld_uniform(p.delta_bias + d * p.delta_bias_stride) : 0.0f;
        skip[c] = p.D && part == 0 ? ld_uniform(p.D + d * p.D_stride) : 0.0f;
        pu[c] = static_cast<const T*>(p.u) + q.row * p.u_stride[0] + d * p.u_stride[1];
        pd[c] = static_cast<const T*>(p.delta) + q.row * p.delta_stride[0] + d * p.delta_stride[1];
        pz[c] = p.z ? static_cast<const T*>(p.z) + q.row * p.z_stride[0] + d * p.z_stride[1] : nullptr;
        po[c] = static_cast<T*>(p.out) + q.row * p.out_stride[0] + d * p.out_stride[1];
        pA[c] = p.A + d * p.A_stride[0];
        tiles[c] = p.tile_states && c < channels ? p.tile_states + (q.slot * p.dim + d) * N : nullptr;
        if (p.cu_seqlens != nullptr && c < channels && part == 0) zero_uncovered<T>(p, s, d, q);
        const float* from = p.initial_states ? p.initial_states + s * p.initial_states_stride[0] + d * p.initial_states_stride[1] : nullptr;
        for (int n = part * 64 + lane; n < N; n += 64 * split) carry[c][n] = from ? from[n * p.initial_states_stride[2]] : 0.0f;
    }
    const T* Bp = static_cast<const T*>(p.B) + q.row * p.B_stride[0] + g * p.B_stride[1];
    const T* Cp = static_cast<const T*>(p.C) + q.row * p.C_stride[0] + g * p.C_stride[1];
    const int32_t* ids = SEQ ? p.seq_idx + q.row * p.seq_idx_stride[0] : nullptr;
    const int64_t is = SEQ ? p.seq_idx_stride[1] : 0;

    Raw<T, K> ru[CHW], rd[CHW];
    StateRows<T, K, 8, TIME> rows;
    auto fetch = [&](Raw<T, K>& r, const T* row, int64_t stride, int t0) {
        if constexpr (UNIT) r.load(row, t0 + lane * K, size);
        else r.each(row, stride, t0 + lane * K, end);
    };
    auto fetch_inputs = [&](int t0) {
#pragma unroll
        for (int c = 0; c < CHW; ++c) {
            fetch(ru[c], pu[c], us, t0);
            fetch(rd[c], pd[c], ds, t0);
        }
    };
    auto fetch_states = [&](int t0, int n0) { rows.load(p, Bp, Cp, n0, N - n0 < kStates ? N - n0 : kStates, t0, end, size); };
    if (begin < end) {
        fetch_inputs(begin);
        fetch_states(begin, 0);
    }
    __syncthreads();

    for (int t0 = begin; t0 < end; t0 += TILE) {
        const int t = t0 + lane * K;
        const bool full = end - t0 >= TILE;
        Channel<K> ch[CHW];
        Raw<T, K> rz[CHW];
        Cuts<K> cuts;
        bool live[K];
#pragma unroll
        for (int j = 0; j < K; ++j) live[j] = t + j < end;
        if constexpr (SEQ) cuts.read(ids, is, t, end - t, live);
        else cuts.none();
#pragma unroll
        for (int c = 0; c < CHW; ++c) {
            if (tiles[c]) {
                for (int n = part * 64 + lane; n < N; n += 64 * split) tiles[c][n] = carry[c][n];
                tiles[c] += p.dim * N;
            }
            if (UNIT && !full) {
                ru[c].fix(t, end, size);
                rd[c].fix(t, end, size);
            }
            steps<K>(rd[c], bias[c], p.delta_softplus != 0, ch[c].dt);
            if (SEQ || !full) {
#pragma unroll
                for (int j = 0; j < K; ++j) ch[c].dt[j] = live[j] ? ch[c].dt[j] : 0.0f;
            }
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < K; ++j) {
                const float u = SEQ && !live[j] ? 0.0f : ru[c].get(j);
                ch[c].du[j] = ch[c].dt[j] * u;
                ch[c].y[j] = skip[c] * u;
                sum += ch[c].dt[j];
            }
            ch[c].step_sum = sum;
        }
        for (int n0 = 0; n0 < N; n0 += kStates) {
            const int nn = N - n0 < kStates ? N - n0 : kStates;
            rows.store(BC, nn, t0, end, size, ids, is);
            __syncthreads();
            // the next values travel while these are used
            if (n0 + kStates < N) fetch_states(t0, n0 + kStates);
            else if (t0 + TILE < end) fetch_states(t0 + TILE, 0);
            if (n0 == 0) {
                if (t0 + TILE < end) fetch_inputs(t0 + TILE);
                if (p.z) {
#pragma unroll
                    for (int c = 0; c < CHW; ++c) fetch(rz[c], pz[c], zs, t0);
                }
            }
#pragma unroll 1
            for (int n = part; n < nn; n += split) {
                float A2[CHW], B[K], C[K];
#pragma unroll
                for (int c = 0; c < CHW; ++c) A2[c] = ld_uniform(pA[c] + (n0 + n) * p.A_stride[1]) * kLog2e;
                read_state<K>(BC, n, lane, B);
                read_state<K>(BC + kStates * TILE, n, lane, C);
                if (SEQ && cuts.any) scan_state<K, CHW, true>(ch, A2, carry, n0 + n, B, C, cuts, lane);
                else scan_state<K, CHW, false>(ch, A2, carry, n0 + n, B, C, cuts, lane);
            }
            __syncthreads();
        }
        if (CHW == 1 && split > 1) {  // the channel's first wavefront adds the parts in order
            float* own = BC + wave * TILE;
#pragma unroll
            for (int qd = 0; qd < K / 4; ++qd)
                *reinterpret_cast<f32x4*>(own + (qd * 64 + lane) * 4) =
                    f32x4{ch[0].y[4 * qd], ch[0].y[4 * qd + 1], ch[0].y[4 * qd + 2], ch[0].y[4 * qd + 3]};
            __syncthreads();
            if (part == 0) {
                for (int w = 1; w < split; ++w) {
#pragma unroll
                    for (int qd = 0; qd < K / 4; ++qd) {
                        const f32x4 v = *reinterpret_cast<const f32x4*>(own + w * TILE + (qd * 64 + lane) * 4);
#pragma unroll
                        for (int j = 0; j < 4; ++j) ch[0].y[4 * qd + j] += v[j];
                    }
                }
            }
            __syncthreads();
        }
        if (part == 0) {
#pragma unroll
            for (int c = 0; c < CHW; ++c) {
                if (c >= channels) break;
                if (p.z) {
                    if (UNIT && !full) rz[c].fix(t, end, size);
#pragma unroll
                    for (int j = 0; j < K; ++j) ch[c].y[j] *= silu(rz[c].get(j));
                }
                if constexpr (SEQ) {
#pragma unroll
                    for (int j = 0; j < K; ++j)
                        if (!live[j]) ch[c].y[j] = 0.0f;
                }
                store_steps<T, K>(po[c], os, t, end, ch[c].y);
            }
        }
    }
    if (p.final_states) {
#pragma unroll
        for (int c = 0; c < CHW; ++c) {
            if (c >= channels) break;
            float* to = p.final_states + s * p.final_states_stride[0] + (g * per + in_group + c) * p.final_states_stride[1];
            for (int n = part * 64 + lane; n < N; n += 64 * split) to[n * p.final_states_stride[2]] = carry[c][n];
        }
    }
}

template <typename T, int K, int CHW, int NCAP> int launch_rows(const ScanFwdArgs& a, hipStream_t stream) {
    const cc1d_scan_params& p = a.p;
    const dim3 grid((unsigned)(a.group_blocks * p.groups * scan_sequences(p))), block(512);
    const bool unit = p.seqlen >= K && p.u_stride[2] == 1 && p.delta_stride[2] == 1 && p.out_stride[2] == 1 && (!p.z || p.z_stride[2] == 1);
    const bool time = p.seqlen >= K && p.B_stride[3] == 1 && p.C_stride[3] == 1;
    return with_flag(p.seq_idx != nullptr, [&](auto seq) {
        return with_flag(unit, [&](auto u) {
            return with_flag(time, [&](auto tm) {
                return launch(scan_fwd_rows<T, K, CHW, NCAP, decltype(seq)::value, decltype(u)::value, decltype(tm)::value>,
                              grid, block, stream, a);
            });
        });
    });
}

}  // namespace

int64_t scan_tile_floats(const cc1d_scan_params& p) { return scan_slots(p) * p.dim * p.dstate; }

int launch_scan_fwd(const cc1d_scan_params& p, hipStream_t stream) {
    ScanFwdArgs a{p, 0, 8};
    const int64_t channels = scan_sequences(p) * p.dim, per = p.dim / p.groups;
    while (a.split > 1 && channels > 512 * (8 / a.split) && per > 8 / a.split && a.split > 1) a.split /= 2;
#ifdef PROBE_TWO
    const bool two = a.split == 1 && channels >= 8192 && per >= 16;
#else
    const bool two = false;
#endif
    a.group_blocks = ceil_div(per, (8 / a.split) * (two ? 2 : 1));
    return with_dtype(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        return with_flag(scan_tile(p.seqlen) == 512, [&](auto wide) {
            constexpr int K = decltype(wide)::value ? 8 : 4;
            return with_flag(p.dstate <= 16, [&](auto few) {
                constexpr int NCAP = decltype(few)::value ? 16 : CC1D_MAX_DSTATE;
#ifdef PROBE_TWO
                if (two) return launch_rows<T, K, 2, NCAP>(a, stream);
#endif
                return launch_rows<T, K, 1, NCAP>(a, stream);
            });
        });
    });
}

}  // namespace cc1d
