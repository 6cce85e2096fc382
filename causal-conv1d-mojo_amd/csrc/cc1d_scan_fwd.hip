// cc1d_scan_fwd.hip -- forward of the selective state space scan.
//
// Vector issue bounds it: 12.7 instructions per position, channel and state
// with 16 states, which fill 97% of the time (13.4 and 88% channel-last): 250
// to 260 us at 4 x 5120 x 2048 bf16. Its 341 MB would take 54.
#include "cc1d_scan_device.hpp"

namespace cc1d {
namespace {

// A block: 8 wavefronts and 8 / split channels of one group and sequence, whose
// B and C they share through LDS (64 KB: two blocks a CU, 16 wavefronts). With
// fewer than 8 channels the wavefronts of a channel take its states in turns
// and add their outputs.
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

// One state of a channel: see cc1d_scan_device.hpp. carry: the channel's states
// ahead of the tile, and of the next one on return.
template <int K, bool CUT>
__device__ __forceinline__ void scan_state(Channel<K>& ch, float A2, float* carry, const float (&B)[K], const float (&C)[K],
                                           const Cuts<K>& cuts, int lane) {
    float a[K];
    const float before = *carry;
#pragma unroll
    for (int j = 0; j < K; ++j) a[j] = __builtin_amdgcn_exp2f(ch.dt[j] * A2);
    float P = __builtin_amdgcn_exp2f(ch.step_sum * A2);
    float h = ch.du[0] * B[0];
#pragma unroll
    for (int j = 1; j < K; ++j) {
        const float b = ch.du[j] * B[j];
        h = CUT && cuts.at[j] ? b : __builtin_fmaf(a[j], h, b);
    }
    const float first = lane == 0 ? before : 0.0f;
    const float entered = __builtin_fmaf(P, first, h);
    float H = CUT && (cuts.met || lane != 0) ? h : entered;
    if constexpr (CUT) wave_prefix_cut(H, P, cuts.absorb);
    else wave_prefix(H, P);
    h = dpp_keep<kDppWaveShr1, 0xf>(first, H);
    if (lane == 63) *carry = H;
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const float b = ch.du[j] * B[j];
        h = CUT && cuts.at[j] ? b : __builtin_fmaf(a[j], h, b);
        ch.y[j] = __builtin_fmaf(C[j], h, ch.y[j]);
    }
}

// UNIT: the time strides of u, delta, z and out are 1, and the rows hold K positions.
template <typename T, int K, bool SEQ, bool UNIT, StateMode MODE>
__global__ void __launch_bounds__(512, UNIT && MODE == kStateTime ? 4 : 2) scan_fwd_rows(const ScanFwdArgs arg) {
    constexpr int TILE = 64 * K;
    __shared__ __attribute__((aligned(16))) float BC[2 * kStates * TILE];
    __shared__ float carries[8 * CC1D_MAX_DSTATE];
    const cc1d_scan_params& p = arg.p;
    const int lane = threadIdx.x & 63, wave = (int)uniform32(threadIdx.x >> 6);
    const int split = arg.split, part = wave % split;
    const int64_t per = p.dim / p.groups;
    const uint32_t order = xcd_block(blockIdx.x, gridDim.x);
    const int64_t blk = order % arg.group_blocks, g = order / arg.group_blocks % p.groups,
                  s = order / arg.group_blocks / p.groups;
    const ScanSpan q = scan_span(p, s, TILE);
    const int64_t in_group = blk * (8 / split) + wave / split;  // the wavefront's channel
    const bool mine = in_group < per;  // a missing channel repeats the group's last one, and stores nothing
    const int N = (int)p.dstate;
    const int begin = (int)q.start, end = (int)(q.start + q.len), size = (int)p.seqlen;

    const int64_t us = UNIT ? 1 : p.u_stride[2], ds = UNIT ? 1 : p.delta_stride[2], zs = UNIT ? 1 : p.z_stride[2],
                  os = UNIT ? 1 : p.out_stride[2];
    const int64_t d = g * per + (mine ? in_group : per - 1);
    float* const carry = carries + wave / split * CC1D_MAX_DSTATE;
    const float bias = p.delta_bias ? ld_uniform(p.delta_bias + d * p.delta_bias_stride) : 0.0f;
    const float skip = p.D && part == 0 ? ld_uniform(p.D + d * p.D_stride) : 0.0f;
    const T* const pu = static_cast<const T*>(p.u) + q.row * p.u_stride[0] + d * p.u_stride[1];
    const T* const pd = static_cast<const T*>(p.delta) + q.row * p.delta_stride[0] + d * p.delta_stride[1];
    const T* const pz = p.z ? static_cast<const T*>(p.z) + q.row * p.z_stride[0] + d * p.z_stride[1] : nullptr;
    T* const po = static_cast<T*>(p.out) + q.row * p.out_stride[0] + d * p.out_stride[1];
    const float* const pA = p.A + d * p.A_stride[0];
    float* tiles = p.tile_states && mine ? p.tile_states + (q.slot * p.dim + d) * N : nullptr;
    if (p.cu_seqlens != nullptr && mine && part == 0) zero_uncovered<T>(p, s, d, q);
    const float* from = p.initial_states ? p.initial_states + s * p.initial_states_stride[0] + d * p.initial_states_stride[1] : nullptr;
    for (int n = part * 64 + lane; n < N; n += 64 * split) carry[n] = from ? from[n * p.initial_states_stride[2]] : 0.0f;
    const T* Bp = static_cast<const T*>(p.B) + q.row * p.B_stride[0] + g * p.B_stride[1];
    const T* Cp = static_cast<const T*>(p.C) + q.row * p.C_stride[0] + g * p.C_stride[1];
    const int32_t* ids = SEQ ? p.seq_idx + q.row * p.seq_idx_stride[0] : nullptr;
    const int64_t is = SEQ ? p.seq_idx_stride[1] : 0;

    Raw<T, K> ru, rd, rz;
    StateRows<T, K, 8, MODE> rows;
    auto fetch = [&](Raw<T, K>& r, const T* row, int64_t stride, int t0) {
        if constexpr (UNIT) r.load(row, t0 + lane * K, size);
        else r.each(row, stride, t0 + lane * K, end);
    };
    auto fetch_inputs = [&](int t0) {
        fetch(ru, pu, us, t0);
        fetch(rd, pd, ds, t0);
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
        Channel<K> ch;
        Cuts<K> cuts;
        bool live[K];
#pragma unroll
        for (int j = 0; j < K; ++j) live[j] = t + j < end;
        if constexpr (SEQ) cuts.read(ids, is, t, end - t, live);
        else cuts.none();
        const uint32_t bits = live_bits<K>(live);
        if (tiles) {
            for (int n = part * 64 + lane; n < N; n += 64 * split) tiles[n] = carry[n];
            tiles += p.dim * N;
        }
        if (UNIT && !full) {
            ru.fix(t, end, size);
            rd.fix(t, end, size);
        }
        steps<K>(rd, bias, p.delta_softplus != 0, ch.dt);
        if (SEQ || !full) {
#pragma unroll
            for (int j = 0; j < K; ++j) ch.dt[j] = live[j] ? ch.dt[j] : 0.0f;
        }
        ch.step_sum = 0.0f;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const float u = SEQ && !live[j] ? 0.0f : ru.get(j);
            ch.du[j] = ch.dt[j] * u;
            ch.y[j] = skip * u;
            ch.step_sum += ch.dt[j];
        }
        for (int n0 = 0; n0 < N; n0 += kStates) {
            const int nn = N - n0 < kStates ? N - n0 : kStates;
            rows.store(BC, n0, nn, N, t0, end, size, bits);
            __syncthreads();
            // the next values travel while these are used
            if (n0 + kStates < N) fetch_states(t0, n0 + kStates);
            else if (t0 + TILE < end) fetch_states(t0 + TILE, 0);
            if (n0 == 0) {
                if (t0 + TILE < end) fetch_inputs(t0 + TILE);
                if (p.z) fetch(rz, pz, zs, t0);
            }
#pragma unroll 1
            for (int n = part; n < nn; n += split) {
                float B[K], C[K];
                const float A2 = ld_uniform(pA + (n0 + n) * p.A_stride[1]) * kLog2e;
                read_state<K>(BC, n, lane, B);
                read_state<K>(BC + kStates * TILE, n, lane, C);
                if (SEQ && cuts.any) scan_state<K, true>(ch, A2, carry + n0 + n, B, C, cuts, lane);
                else scan_state<K, false>(ch, A2, carry + n0 + n, B, C, cuts, lane);
            }
            __syncthreads();
        }
        if (split > 1) {  // the channel's first wavefront adds the parts in order
            float* own = BC + wave * TILE;
#pragma unroll
            for (int k = 0; k < K / 4; ++k)
                *reinterpret_cast<f32x4*>(own + (k * 64 + lane) * 4) =
                    f32x4{ch.y[4 * k], ch.y[4 * k + 1], ch.y[4 * k + 2], ch.y[4 * k + 3]};
            __syncthreads();
            if (part == 0) {
                for (int w = 1; w < split; ++w) {
#pragma unroll
                    for (int k = 0; k < K / 4; ++k) {
                        const f32x4 v = *reinterpret_cast<const f32x4*>(own + w * TILE + (k * 64 + lane) * 4);
#pragma unroll
                        for (int j = 0; j < 4; ++j) ch.y[4 * k + j] += v[j];
                    }
                }
            }
            __syncthreads();
        }
        if (part == 0 && mine) {
            if (p.z) {
                if (UNIT && !full) rz.fix(t, end, size);
#pragma unroll
                for (int j = 0; j < K; ++j) ch.y[j] *= silu(rz.get(j));
            }
            if constexpr (SEQ) {
#pragma unroll
                for (int j = 0; j < K; ++j)
                    if (!live[j]) ch.y[j] = 0.0f;
            }
            store_steps<T, K>(po, os, t, end, ch.y);
        }
    }
    if (p.final_states && mine) {
        float* to = p.final_states + s * p.final_states_stride[0] + d * p.final_states_stride[1];
        for (int n = part * 64 + lane; n < N; n += 64 * split) to[n * p.final_states_stride[2]] = carry[n];
    }
}

// Channel-last tensors (unit channel stride in u, delta, z and out): tiles pass
// through LDS, one tensor after the other through one buffer, so that two
// blocks fit a CU. A block's 8 wavefronts have one channel each: 16 bytes of a
// position (16-bit types), the rest of the 128-byte line being for the 7
// neighbouring blocks on the same XCD. Blocks of 16 and 32 channels read 32 and
// 64 bytes at once, but a CU holds one of them: 333 and 452 us against 296 at
// 4 x 5120 x 2048.
template <typename T, int K, int NCAP, bool SEQ, StateMode MODE>
__global__ void __launch_bounds__(512, sizeof(T) == 2 && NCAP <= 128 ? 4 : 2) scan_fwd_last(const ScanFwdArgs arg) {
    constexpr int TILE = 64 * K, CB = 8;
    typedef ChannelTile<T, K, CB, 512> Tile;
    __shared__ __attribute__((aligned(16))) float BC[2 * kStates * TILE];
    __shared__ __attribute__((aligned(16))) T buf[Tile::BYTES / sizeof(T)];
    __shared__ float carries[CB * NCAP];
    const cc1d_scan_params& p = arg.p;
    const int lane = threadIdx.x & 63, wave = (int)uniform32(threadIdx.x >> 6);
    const uint32_t order = xcd_block(blockIdx.x, gridDim.x);
    const int64_t per = p.dim / p.groups;
    const int64_t blk = order % arg.group_blocks, g = order / arg.group_blocks % p.groups, s = order / arg.group_blocks / p.groups;
    const ScanSpan q = scan_span(p, s, TILE);
    const int channels = (int)(per - blk * CB < CB ? per - blk * CB : CB);  // the block's, from c0 on
    const int c0 = (int)(g * per + blk * CB), dim = (int)p.dim, N = (int)p.dstate;
    const int begin = (int)q.start, end = (int)(q.start + q.len), size = (int)p.seqlen;
    const bool mine = wave < channels;  // a missing channel repeats the last one, and stores nothing
    const int64_t d = c0 + (mine ? wave : channels - 1);
    float* const carry = carries + wave * NCAP;
    const float bias = p.delta_bias ? ld_uniform(p.delta_bias + d * p.delta_bias_stride) : 0.0f;
    const float skip = p.D ? ld_uniform(p.D + d * p.D_stride) : 0.0f;
    const float* const pA = p.A + d * p.A_stride[0];
    if (p.cu_seqlens != nullptr && mine) zero_uncovered<T>(p, s, d, q);
    const float* from = p.initial_states ? p.initial_states + s * p.initial_states_stride[0] + d * p.initial_states_stride[1] : nullptr;
    for (int n = lane; n < N; n += 64) carry[n] = from ? from[n * p.initial_states_stride[2]] : 0.0f;
    float* tiles = p.tile_states && mine ? p.tile_states + (q.slot * p.dim + d) * N : nullptr;
    const T* const pu = static_cast<const T*>(p.u) + q.row * p.u_stride[0];
    const T* const pd = static_cast<const T*>(p.delta) + q.row * p.delta_stride[0];
    const T* const pz = p.z ? static_cast<const T*>(p.z) + q.row * p.z_stride[0] : nullptr;
    T* const po = static_cast<T*>(p.out) + q.row * p.out_stride[0];
    const T* const Bp = static_cast<const T*>(p.B) + q.row * p.B_stride[0] + g * p.B_stride[1];
    const T* const Cp = static_cast<const T*>(p.C) + q.row * p.C_stride[0] + g * p.C_stride[1];
    const int32_t* ids = SEQ ? p.seq_idx + q.row * p.seq_idx_stride[0] : nullptr;
    const int64_t is = SEQ ? p.seq_idx_stride[1] : 0;

    Tile tu, td, tz;
    StateRows<T, K, 8, MODE> rows;
    auto fetch_inputs = [&](int t0) {
        tu.load(pu, p.u_stride[2], c0, dim, t0, end);
        td.load(pd, p.delta_stride[2], c0, dim, t0, end);
    };
    auto fetch_states = [&](int t0, int n0) { rows.load(p, Bp, Cp, n0, N - n0 < kStates ? N - n0 : kStates, t0, end, size); };
    if (begin < end) {
        fetch_inputs(begin);
        fetch_states(begin, 0);
    }
    for (int t0 = begin; t0 < end; t0 += TILE) {
        const int t = t0 + lane * K;
        const bool full = end - t0 >= TILE;
        Channel<K> ch;
        Cuts<K> cuts;
        bool live[K];
#pragma unroll
        for (int j = 0; j < K; ++j) live[j] = t + j < end;
        if constexpr (SEQ) cuts.read(ids, is, t, end - t, live);
        else cuts.none();
        const uint32_t bits = live_bits<K>(live);
        Raw<T, K> ru, rd;
        __syncthreads();  // the last tile's outputs have left the buffer
        tu.to_lds(buf, c0, dim);
        __syncthreads();
        Tile::row(buf, wave, lane, ru);
        __syncthreads();
        td.to_lds(buf, c0, dim);
        __syncthreads();
        Tile::row(buf, wave, lane, rd);
        if (tiles) {
            for (int n = lane; n < N; n += 64) tiles[n] = carry[n];
            tiles += p.dim * N;
        }
        steps<K>(rd, bias, p.delta_softplus != 0, ch.dt);
        ch.step_sum = 0.0f;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const bool in = SEQ ? live[j] : full || live[j];
            ch.dt[j] = in ? ch.dt[j] : 0.0f;
            const float u = in ? ru.get(j) : 0.0f;
            ch.du[j] = ch.dt[j] * u;
            ch.y[j] = skip * u;
            ch.step_sum += ch.dt[j];
        }
        if (p.z) tz.load(pz, p.z_stride[2], c0, dim, t0, end);
        for (int n0 = 0; n0 < N; n0 += kStates) {
            const int nn = N - n0 < kStates ? N - n0 : kStates;
            rows.store(BC, n0, nn, N, t0, end, size, bits);
            __syncthreads();
            if (n0 + kStates < N) fetch_states(t0, n0 + kStates);
            else if (t0 + TILE < end) fetch_states(t0 + TILE, 0);
            if (n0 == 0 && t0 + TILE < end) fetch_inputs(t0 + TILE);
#pragma unroll 1
            for (int n = 0; n < nn; ++n) {
                float B[K], C[K];
                const float A2 = ld_uniform(pA + (n0 + n) * p.A_stride[1]) * kLog2e;
                read_state<K>(BC, n, lane, B);
                read_state<K>(BC + kStates * TILE, n, lane, C);
                if (SEQ && cuts.any) scan_state<K, true>(ch, A2, carry + n0 + n, B, C, cuts, lane);
                else scan_state<K, false>(ch, A2, carry + n0 + n, B, C, cuts, lane);
            }
            __syncthreads();
        }
        if (p.z) {
            tz.to_lds(buf, c0, dim);
            __syncthreads();
            Raw<T, K> rz;
            Tile::row(buf, wave, lane, rz);
#pragma unroll
            for (int j = 0; j < K; ++j) ch.y[j] *= silu(rz.get(j));
        }
        if constexpr (SEQ) {
#pragma unroll
            for (int j = 0; j < K; ++j)
                if (!live[j]) ch.y[j] = 0.0f;
        }
        Tile::put_row(buf, wave, lane, ch.y);  // (in place of z, which no other wavefront reads)
        __syncthreads();
        Tile::store(buf, po, p.out_stride[2], c0, channels, t0, end);
    }
    if (p.final_states && mine) {
        wave_lds_sync();
        float* to = p.final_states + s * p.final_states_stride[0] + d * p.final_states_stride[1];
        for (int n = lane; n < N; n += 64) to[n * p.final_states_stride[2]] = carry[n];
    }
}

// Rows of at most 64 positions: a block takes 32 channels.
template <typename T, bool SEQ, bool UNIT> __global__ void __launch_bounds__(512, 4) scan_fwd_short(const ScanFwdArgs arg) {
    constexpr int K = kShortK;
    __shared__ __attribute__((aligned(16))) float BC[2 * kStates * kShort];
    const cc1d_scan_params& p = arg.p;
    const int lane = threadIdx.x & 63, l = lane & 15, t = l * K, end = (int)p.seqlen, N = (int)p.dstate;
    const int64_t per = p.dim / p.groups;
    const int64_t blk = blockIdx.x % arg.group_blocks, g = blockIdx.x / arg.group_blocks % p.groups, s = blockIdx.x / arg.group_blocks / p.groups;
    const int64_t in_group = blk * 32 + threadIdx.x / 16;
    const bool mine = in_group < per;  // a missing channel repeats the last one, and stores nothing
    const int64_t d = g * per + (mine ? in_group : per - 1);
    const T* const Bp = static_cast<const T*>(p.B) + s * p.B_stride[0] + g * p.B_stride[1];
    const T* const Cp = static_cast<const T*>(p.C) + s * p.C_stride[0] + g * p.C_stride[1];
    const int32_t* ids = SEQ ? p.seq_idx + s * p.seq_idx_stride[0] : nullptr;
    const int64_t is = SEQ ? p.seq_idx_stride[1] : 0;
    ShortCuts cuts;
    bool live[K];
#pragma unroll
    for (int j = 0; j < K; ++j) live[j] = t + j < end;
    if constexpr (SEQ) cuts.read(ids, is, t, end, live);
    else cuts.none();
    auto input = [&](Raw<T, K>& r, const void* base, const int64_t* stride) {
        const T* row = static_cast<const T*>(base) + s * stride[0] + d * stride[1];
        if constexpr (UNIT) r.load(row, t, end);
        else r.each(row, stride[2], t, end);
    };
    Raw<T, K> ru, rd, rz;
    input(ru, p.u, p.u_stride);
    input(rd, p.delta, p.delta_stride);
    if (p.z) input(rz, p.z, p.z_stride);
    if constexpr (UNIT) {
        ru.fix(t, end, end);
        rd.fix(t, end, end);
        if (p.z) rz.fix(t, end, end);
    }
    float dt[K], du[K], y[K], step_sum = 0.0f;
    steps<K>(rd, p.delta_bias ? p.delta_bias[d * p.delta_bias_stride] : 0.0f, p.delta_softplus != 0, dt);
    const float skip = p.D ? p.D[d * p.D_stride] : 0.0f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
        dt[j] = live[j] ? dt[j] : 0.0f;
        const float u = live[j] ? ru.get(j) : 0.0f;
        du[j] = dt[j] * u;
        y[j] = skip * u;
        step_sum += dt[j];
    }
    for (int n0 = 0; n0 < N; n0 += kStates) {
        const int nn = N - n0 < kStates ? N - n0 : kStates;
        float A_l = 0.0f, before_l = 0.0f, after_l = 0.0f;
        if (l < nn) {
            A_l = p.A[d * p.A_stride[0] + (n0 + l) * p.A_stride[1]] * kLog2e;
            if (p.initial_states)
                before_l = p.initial_states[s * p.initial_states_stride[0] + d * p.initial_states_stride[1] +
                                            (n0 + l) * p.initial_states_stride[2]];
            if (p.tile_states && mine) p.tile_states[(s * p.dim + d) * N + n0 + l] = before_l;
        }
        __syncthreads();
        short_states<T>(BC, p, Bp, Cp, n0, nn, ids, is);
        __syncthreads();
#pragma unroll 2
        for (int n = 0; n < nn; ++n) {
            float B[K], C[K], a[K];
            short_state(BC, n, l, B);
            short_state(BC, kStates + n, l, C);
            const float A2 = row_lane(A_l, n), before = row_lane(before_l, n);
#pragma unroll
            for (int j = 0; j < K; ++j) a[j] = __builtin_amdgcn_exp2f(dt[j] * A2);
            float P = __builtin_amdgcn_exp2f(step_sum * A2);
            float h = du[0] * B[0];
#pragma unroll
            for (int j = 1; j < K; ++j) {
                const float b = du[j] * B[j];
                h = SEQ && cuts.at[j] ? b : __builtin_fmaf(a[j], h, b);
            }
            const float first = l == 0 ? before : 0.0f, entered = __builtin_fmaf(P, first, h);
            float H = SEQ && (cuts.met || l != 0) ? h : entered;
            if constexpr (SEQ) row_prefix_cut(H, P, cuts.absorb);
            else row_prefix(H, P);
            h = dpp_keep<kDppRowShr + 1, 0xf>(first, H);
#pragma unroll
            for (int j = 0; j < K; ++j) {
                const float b = du[j] * B[j];
                h = SEQ && cuts.at[j] ? b : __builtin_fmaf(a[j], h, b);
                y[j] = __builtin_fmaf(C[j], h, y[j]);
            }
            if (p.final_states) {
                const float final = row_lane(H, 15);
                after_l = l == n ? final : after_l;
            }
        }
        if (p.final_states && mine && l < nn)
            p.final_states[s * p.final_states_stride[0] + d * p.final_states_stride[1] + (n0 + l) * p.final_states_stride[2]] = after_l;
    }
#pragma unroll
    for (int j = 0; j < K; ++j) {
        if (p.z) y[j] *= silu(rz.get(j));
        y[j] = live[j] ? y[j] : 0.0f;
    }
    if (mine)
        store_steps<T, K>(static_cast<T*>(p.out) + s * p.out_stride[0] + d * p.out_stride[1], UNIT ? 1 : p.out_stride[2], t, end, y);
}

template <typename T> int launch_short(ScanFwdArgs a, bool unit, hipStream_t stream) {
    const cc1d_scan_params& p = a.p;
    a.group_blocks = ceil_div(p.dim / p.groups, 32);
    const dim3 grid((unsigned)(a.group_blocks * p.groups * p.batch)), block(512);
    return with_flag(p.seq_idx != nullptr, [&](auto seq) {
        return with_flag(unit, [&](auto un) {
            return launch(scan_fwd_short<T, decltype(seq)::value, decltype(un)::value>, grid, block, stream, a);
        });
    });
}

template <typename T, int K> int launch_rows(ScanFwdArgs a, bool unit, StateMode mode, hipStream_t stream) {
    const cc1d_scan_params& p = a.p;
    // A channel's states stay with one wavefront once the card has 512 blocks
    // (two a CU beside each other) of 8 channels; before, more wavefronts share them.
    const int64_t channels = scan_sequences(p) * p.dim, per = p.dim / p.groups;
    a.split = 8;
    while (a.split > 1 && channels > 512 * (8 / a.split) && per > 8 / a.split) a.split /= 2;
    a.group_blocks = ceil_div(per, 8 / a.split);
    const dim3 grid((unsigned)(a.group_blocks * p.groups * scan_sequences(p))), block(512);
    return with_flag(p.seq_idx != nullptr, [&](auto seq) {
        constexpr bool SEQ = decltype(seq)::value;
        if (!unit || mode == kStateAny) return launch(scan_fwd_rows<T, K, SEQ, false, kStateAny>, grid, block, stream, a);
        if (mode == kStateTime) return launch(scan_fwd_rows<T, K, SEQ, true, kStateTime>, grid, block, stream, a);
        return launch(scan_fwd_rows<T, K, SEQ, true, kStateLast>, grid, block, stream, a);
    });
}

template <typename T, int K> int launch_last(ScanFwdArgs a, StateMode mode, hipStream_t stream) {
    const cc1d_scan_params& p = a.p;
    a.group_blocks = ceil_div(p.dim / p.groups, 8);
    const dim3 grid((unsigned)(a.group_blocks * p.groups * scan_sequences(p))), block(512);
    return with_flag(p.seq_idx != nullptr, [&](auto seq) {
        return with_flag(mode == kStateTime, [&](auto tm) {
            return with_flag(p.dstate <= 128, [&](auto few) {
                constexpr StateMode MODE = decltype(tm)::value ? kStateTime : kStateLast;
                constexpr int NCAP = decltype(few)::value ? 128 : CC1D_MAX_DSTATE;
                return launch(scan_fwd_last<T, K, NCAP, decltype(seq)::value, MODE>, grid, block, stream, a);
            });
        });
    });
}

}  // namespace

int64_t scan_tile_floats(const cc1d_scan_params& p) { return scan_slots(p) * p.dim * p.dstate; }

int launch_scan_fwd(const cc1d_scan_params& p, hipStream_t stream) {
    const ScanFwdArgs a{p, 0, 1};
    return with_dtype(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        // Four channels a wavefront against one, or fewer channels with their states over several, us, 1 x dim x 40
        // bf16: the former's time hardly depends on dim (N = 16: 7.5, 32: 11.5, 64: 19.7, 128: 35.7, 256: 68), the
        // latter's does (N = 16: 6.1 at 64 channels, 9.4 at 1024; 64: 9.9, 14.1 at 512, 16.7 at 1024, 21.6 at 1536, 32
        // at 4096; 128: 26 at 1024, 36 at 1536 and 2048, 57 at 4096; 256: 66 at 1536 and 2048, 108 at 4096).
        if (scan_is_short(p) && (p.dstate <= 64 || p.batch * p.dim >= 2048))
            return launch_short<T>(a, p.seqlen >= kShortK && p.u_stride[2] == 1 && p.delta_stride[2] == 1 && p.out_stride[2] == 1 &&
                                          (!p.z || p.z_stride[2] == 1), stream);
        return with_flag(scan_tile(p.seqlen) == 512, [&](auto wide) {
            constexpr int K = decltype(wide)::value ? 8 : 4;
            const StateMode mode = state_mode<T, K>(p);
            const bool unit = p.seqlen >= K && p.u_stride[2] == 1 && p.delta_stride[2] == 1 && p.out_stride[2] == 1 &&
                              (!p.z || p.z_stride[2] == 1);
            const bool last = !unit && mode != kStateAny && p.dim >= elems16<T>::value && p.u_stride[1] == 1 &&
                              p.delta_stride[1] == 1 && p.out_stride[1] == 1 && (!p.z || p.z_stride[1] == 1);
            return last ? launch_last<T, K>(a, mode, stream) : launch_rows<T, K>(a, unit, mode, stream);
        });
    });
}

}  // namespace cc1d
