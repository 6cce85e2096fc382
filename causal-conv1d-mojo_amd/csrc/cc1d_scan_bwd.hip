// cc1d_scan_bwd.hip -- backward of the selective state space scan.
//
// With g[t] = dL/dh[t], and dy = dout (times silu(z) when gated):
//   g[t] = C[t] dy[t] + a[t+1] g[t+1],  w[t] = g[t] a[t] h[t-1]
//   du = D dy + dt sum_n g B        ddt = u sum_n g B + sum_n A w
//   dA = sum_t dt w                 dB[t] = sum_d g dt u,  dC[t] = sum_d dy h
#include "cc1d_scan_device.hpp"

namespace cc1d {
namespace {

struct ScanBwdArgs {
    cc1d_scan_bwd_params p;
    float* carry;        // (sequences, dim, dstate): a g of the position after the tile being worked on
    float* pA;           // (sequences, dim, dstate)
    float *pD, *pbias;   // (sequences, dim)
    float* pBC;          // (rows, groups, group_blocks, [B, C], dstate, span): each block's share of dB and dC
    int64_t group_blocks;
    // What this launch works on: rows (sequences) from `first` on, and of each its tiles tile0 .. tile1 - 1, which
    // are positions from t0 on, `span` at most.
    int64_t first, t0, span;
    int tile0, tile1;
};

template <typename T> __device__ void zero_uncovered(const cc1d_scan_bwd_params& p, int64_t d, int64_t from, int64_t to) {
    for (int64_t t = from + (threadIdx.x & 63); t < to; t += 64) {
        static_cast<T*>(p.du)[d * p.du_stride[1] + t * p.du_stride[2]] = T{};
        static_cast<T*>(p.ddelta)[d * p.ddelta_stride[1] + t * p.ddelta_stride[2]] = T{};
        if (p.fwd.z) static_cast<T*>(p.dz)[d * p.dz_stride[1] + t * p.dz_stride[2]] = T{};
    }
}

// What one channel's tile holds in registers.
template <int K> struct Channel {
    float dt[K], du[K], dy[K];       // du: dt u
    float y[K], along[K], wsum[K];   // sums over the states: C h, g B, A w
    float step_sum;
};

// One state of a channel. before / after: h ahead of the tile and a g behind
// it; on return after is a g of the tile's first position. dB, dC: the
// channel's terms are added. Returns the lane's share of the state's dA.
template <int K, bool CUT>
__device__ __forceinline__ float scan_state_bwd(Channel<K>& ch, float A, float before, float& after, const float (&B)[K],
                                                const float (&C)[K], float (&dB)[K], float (&dC)[K], const Cuts<K>& cuts,
                                                bool met_back, int lane) {
    float a[K], h[K];
    const float A2 = A * kLog2e;
#pragma unroll
    for (int j = 0; j < K; ++j) a[j] = __builtin_amdgcn_exp2f(ch.dt[j] * A2);
    float P = __builtin_amdgcn_exp2f(ch.step_sum * A2);
    float Pr = lane_get(P, 63 - lane);  // the lanes in reverse, for the prefix from the end
    float H = ch.du[0] * B[0];
#pragma unroll
    for (int j = 1; j < K; ++j) {
        const float b = ch.du[j] * B[j];
        H = CUT && cuts.at[j] ? b : __builtin_fmaf(a[j], H, b);
    }
    // Q = a g of the lane's first position
    float x = 0.0f;
#pragma unroll
    for (int j = K - 1; j >= 0; --j) {
        x = a[j] * __builtin_fmaf(C[j], ch.dy[j], x);
        if (CUT && cuts.at[j]) x = 0.0f;
    }
    float Q = lane_get(x, 63 - lane);
    const float first = lane == 0 ? before : 0.0f, behind = lane == 0 ? after : 0.0f;
    const float Hin = __builtin_fmaf(P, first, H), Qin = __builtin_fmaf(Pr, behind, Q);
    H = CUT && (cuts.met || lane != 0) ? H : Hin;
    Q = CUT && (met_back || lane != 0) ? Q : Qin;
    if constexpr (CUT) {
        wave_prefix_cut(H, P, cuts.absorb);
        wave_prefix_cut(Q, Pr, cuts.back);
    } else {
        wave_prefix2(H, P, Q, Pr);
    }
    const float ahead = dpp_keep<kDppWaveShr1, 0xf>(first, H);  // h before the lane's first position
    x = dpp_keep<kDppWaveShr1, 0xf>(behind, Q);                 // a g after its last one, lanes in reverse
    after = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(Q), 63));
    x = lane_get(x, 63 - lane);
    float v = ahead;
#pragma unroll
    for (int j = 0; j < K; ++j) {
        const float b = ch.du[j] * B[j];
        v = CUT && cuts.at[j] ? b : __builtin_fmaf(a[j], v, b);
        h[j] = v;
        ch.y[j] = __builtin_fmaf(C[j], v, ch.y[j]);
        dC[j] = __builtin_fmaf(ch.dy[j], v, dC[j]);
    }
    float dA = 0.0f;
#pragma unroll
    for (int j = K - 1; j >= 0; --j) {
        const float g = __builtin_fmaf(C[j], ch.dy[j], x);
        dB[j] = __builtin_fmaf(g, ch.du[j], dB[j]);
        ch.along[j] = __builtin_fmaf(g, B[j], ch.along[j]);
        x = a[j] * g;
        float w = x * (j > 0 ? h[j > 0 ? j - 1 : 0] : ahead);
        if (CUT && cuts.at[j]) x = w = 0.0f;
        ch.wsum[j] = __builtin_fmaf(A, w, ch.wsum[j]);
        dA = __builtin_fmaf(ch.dt[j], w, dA);
    }
    return dA;
}

// How u, delta, z, dout and their gradients lie: unit time stride, unit channel
// stride (through LDS), or any strides.
enum Layout { kRows, kLast, kAny };

// A wavefront's tile of one channel in LDS, as it lies in registers.
template <typename R> __device__ __forceinline__ void keep(uint32_t* lds, int lane, const R& r) {
    if constexpr (R::DW == 2) {
        reinterpret_cast<u32x2*>(lds)[lane] = u32x2{r.w[0], r.w[1]};
    } else {
#pragma unroll
        for (int q = 0; q < R::DW / 4; ++q)
            reinterpret_cast<u32x4*>(lds)[q * 64 + lane] = u32x4{r.w[4 * q], r.w[4 * q + 1], r.w[4 * q + 2], r.w[4 * q + 3]};
    }
}
template <typename R> __device__ __forceinline__ void kept(const uint32_t* lds, int lane, R& r) {
    if constexpr (R::DW == 2) {
        const u32x2 w = reinterpret_cast<const u32x2*>(lds)[lane];
        r.w[0] = w[0];
        r.w[1] = w[1];
    } else {
#pragma unroll
        for (int q = 0; q < R::DW / 4; ++q) {
            const u32x4 w = reinterpret_cast<const u32x4*>(lds)[q * 64 + lane];
#pragma unroll
            for (int j = 0; j < 4; ++j) r.w[4 * q + j] = w[j];
        }
    }
}

// A block: 8 wavefronts of CHW channels each, `rounds` times, of one group and
// sequence; tiles from the last to the first. In a tile, each round's channels
// run through 16 states at a time, each wavefront at others (of 16, in step i
// the two from 2 ((i + its number) mod 8) on), so that the block's sums for dB
// and dC of a state, in LDS, belong to one wavefront at a time and grow in a
// fixed order. (Added to by LDS atomics instead, 3870 us against 700 at
// 4 x 5120 x 2048 with 16 states.)
//
// Vector issue bounds it: 28.6 instructions per position, channel and state,
// which fill 74% of the time at that size. What remains is the barrier per two
// states and the start and end of each tile, which one block a CU does not
// cover. A barrier per state instead of two, in a row of launches at 4 x 5120 x
// 2048: 682 us against 719, channel-last 1100 against 1060, with ids 1092
// against 1081, fp32 854 against 858.
//
// Two channels a wavefront and their loads in flight are more than 256 registers
// hold in most forms: bytes of scratch a lane at 512 positions, 16-bit types and
// fp32: rows 0 and 136 (with ids 152 and 292), channel-last 276 and 560 (444 and
// 740), any strides 360 and 640 (540 and 812). Channel-last takes 1010 to 1060
// us at that size (fp32 1670), with ids in rows 1065.
constexpr int kWaves = 8;
template <typename T, int K, int CHW, bool SEQ, Layout LAY, StateMode MODE>
__global__ void __launch_bounds__(64 * kWaves, kWaves / 4) scan_bwd_rows(const ScanBwdArgs arg) {
    constexpr int TILE = 64 * K, CB = kWaves * CHW;
    constexpr bool UNIT = LAY == kRows, LAST = LAY == kLast;
    // (16 channels of 512 positions in 32 bits fill the 160 KB of a CU with no gap between rows)
    typedef ChannelTile<T, K, CB, 64 * kWaves, CB * TILE * sizeof(T) < 32768 ? elems16<T>::value : 0> Tile;
    __shared__ __attribute__((aligned(16))) float BC[2 * kStates * TILE];
    __shared__ __attribute__((aligned(16))) float acc[2 * kStates * TILE];
    // Rows: u, and delta where there is space, stay in LDS for the end of the tile
    // (fp32, 2 x 2048 x 4096: 408 us instead of 432; 16-bit types: no change).
    constexpr int KEEP = CB * TILE * (int)sizeof(T);
    constexpr bool KEEP_U = UNIT, KEEP_DELTA = UNIT && 2 * KEEP <= 32768;
    __shared__ __attribute__((aligned(16))) uint32_t stay[(KEEP_U ? KEEP : 16) / 4 + (KEEP_DELTA ? KEEP / 4 : 0)];
    __shared__ __attribute__((aligned(16))) T buf[LAST ? Tile::BYTES / sizeof(T) : 16 / sizeof(T)];
    const cc1d_scan_bwd_params& b = arg.p;
    const cc1d_scan_params& p = b.fwd;
    const int lane = threadIdx.x & 63, wave = (int)uniform32(threadIdx.x >> 6);
    const int64_t per = p.dim / p.groups;
    const uint32_t order = xcd_block(blockIdx.x, gridDim.x);
    const int64_t blk = order % arg.group_blocks, grp = order / arg.group_blocks % p.groups,
                  s = arg.first + order / arg.group_blocks / p.groups;
    const ScanSpan q = scan_span(p, s, TILE);
    const int N = (int)p.dstate;
    const int begin = (int)q.start, end = (int)(q.start + q.len), size = (int)p.seqlen;
    const T* Bp = static_cast<const T*>(p.B) + q.row * p.B_stride[0] + grp * p.B_stride[1];
    const T* Cp = static_cast<const T*>(p.C) + q.row * p.C_stride[0] + grp * p.C_stride[1];
    float* pBC = arg.pBC + (((q.row - arg.first) * p.groups + grp) * arg.group_blocks + blk) * 2 * N * arg.span;
    const int32_t* ids = SEQ ? p.seq_idx + q.row * p.seq_idx_stride[0] : nullptr;
    const int64_t is = SEQ ? p.seq_idx_stride[1] : 0;
    const int tiles = (int)((q.len + TILE - 1) / TILE);
    // In a round, neighbouring blocks take neighbouring channels: they share the lines of channel-last tensors.
    auto first_of = [&](int round) { return (round * arg.group_blocks + blk) * CB; };
    const int rounds = (int)(((per + CB - 1) / CB - blk + arg.group_blocks - 1) / arg.group_blocks);

    if (tiles == 0 || p.cu_seqlens) {
        for (int64_t i = wave; i < (int64_t)rounds * CB; i += kWaves) {
            const int64_t in_group = first_of((int)(i / CB)) + i % CB;
            if (in_group >= per) break;
            const int64_t d = grp * per + in_group;
            if (p.cu_seqlens && s == 0) zero_uncovered<T>(b, d, 0, q.start);
            if (p.cu_seqlens && s == p.num_seqs - 1) zero_uncovered<T>(b, d, q.start + q.len, p.seqlen);
            if (tiles > 0) continue;
            for (int n = lane; n < N; n += 64) {
                arg.pA[(s * p.dim + d) * N + n] = 0.0f;
                if (b.dinitial_states)
                    b.dinitial_states[(s * p.dim + d) * N + n] =
                        b.dfinal_states ? b.dfinal_states[s * b.dfinal_states_stride[0] + d * b.dfinal_states_stride[1] +
                                                          n * b.dfinal_states_stride[2]]
                                        : 0.0f;
            }
            if (lane == 0) arg.pD[s * p.dim + d] = arg.pbias[s * p.dim + d] = 0.0f;
        }
    }

    for (int tile = (tiles < arg.tile1 ? tiles : arg.tile1) - 1; tile >= arg.tile0; --tile) {
        const int t0 = begin + tile * TILE, t = t0 + lane * K;
        const bool full = end - t0 >= TILE, last = tile == tiles - 1;
        Cuts<K> cuts;
        bool live[K];
#pragma unroll
        for (int j = 0; j < K; ++j) live[j] = t + j < end;
        if constexpr (SEQ) cuts.read(ids, is, t, end - t, live);
        else cuts.none();
        const uint32_t bits = live_bits<K>(live);
        auto counts = [&](int j) { return SEQ ? live[j] : !LAST || full || live[j]; };  // (of rows, fix() clears the others)
        const bool met_back = SEQ && __shfl((int)cuts.met, 63 - lane) != 0;
        // With more than 16 states a block has one round, and its channels keep
        // their sums in registers from one lot of states to the next.
        for (int round = 0; round < rounds; ++round) {
            Channel<K> ch[CHW];
            int64_t d[CHW];
            bool mine[CHW];  // a missing channel is the group's last one with u, dout and states 0, and stores nothing
            const int64_t round_first = first_of(round);
            const int channels = (int)(per - round_first < CB ? per - round_first : CB), c0 = (int)(grp * per + round_first);
#pragma unroll
            for (int c = 0; c < CHW; ++c) {
                mine[c] = wave * CHW + c < channels;
                d[c] = c0 + (mine[c] ? wave * CHW + c : channels - 1);
            }
            // A round's share of a tensor: fetch() issues the loads, take() waits
            // for them (kLast: through LDS), give() stores.
            struct Rows {
                Raw<T, K> r[CHW];
            };
            typedef typename std::conditional<LAST, Tile, Rows>::type In;
            auto fetch = [&](In& in, const void* base, const int64_t* stride) {
                const T* row = static_cast<const T*>(base) + q.row * stride[0];
                if constexpr (LAST) {
                    in.load(row, stride[2], c0, (int)p.dim, t0, end);
                } else {
#pragma unroll
                    for (int c = 0; c < CHW; ++c) {
                        if constexpr (UNIT) in.r[c].load(row + d[c] * stride[1], t, size);
                        else in.r[c].each(row + d[c] * stride[1], stride[2], t, end);
                    }
                }
            };
            auto take = [&](In& in, Raw<T, K> (&r)[CHW]) {
                if constexpr (LAST) {
                    __syncthreads();
                    in.to_lds(buf, c0, (int)p.dim);
                    __syncthreads();
                }
#pragma unroll
                for (int c = 0; c < CHW; ++c) {
                    if constexpr (LAST) Tile::row(buf, (int)(d[c] - c0), lane, r[c]);
                    else r[c] = in.r[c];
                    if (UNIT && !full) r[c].fix(t, end, size);
                }
            };
            auto give = [&](void* base, const int64_t* stride, auto value) {
                T* row = static_cast<T*>(base) + q.row * stride[0];
                if constexpr (LAST) {
                    __syncthreads();
#pragma unroll
                    for (int c = 0; c < CHW; ++c) Tile::put_row(buf, wave * CHW + c, lane, value(c));
                    __syncthreads();
                    Tile::store(buf, row, stride[2], c0, channels, t0, end);
                } else {
#pragma unroll
                    for (int c = 0; c < CHW; ++c)
                        if (mine[c]) store_steps<T, K>(row + d[c] * stride[1], UNIT ? 1 : stride[2], t, end, value(c));
                }
            };
            auto stays = [&](int c) { return stay + (wave * CHW + c) * (KEEP / CB / 4); };
            float bias[CHW];
#pragma unroll
            for (int c = 0; c < CHW; ++c) bias[c] = p.delta_bias ? ld_uniform(p.delta_bias + d[c] * p.delta_bias_stride) : 0.0f;
            {
                In iu, id, iz, io;
                Raw<T, K> r[CHW];
                fetch(id, p.delta, p.delta_stride);
                fetch(iu, p.u, p.u_stride);
                take(id, r);
                if constexpr (KEEP_DELTA) {
#pragma unroll
                    for (int c = 0; c < CHW; ++c) keep(stays(c) + KEEP / 4, lane, r[c]);
                }
                fetch(io, b.dout, b.dout_stride);
#pragma unroll
                for (int c = 0; c < CHW; ++c) {
                    steps<K>(r[c], bias[c], p.delta_softplus != 0, ch[c].dt);
                    ch[c].step_sum = 0.0f;
#pragma unroll
                    for (int j = 0; j < K; ++j) {
                        if (SEQ || !full) ch[c].dt[j] = live[j] ? ch[c].dt[j] : 0.0f;
                        ch[c].step_sum += ch[c].dt[j];
                        ch[c].y[j] = ch[c].along[j] = ch[c].wsum[j] = 0.0f;
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
                take(iu, r);
                if constexpr (KEEP_U) {
#pragma unroll
                    for (int c = 0; c < CHW; ++c) keep(stays(c), lane, r[c]);
                }
                if (p.z) fetch(iz, p.z, p.z_stride);
#pragma unroll
                for (int c = 0; c < CHW; ++c)
#pragma unroll
                    for (int j = 0; j < K; ++j) ch[c].du[j] = mine[c] && counts(j) ? ch[c].dt[j] * r[c].get(j) : 0.0f;
                take(io, r);
#pragma unroll
                for (int c = 0; c < CHW; ++c)
#pragma unroll
                    for (int j = 0; j < K; ++j) ch[c].dy[j] = mine[c] && counts(j) ? r[c].get(j) : 0.0f;
                if (p.z) {
                    take(iz, r);
#pragma unroll
                    for (int c = 0; c < CHW; ++c)
#pragma unroll
                        for (int j = 0; j < K; ++j)
                            if (mine[c] && counts(j)) ch[c].dy[j] *= silu(r[c].get(j));
                }
            }
            for (int n0 = 0; n0 < N; n0 += kStates) {
                const int nn = N - n0 < kStates ? N - n0 : kStates;
                // lane i holds state n0 + i's
                float before_l[CHW], after_l[CHW], dA_l[CHW];
#pragma unroll
                for (int c = 0; c < CHW; ++c) {
                    before_l[c] = after_l[c] = dA_l[c] = 0.0f;
                    if (lane < nn && mine[c]) {
                        const int n = n0 + lane;
                        before_l[c] = p.tile_states[((q.slot + tile) * p.dim + d[c]) * N + n];
                        if (!last) after_l[c] = arg.carry[(s * p.dim + d[c]) * N + n];
                        else if (b.dfinal_states)
                            after_l[c] = b.dfinal_states[s * b.dfinal_states_stride[0] + d[c] * b.dfinal_states_stride[1] +
                                                         n * b.dfinal_states_stride[2]];
                        if (!last) dA_l[c] = arg.pA[(s * p.dim + d[c]) * N + n];
                    }
                }
                if (round == 0) {
                    StateRows<T, K, kWaves, MODE> rows;
                    rows.load(p, Bp, Cp, n0, nn, t0, end, size);
                    __syncthreads();  // the last lot is done with
                    rows.store(BC, n0, nn, N, t0, end, size, bits);
                    for (int i = threadIdx.x; i < 2 * kStates * TILE / 4; i += 64 * kWaves)
                        reinterpret_cast<f32x4*>(acc)[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                }
                __syncthreads();
                const int turn = (nn + kWaves - 1) / kWaves;  // states per wavefront between two barriers
#pragma unroll 1
                for (int i = 0; i < kWaves; ++i) {
#pragma unroll 1
                    for (int k = 0; k < turn; ++k) {
                        const int n = (i + wave) % kWaves * turn + k;
                        if (n >= nn) break;
                        float B[K], C[K], dB[K], dC[K];
                        read_state<K>(BC, n, lane, B);
                        read_state<K>(BC + kStates * TILE, n, lane, C);
                        read_state<K>(acc, n, lane, dB);
                        read_state<K>(acc + kStates * TILE, n, lane, dC);
#pragma unroll
                        for (int c = 0; c < CHW; ++c) {
                            const float A = ld_uniform(p.A + d[c] * p.A_stride[0] + (n0 + n) * p.A_stride[1]);
                            const float before = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(before_l[c]), n));
                            float after = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(after_l[c]), n));
                            const float dA = SEQ && cuts.any
                                ? scan_state_bwd<K, true>(ch[c], A, before, after, B, C, dB, dC, cuts, met_back, lane)
                                : scan_state_bwd<K, false>(ch[c], A, before, after, B, C, dB, dC, cuts, met_back, lane);
                            const float sum = wave_sum(dA);
                            dA_l[c] = lane == n ? dA_l[c] + sum : dA_l[c];
                            after_l[c] = lane == n ? after : after_l[c];
                            // one channel after the other: both at once would need more registers than there are
                            __builtin_amdgcn_sched_barrier(0);
                        }
#pragma unroll
                        for (int q = 0; q < K / 4; ++q) {
                            *reinterpret_cast<f32x4*>(acc + ((n * (K / 4) + q) * 64 + lane) * 4) =
                                f32x4{dB[4 * q], dB[4 * q + 1], dB[4 * q + 2], dB[4 * q + 3]};
                            *reinterpret_cast<f32x4*>(acc + kStates * TILE + ((n * (K / 4) + q) * 64 + lane) * 4) =
                                f32x4{dC[4 * q], dC[4 * q + 1], dC[4 * q + 2], dC[4 * q + 3]};
                        }
                    }
                    __syncthreads();
                }
#pragma unroll
                for (int c = 0; c < CHW; ++c) {
                    if (lane >= nn || !mine[c]) continue;
                    const int64_t at = (s * p.dim + d[c]) * N + n0 + lane;
                    arg.pA[at] = dA_l[c];
                    if (tile > 0) arg.carry[at] = after_l[c];
                    else if (b.dinitial_states) b.dinitial_states[at] = after_l[c];
                }
                if (round == rounds - 1) {
                    constexpr int ROWS = 2 * kStates / kWaves;
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) {
                        const int row = wave * ROWS + r, n = row % kStates;
                        if (n >= nn) continue;
                        float v[K];
                        read_state<K>(acc, row, lane, v);
                        float* to = pBC + ((row / kStates) * N + n0 + n) * arg.span + (t - arg.tile0 * TILE);
                        if (t + K <= end) {
#pragma unroll
                            for (int k = 0; k < K / 4; ++k)
                                *reinterpret_cast<AnyAddr<4>::v4*>(to + 4 * k) =
                                    u32x4{__float_as_uint(v[4 * k]), __float_as_uint(v[4 * k + 1]), __float_as_uint(v[4 * k + 2]),
                                          __float_as_uint(v[4 * k + 3])};
                        } else {
#pragma unroll
                            for (int j = 0; j < K; ++j)
                                if (t + j < end) to[j] = v[j];
                        }
                    }
                }
            }
            // The inputs again, from LDS or L2: to have kept them in registers would
            // have cost the states' loop its own. From here on along is du, wsum
            // ddelta and y dz.
            In iu, id, iz, io;
            Raw<T, K> r[CHW];
            if constexpr (!KEEP_U) fetch(iu, p.u, p.u_stride);
            if constexpr (!KEEP_DELTA) fetch(id, p.delta, p.delta_stride);
            if (KEEP_DELTA && p.z) fetch(io, b.dout, b.dout_stride);
            float dD[CHW], dbias[CHW];
            if constexpr (KEEP_U) {
#pragma unroll
                for (int c = 0; c < CHW; ++c) kept(stays(c), lane, r[c]);
            } else {
                take(iu, r);
            }
#pragma unroll
            for (int c = 0; c < CHW; ++c) {
                const float skip = p.D ? ld_uniform(p.D + d[c] * p.D_stride) : 0.0f;
                dD[c] = 0.0f;
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    const float u = counts(j) ? r[c].get(j) : 0.0f;
                    ch[c].wsum[j] = __builtin_fmaf(u, ch[c].along[j], ch[c].wsum[j]);
                    ch[c].along[j] = __builtin_fmaf(skip, ch[c].dy[j], ch[c].dt[j] * ch[c].along[j]);
                    ch[c].y[j] = __builtin_fmaf(skip, u, ch[c].y[j]);
                    dD[c] = __builtin_fmaf(ch[c].dy[j], u, dD[c]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (!KEEP_DELTA && p.z) fetch(io, b.dout, b.dout_stride);
            if (KEEP_DELTA && p.z) fetch(iz, p.z, p.z_stride);
            give(b.du, b.du_stride, [&](int c) -> const float(&)[K] { return ch[c].along; });
            if constexpr (KEEP_DELTA) {
#pragma unroll
                for (int c = 0; c < CHW; ++c) kept(stays(c) + KEEP / 4, lane, r[c]);
            } else {
                take(id, r);
            }
#pragma unroll
            for (int c = 0; c < CHW; ++c) {
                dbias[c] = 0.0f;
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    if (p.delta_softplus) ch[c].wsum[j] *= counts(j) ? sigmoid(r[c].get(j) + bias[c]) : 0.0f;
                    if (SEQ || !full) ch[c].wsum[j] = live[j] ? ch[c].wsum[j] : 0.0f;
                    dbias[c] += ch[c].wsum[j];
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (!KEEP_DELTA && p.z) fetch(iz, p.z, p.z_stride);
            give(b.ddelta, b.ddelta_stride, [&](int c) -> const float(&)[K] { return ch[c].wsum; });
            if (p.z) {
                take(io, r);
#pragma unroll
                for (int c = 0; c < CHW; ++c)
#pragma unroll
                    for (int j = 0; j < K; ++j) ch[c].y[j] *= r[c].get(j);
                take(iz, r);
#pragma unroll
                for (int c = 0; c < CHW; ++c)
#pragma unroll
                    for (int j = 0; j < K; ++j) ch[c].y[j] = counts(j) ? ch[c].y[j] * silu_grad(r[c].get(j)) : 0.0f;
                give(b.dz, b.dz_stride, [&](int c) -> const float(&)[K] { return ch[c].y; });
            }
#pragma unroll
            for (int c = 0; c < CHW; ++c) {
                const float sD = wave_sum(dD[c]), sb = wave_sum(dbias[c]);
                if (lane == 0 && mine[c]) {
                    const int64_t at = s * p.dim + d[c];
                    arg.pD[at] = last ? sD : arg.pD[at] + sD;
                    arg.pbias[at] = last ? sb : arg.pbias[at] + sb;
                }
            }
        }
    }
}

// Rows of at most 64 positions: a round of a block takes 32 channels. The LDS
// sums have a copy for each of a wavefront's four channels, added at the end.
template <typename T, bool SEQ, bool UNIT> __global__ void __launch_bounds__(512, 4) scan_bwd_short(const ScanBwdArgs arg) {
    constexpr int K = kShortK, TILE = 64 * K;
    __shared__ __attribute__((aligned(16))) float BC[2 * kStates * kShort];
    __shared__ __attribute__((aligned(16))) float acc[2 * kStates * TILE];
    const cc1d_scan_bwd_params& b = arg.p;
    const cc1d_scan_params& p = b.fwd;
    const int lane = threadIdx.x & 63, wave = (int)uniform32(threadIdx.x >> 6), l = lane & 15, t = l * K;
    const int end = (int)p.seqlen, N = (int)p.dstate;
    const int64_t per = p.dim / p.groups;
    const int64_t blk = blockIdx.x % arg.group_blocks, g = blockIdx.x / arg.group_blocks % p.groups,
                  row = blockIdx.x / arg.group_blocks / p.groups, s = arg.first + row;
    const T* const Bp = static_cast<const T*>(p.B) + s * p.B_stride[0] + g * p.B_stride[1];
    const T* const Cp = static_cast<const T*>(p.C) + s * p.C_stride[0] + g * p.C_stride[1];
    float* const pBC = arg.pBC + ((row * p.groups + g) * arg.group_blocks + blk) * 2 * N * p.seqlen;
    const int32_t* ids = SEQ ? p.seq_idx + s * p.seq_idx_stride[0] : nullptr;
    const int64_t is = SEQ ? p.seq_idx_stride[1] : 0;
    const int rounds = (int)(((per + 31) / 32 - blk + arg.group_blocks - 1) / arg.group_blocks);
    ShortCuts cuts;
    bool live[K];
#pragma unroll
    for (int j = 0; j < K; ++j) live[j] = t + j < end;
    if constexpr (SEQ) cuts.read(ids, is, t, end, live);
    else cuts.none();

    // (more than 16 states: one round)
    for (int round = 0; round < rounds; ++round) {
        const int64_t in_group = (round * arg.group_blocks + blk) * 32 + threadIdx.x / 16;
        const bool mine = in_group < per;  // a missing channel: the group's last one with u, dout and states 0
        const int64_t d = g * per + (mine ? in_group : per - 1), sd = s * p.dim + d;
        auto input = [&](Raw<T, K>& r, const void* base, const int64_t* stride) {
            const T* row = static_cast<const T*>(base) + s * stride[0] + d * stride[1];
            if constexpr (UNIT) r.load(row, t, end);
            else r.each(row, stride[2], t, end);
        };
        Raw<T, K> ru, rd, rz, ro;
        input(ru, p.u, p.u_stride);
        input(rd, p.delta, p.delta_stride);
        input(ro, b.dout, b.dout_stride);
        if (p.z) input(rz, p.z, p.z_stride);
        if constexpr (UNIT) {
            ru.fix(t, end, end);
            rd.fix(t, end, end);
            ro.fix(t, end, end);
            if (p.z) rz.fix(t, end, end);
        }
        const float bias = p.delta_bias ? p.delta_bias[d * p.delta_bias_stride] : 0.0f;
        const float skip = p.D ? p.D[d * p.D_stride] : 0.0f;
        float dt[K], du[K], dy[K], y[K], along[K], wsum[K], step_sum = 0.0f;
        steps<K>(rd, bias, p.delta_softplus != 0, dt);
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const bool in = mine && live[j];
            dt[j] = live[j] ? dt[j] : 0.0f;
            step_sum += dt[j];
            du[j] = in ? dt[j] * ru.get(j) : 0.0f;
            dy[j] = in ? ro.get(j) : 0.0f;
            if (p.z && in) dy[j] *= silu(rz.get(j));
            y[j] = along[j] = wsum[j] = 0.0f;
        }
        for (int n0 = 0; n0 < N; n0 += kStates) {
            const int nn = N - n0 < kStates ? N - n0 : kStates;
            float A_l = 0.0f, before_l = 0.0f, behind_l = 0.0f, dA_l = 0.0f, dinit_l = 0.0f;
            if (l < nn) {
                A_l = p.A[d * p.A_stride[0] + (n0 + l) * p.A_stride[1]];
                if (mine) before_l = p.tile_states[sd * N + n0 + l];
                if (mine && b.dfinal_states)
                    behind_l = b.dfinal_states[s * b.dfinal_states_stride[0] + d * b.dfinal_states_stride[1] +
                                               (n0 + l) * b.dfinal_states_stride[2]];
            }
            if (round == 0) {
                __syncthreads();  // the last lot is done with
                short_states<T>(BC, p, Bp, Cp, n0, nn, ids, is);
                for (int i = threadIdx.x; i < 2 * kStates * TILE / 4; i += 512)
                    reinterpret_cast<f32x4*>(acc)[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
            __syncthreads();
            const int turn = (nn + kWaves - 1) / kWaves;
#pragma unroll 1
            for (int i = 0; i < kWaves; ++i) {
#pragma unroll 1
                for (int k = 0; k < turn; ++k) {
                    const int n = (i + wave) % kWaves * turn + k;
                    if (n >= nn) break;
                    float B[K], C[K], dB[K], dC[K], a[K], h[K];
                    short_state(BC, n, l, B);
                    short_state(BC, kStates + n, l, C);
                    read_state<K>(acc, n, lane, dB);
                    read_state<K>(acc + kStates * TILE, n, lane, dC);
                    const float A = row_lane(A_l, n), A2 = A * kLog2e;
                    const float before = row_lane(before_l, n), after = row_lane(behind_l, n);
#pragma unroll
                    for (int j = 0; j < K; ++j) a[j] = __builtin_amdgcn_exp2f(dt[j] * A2);
                    float P = __builtin_amdgcn_exp2f(step_sum * A2), Pr = row_reverse(P);
                    float H = du[0] * B[0];
#pragma unroll
                    for (int j = 1; j < K; ++j) {
                        const float v = du[j] * B[j];
                        H = SEQ && cuts.at[j] ? v : __builtin_fmaf(a[j], H, v);
                    }
                    float x = 0.0f;
#pragma unroll
                    for (int j = K - 1; j >= 0; --j) {
                        x = a[j] * __builtin_fmaf(C[j], dy[j], x);
                        if (SEQ && cuts.at[j]) x = 0.0f;
                    }
                    float Q = row_reverse(x);
                    const float first = l == 0 ? before : 0.0f, behind = l == 0 ? after : 0.0f;
                    const float Hin = __builtin_fmaf(P, first, H), Qin = __builtin_fmaf(Pr, behind, Q);
                    H = SEQ && (cuts.met || l != 0) ? H : Hin;
                    Q = SEQ && (cuts.met_back || l != 0) ? Q : Qin;
                    if constexpr (SEQ) {
                        row_prefix_cut(H, P, cuts.absorb);
                        row_prefix_cut(Q, Pr, cuts.back);
                    } else {
                        row_prefix2(H, P, Q, Pr);
                    }
                    const float ahead = dpp_keep<kDppRowShr + 1, 0xf>(first, H);
                    x = row_reverse(dpp_keep<kDppRowShr + 1, 0xf>(behind, Q));
                    const float dinit = row_lane(Q, 15);
                    float v = ahead;
#pragma unroll
                    for (int j = 0; j < K; ++j) {
                        const float w = du[j] * B[j];
                        v = SEQ && cuts.at[j] ? w : __builtin_fmaf(a[j], v, w);
                        h[j] = v;
                        y[j] = __builtin_fmaf(C[j], v, y[j]);
                        dC[j] = __builtin_fmaf(dy[j], v, dC[j]);
                    }
                    float dA = 0.0f;
#pragma unroll
                    for (int j = K - 1; j >= 0; --j) {
                        const float gr = __builtin_fmaf(C[j], dy[j], x);
                        dB[j] = __builtin_fmaf(gr, du[j], dB[j]);
                        along[j] = __builtin_fmaf(gr, B[j], along[j]);
                        x = a[j] * gr;
                        float w = x * (j > 0 ? h[j > 0 ? j - 1 : 0] : ahead);
                        if (SEQ && cuts.at[j]) x = w = 0.0f;
                        wsum[j] = __builtin_fmaf(A, w, wsum[j]);
                        dA = __builtin_fmaf(dt[j], w, dA);
                    }
                    dA = lanes_sum<16>(dA);
                    dA_l = l == n ? dA : dA_l;
                    dinit_l = l == n ? dinit : dinit_l;
                    *reinterpret_cast<f32x4*>(acc + (n * 64 + lane) * 4) = f32x4{dB[0], dB[1], dB[2], dB[3]};
                    *reinterpret_cast<f32x4*>(acc + kStates * TILE + (n * 64 + lane) * 4) = f32x4{dC[0], dC[1], dC[2], dC[3]};
                }
                __syncthreads();
            }
            if (l < nn && mine) {
                arg.pA[sd * N + n0 + l] = dA_l;
                if (b.dinitial_states) b.dinitial_states[sd * N + n0 + l] = dinit_l;
            }
            if (round == rounds - 1) {
                for (int i = threadIdx.x; i < 2 * nn * end; i += 512) {
                    const int at = i % end, row = i / end, n = row < nn ? row : row - nn;
                    const float* sums = acc + (row < nn ? 0 : kStates * TILE) + (n * 64 + at / K) * 4 + at % K;
                    pBC[((row < nn ? 0 : N) + n0 + n) * p.seqlen + at] = (sums[0] + sums[64]) + (sums[128] + sums[192]);
                }
            }
        }
        float dD = 0.0f, dbias = 0.0f;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const float u = live[j] ? ru.get(j) : 0.0f;
            wsum[j] = __builtin_fmaf(u, along[j], wsum[j]);
            along[j] = __builtin_fmaf(skip, dy[j], dt[j] * along[j]);
            dD = __builtin_fmaf(dy[j], u, dD);
            if (p.delta_softplus) wsum[j] *= live[j] ? sigmoid(rd.get(j) + bias) : 0.0f;
            wsum[j] = live[j] ? wsum[j] : 0.0f;
            dbias += wsum[j];
            if (p.z) y[j] = live[j] ? ro.get(j) * __builtin_fmaf(skip, u, y[j]) * silu_grad(rz.get(j)) : 0.0f;
        }
        dD = lanes_sum<16>(dD);
        dbias = lanes_sum<16>(dbias);
        if (!mine) continue;
        auto give = [&](void* base, const int64_t* stride, const float (&v)[K]) {
            store_steps<T, K>(static_cast<T*>(base) + s * stride[0] + d * stride[1], UNIT ? 1 : stride[2], t, end, v);
        };
        give(b.du, b.du_stride, along);
        give(b.ddelta, b.ddelta_stride, wsum);
        if (p.z) give(b.dz, b.dz_stride, y);
        if (l == 0) {
            arg.pD[sd] = dD;
            arg.pbias[sd] = dbias;
        }
    }
}

// dB and dC of the launch's rows and positions (`count` of them): four positions
// per thread, the shares of the group's blocks in order; where that leaves the card idle, `split` threads take every split-th
// share each (1 x 6137 x 7, 8 states: 192 shares for 28 threads took 108 us).
template <typename T> __global__ void __launch_bounds__(256) scan_bwd_reduce_bc(const ScanBwdArgs arg, int64_t items, int64_t count, int split) {
    __shared__ f32x4 parts[256];
    const cc1d_scan_params& p = arg.p.fwd;
    const int64_t quads = (count + 3) / 4;
    const int wide = 256 / split, part = (int)threadIdx.x / wide;
    const int64_t idx = (int64_t)blockIdx.x * wide + threadIdx.x % wide;
    const int64_t t = idx % quads * 4, row = idx / quads, n2 = row % (2 * p.dstate), rg = row / (2 * p.dstate);
    const int have = idx < items ? (int)(count - t < 4 ? count - t : 4) : 0;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    const float* from = arg.pBC + (rg * arg.group_blocks * 2 * p.dstate + n2) * arg.span + t;
    const int64_t step = 2 * p.dstate * arg.span;
    if (have == 4) {
#pragma unroll 4
        for (int64_t k = part; k < arg.group_blocks; k += split) {
            const u32x4 v = *reinterpret_cast<const AnyAddr<4>::v4*>(from + k * step);
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[j] += __uint_as_float(v[j]);
        }
    } else {
        for (int64_t k = part; k < arg.group_blocks; k += split)
            for (int j = 0; j < have; ++j) sum[j] += from[k * step + j];
    }
    if (split > 1) {
        parts[threadIdx.x] = sum;
        __syncthreads();
        if (part > 0) return;
        for (int k = 1; k < split; ++k) sum += parts[threadIdx.x + k * wide];
    }
    const int64_t lo = p.cu_seqlens ? clamp_pos(p.cu_seqlens[0], p.seqlen) : 0;
    const int64_t hi = p.cu_seqlens ? clamp_pos(p.cu_seqlens[p.num_seqs], p.seqlen) : p.seqlen;
    const int64_t at = arg.t0 + t;
    T* to = static_cast<T*>(n2 < p.dstate ? arg.p.dB : arg.p.dC) +
            ((arg.first * p.groups + rg) * p.dstate + n2 % p.dstate) * p.seqlen + at;
    for (int j = 0; j < have; ++j) to[j] = from_f32<T>(at + j >= lo && at + j < hi ? sum[j] : 0.0f);
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

// What a block takes: its wavefronts' channels at a time (1 or 2), and with
// group_blocks how many rounds of them. What a launch takes: `rows` rows and
// `tiles` tiles of each, `span` positions.
struct BwdPlan {
    int chw;
    int64_t group_blocks, rows, tiles, span;
};

// `all` in parts of at most `most` (one at least), of about one size
int64_t evenly(int64_t all, int64_t most) { return ceil_div(all, ceil_div(all, most > 1 ? most : 1)); }

// The shares of dB and dC would otherwise grow with everything at once (17 GB
// at 8 x 8192 x 4096 with 128 states, where u has 0.5), so a call of more than
// this, 4 GiB, takes several launches, each followed by its sum: tiles from
// the last to the first, which leaves every launch all rows, and where one
// tile of all rows is too much, rows. That costs nothing (43.0 ms either way
// at that size); parts of 1 GiB cost up to 5% (45.0 there), as fewer blocks
// run beside each other at the end of each. Packed prompts (cu_seqlens) have
// one row and lengths that only the device knows: one launch. (Parts of the row,
// with the tiles that start in them: four prompts of 16384 x 1024 channels with
// 256 states run one after the other, 44.2 ms against 21.9, and the tiles' bounds
// kept in scalars cost other forms up to 5%.)
constexpr double kShareFloats = 1 << 30;

// A CU holds one block (128 KB of LDS and more; tiles of 256 positions have half
// of that, which is not counted), so the choice that leaves the card the least
// to do one after the other; a round of one channel each is taken for 2/3 of one
// of two. Measured where either fills the card, with 16 states, one and two
// channels, us: 4 x 5120 x 2048 bf16 850 and 719 (0.59 a round), channel-last
// 1150 and 1051, with ids 1137 and 1080, fp32 870 and 856; 4 x 2048 x 2048 fp32
// channel-last 693 and 713; 4 x 5120 x 200 122 and 129. Of equals the largest:
// its dB and dC have the fewest shares to add. More than 16 states: one round.
BwdPlan bwd_plan(const cc1d_scan_params& p) {
    const int64_t per = p.dim / p.groups, rows = scan_sequences(p) * p.groups;
    // Short rows: rounds once 1024 blocks (four wavefronts a SIMD, twice over) have some. From 512, 1024 and 4096 on, us,
    // 16 states bf16: 8 x 4096 x 64 53, 56, 56; 64 x 4096 x 64 297, 291, 305; 32 x 8192 x 64 288, 280, 297.
    if (scan_is_short(p)) {
        const int64_t blocks = ceil_div(per, 32), r = p.dstate > kStates ? 1 : ceil_div(rows * blocks, 1024);
        BwdPlan plan{0, ceil_div(blocks, r), p.batch, 1, p.seqlen};
        const double row = 2.0 * p.groups * plan.group_blocks * p.dstate * p.seqlen;
        if (p.batch * row > kShareFloats) plan.rows = evenly(p.batch, (int64_t)(kShareFloats / row));
        return plan;
    }
    BwdPlan best{0, 0, p.batch, INT32_MAX, p.seqlen};
    int64_t least = 0;
    for (int r = 1; r <= (p.dstate > kStates ? 1 : 8); ++r)
        for (int chw = 1; chw <= 2; ++chw) {
            const int64_t blocks = ceil_div(per, kWaves * chw * r);
            const int64_t cost = ceil_div(rows * blocks, 256) * r * (chw + 1);
            if (best.chw == 0 || cost <= least) {
                least = cost;
                best.chw = chw;
                best.group_blocks = blocks;
            }
        }
    const int64_t tile = scan_tile(p.seqlen);
    const double one = 2.0 * p.groups * best.group_blocks * p.dstate * tile;  // a tile's of a row
    if (p.cu_seqlens == nullptr && p.batch * (one / tile) * p.seqlen > kShareFloats) {
        best.tiles = evenly(ceil_div(p.seqlen, tile), (int64_t)(kShareFloats / (p.batch * one)));
        if (best.tiles == 1 && p.batch * one > kShareFloats) best.rows = evenly(p.batch, (int64_t)(kShareFloats / one));
        if (best.tiles * tile < p.seqlen) best.span = best.tiles * tile;
    }
    return best;
}

// rows: of the launch
template <typename T, int K> int launch_rows(const ScanBwdArgs& a, int chw, int64_t rows, hipStream_t stream) {
    const cc1d_scan_bwd_params& b = a.p;
    const cc1d_scan_params& p = b.fwd;
    const dim3 grid((unsigned)(a.group_blocks * p.groups * rows)), block(64 * kWaves);
    auto unit = [&](int i) {
        return p.u_stride[i] == 1 && p.delta_stride[i] == 1 && b.dout_stride[i] == 1 && b.du_stride[i] == 1 &&
               b.ddelta_stride[i] == 1 && (!p.z || (p.z_stride[i] == 1 && b.dz_stride[i] == 1));
    };
    const StateMode mode = state_mode<T, K>(p);
    const Layout lay = mode == kStateAny ? kAny : p.seqlen >= K && unit(2) ? kRows : p.dim >= elems16<T>::value && unit(1) ? kLast : kAny;
    return with_flag(p.seq_idx != nullptr, [&](auto seq) {
        return with_flag(chw == 2, [&](auto two) {
            constexpr bool SEQ = decltype(seq)::value;
            constexpr int CHW = decltype(two)::value ? 2 : 1;
            if (lay == kAny) return launch(scan_bwd_rows<T, K, CHW, SEQ, kAny, kStateAny>, grid, block, stream, a);
            return with_flag(mode == kStateTime, [&](auto tm) {
                constexpr StateMode MODE = decltype(tm)::value ? kStateTime : kStateLast;
                if (lay == kRows) return launch(scan_bwd_rows<T, K, CHW, SEQ, kRows, MODE>, grid, block, stream, a);
                return launch(scan_bwd_rows<T, K, CHW, SEQ, kLast, MODE>, grid, block, stream, a);
            });
        });
    });
}

template <typename T> int launch_short(const ScanBwdArgs& a, int64_t rows, hipStream_t stream) {
    const cc1d_scan_bwd_params& b = a.p;
    const cc1d_scan_params& p = b.fwd;
    const dim3 grid((unsigned)(a.group_blocks * p.groups * rows)), block(512);
    const bool unit = p.seqlen >= kShortK && p.u_stride[2] == 1 && p.delta_stride[2] == 1 && b.dout_stride[2] == 1 &&
                      b.du_stride[2] == 1 && b.ddelta_stride[2] == 1 && (!p.z || (p.z_stride[2] == 1 && b.dz_stride[2] == 1));
    return with_flag(p.seq_idx != nullptr, [&](auto seq) {
        return with_flag(unit, [&](auto un) {
            return launch(scan_bwd_short<T, decltype(seq)::value, decltype(un)::value>, grid, block, stream, a);
        });
    });
}

}  // namespace

int64_t scan_bwd_workspace_floats(const cc1d_scan_bwd_params& b) {
    const cc1d_scan_params& p = b.fwd;
    const BwdPlan plan = bwd_plan(p);
    return 2 * plan.rows * p.groups * plan.group_blocks * p.dstate * plan.span + scan_sequences(p) * p.dim * (2 * p.dstate + 2);
}

int launch_scan_bwd(const cc1d_scan_bwd_params& b, hipStream_t stream) {
    const cc1d_scan_params& p = b.fwd;
    const int64_t seqs = scan_sequences(p), states = seqs * p.dim * p.dstate, tile = scan_tile(p.seqlen);
    const BwdPlan plan = bwd_plan(p);
    ScanBwdArgs a{};
    a.p = b;
    a.group_blocks = plan.group_blocks;
    a.span = plan.span;
    a.carry = b.workspace;
    a.pA = a.carry + states;
    a.pD = a.pA + states;
    a.pbias = a.pD + seqs * p.dim;
    a.pBC = a.pbias + seqs * p.dim;
    // of a launch: rows (with cu_seqlens the sequences of the one row), and threads of its sum
    const int64_t rows = p.cu_seqlens != nullptr ? seqs : plan.rows;
    const int64_t most = plan.rows * p.groups * 2 * p.dstate * ceil_div(plan.span, 4);
    // Shares of dB and dC per thread of their sum: 1024 blocks of threads fill the card. Against one thread for all of
    // them and 32 everywhere, backward in all, us: 1 x 4096 x 512 with 16 states 57 (73 and 56), 4 x 2048 x 2041 326 (345
    // and 332), 4 x 5120 x 2048 721 (725 and 725), 1 x 8192 x 16384 2415 (2404 and 2426).
    int split = 1;
    while (split < 32 && most * split < 262144 && a.group_blocks >= 4 * split) split *= 2;
    const int64_t param_blocks = ceil_div(p.dim * (p.dstate + 2), 256);
    if (!threads_fit(a.group_blocks * p.groups * rows, 64 * kWaves) || !threads_fit(ceil_div(most * split, 256), 256) ||
        !threads_fit(param_blocks, 256))
        return CC1D_ERR_SHAPE;  // before any of them runs
    return with_dtype(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        int st = CC1D_OK;
        for (a.first = 0; st == CC1D_OK && a.first < seqs; a.first += rows) {
            const int64_t count = seqs - a.first < rows ? seqs - a.first : rows;  // of sequences
            const int64_t in_rows = p.cu_seqlens != nullptr ? 1 : count, all = ceil_div(p.seqlen, tile);
            for (int64_t w = all > plan.tiles ? ceil_div(all, plan.tiles) - 1 : 0; st == CC1D_OK && w >= 0; --w) {
                a.tile0 = (int)(w * plan.tiles);
                a.tile1 = (int)(plan.tiles < all ? (w + 1) * plan.tiles : INT32_MAX);
                a.t0 = a.tile0 * tile;
                const int64_t positions = p.seqlen - a.t0 < plan.span ? p.seqlen - a.t0 : plan.span;
                const int64_t items = in_rows * p.groups * 2 * p.dstate * ceil_div(positions, 4);
                if (scan_is_short(p)) st = launch_short<T>(a, count, stream);
                else
                    st = tile == 512 ? launch_rows<T, 8>(a, plan.chw, count, stream) : launch_rows<T, 4>(a, plan.chw, count, stream);
                if (st == CC1D_OK && items > 0)
                    st = launch(scan_bwd_reduce_bc<T>, dim3((unsigned)ceil_div(items * split, 256)), dim3(256), stream, a, items,
                                positions, split);
            }
        }
        if (st == CC1D_OK) st = launch(scan_bwd_reduce_params, dim3((unsigned)param_blocks), dim3(256), stream, a, seqs);
        return st;
    });
}

}  // namespace cc1d
