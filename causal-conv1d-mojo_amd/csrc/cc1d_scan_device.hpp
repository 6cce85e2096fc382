// cc1d_scan_device.hpp -- shared by the kernels of the selective state space scan.
//
// The recurrence h[t] = a[t] h[t-1] + b[t] (a = exp(dt A), b = dt u B) is a
// prefix over pairs (a, b) under (a2, b2) o (a1, b1) = (a2 a1, a2 b1 + b2). A
// wavefront takes one channel's tile of 64 K positions, K consecutive ones per
// lane: each lane runs its K steps from 0, the lanes' pairs are combined over
// the wavefront, and each lane runs its steps again from the state that
// reaches it. The decay over a lane's steps is one exponential, exp(A sum dt).
//
// Time lies along the lanes, and not channels, because a (batch, channel) row
// is then a wavefront's work of its own: 768 channels already fill the card
// without cutting the sequence into chunks that are walked twice. Per position
// and state the steps cost 7 issue slots (one exponential is two, measured 8
// cycles a wavefront against 4 for a multiply-add) and the wavefront's prefix
// 17 per K; channels along the lanes would cost 6, but fill the card from 5120
// channels x 4 rows on only, and 11 with the sequence cut into chunks. (Counts:
// that form was not built, nor one that also spreads a channel's states over
// wavefronts, which fills the card with fewer channels.)
#pragma once

#include "cc1d_internal.hpp"
#include "cc1d_steps.hpp"

namespace cc1d {

// Positions of a wavefront's tile, a rule on seqlen alone: 512 (8 a lane), or
// 256 where the row has no more, which would leave half the lanes idle.
__host__ __device__ constexpr int64_t scan_tile(int64_t seqlen) { return seqlen <= 256 ? 256 : 512; }

// dt = softplus(raw) = max(raw, 0) + log1p(e), e = exp(-|raw|), with
// log1p(e) = 2 atanh(s), s = e / (2 + e) <= 1/3, and atanh(s) / s a polynomial
// in s^2, fitted on [0, 1/9] at Chebyshev points (8e-9 off at most). Steps are
// small numbers (1e-3 and below), so the relative error counts, and
// log2(1 + e) would lose it. The exponent's rounding (|raw| log2(e) may reach
// 20) is taken back with the product's remainder.
__device__ __forceinline__ float softplus(float raw) {
    const float x = fminf(__builtin_fabsf(raw), 100.0f);
    const float q = -kLog2e * x;
    const float near = __builtin_amdgcn_exp2f(q);
    const float e = __builtin_fmaf(near * kLn2, __builtin_fmaf(-kLog2e, x, -q), near);
    const float s = e * __builtin_amdgcn_rcpf(2.0f + e);
    const float s2 = s * s;
    float p = __builtin_fmaf(s2, 0.1408732831f, 0.1398070902f);
    p = __builtin_fmaf(s2, p, 0.2001242638f);
    p = __builtin_fmaf(s2, p, 0.3333315849f);
    p = __builtin_fmaf(s2, p, 1.0f);
    return __builtin_fmaf(s + s, p, raw < 0.0f ? 0.0f : raw);  // (a NaN is not below 0)
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
inline int64_t scan_slots(const cc1d_scan_params& p) {
    const int64_t tile = scan_tile(p.seqlen);
    return p.cu_seqlens != nullptr ? p.seqlen / tile + p.num_seqs : p.batch * ceil_div(p.seqlen, tile);
}

constexpr int kShort = 64, kShortK = 4;

// Rows for the kernels of four channels a wavefront.
inline bool scan_is_short(const cc1d_scan_params& p) {
    return p.cu_seqlens == nullptr && p.batch * p.dim > 0 && p.seqlen >= 1 && p.seqlen <= kShort;
}

// dt of a lane's positions
template <int K, typename R> __device__ __forceinline__ void steps(const R& raw, float bias, bool soft, float (&dt)[K]) {
#pragma unroll
    for (int j = 0; j < K; ++j) dt[j] = raw.get(j) + bias;
    if (soft) {
#pragma unroll
        for (int j = 0; j < K; ++j) dt[j] = softplus(dt[j]);
    }
}

constexpr int kDppWaveShr1 = 0x138;  // lane l takes lane l - 1's value
constexpr int kDppRowShr = 0x110;    // + w: lane l takes lane l - w's, within 16 lanes

// Where a lane's steps and the wavefront's prefix must not reach across a
// sequence's start (seq_idx). All of it is the same for every state.
template <int K> struct Cuts {
    bool at[K];      // the state starts at 0 at the lane's step j
    bool met;        // ... at one of them
    bool absorb[6];  // level i of the prefix may take in the lanes it reads
    bool back[6];    // ... of the prefix from the end, lanes in reverse
    bool any;        // a lane of the wavefront has a cut

    __device__ __forceinline__ void none() {
        any = met = false;
#pragma unroll
        for (int j = 0; j < K; ++j) at[j] = false;
    }
    // ids of the row from its position 0; t the lane's first position, count of them in the row
    __device__ __forceinline__ void read(const int32_t* ids, int64_t stride, int64_t t, int count, bool (&live)[K]) {
        const int lane = threadIdx.x & 63;
        int32_t id[K];
        if (stride == 1 && count >= K) {
#pragma unroll
            for (int q = 0; q < K / 4; ++q) {
                const u32x4 w = *reinterpret_cast<const AnyAddr<4>::v4*>(ids + t + 4 * q);
#pragma unroll
                for (int j = 0; j < 4; ++j) id[4 * q + j] = (int32_t)w[j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < K; ++j) id[j] = j < count ? ids[(t + j) * stride] : 0;
        }
        const int32_t ahead = lane == 0 && t > 0 && count > 0 ? ids[(t - 1) * stride] : 0;
        int32_t prev = __builtin_amdgcn_update_dpp(ahead, id[K - 1], kDppWaveShr1, 0xf, 0xf, false);
        met = false;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            at[j] = j < count && (id[j] != prev || t + j == 0);
            live[j] = j < count && id[j] >= 0;
            met |= at[j];
            prev = id[j];
        }
        const uint64_t m = __ballot(met);
        any = m != 0;
        const uint64_t upto = m & (~0ull >> (63 - lane));
        const int last = upto ? 63 - __builtin_clzll(upto) : -1;  // the nearest lane at or before this one with a cut
#pragma unroll
        for (int i = 0; i < 4; ++i) absorb[i] = last + (1 << i) <= lane;
        absorb[4] = last < (lane & ~15);
        absorb[5] = last < 32;
        const uint64_t from = __builtin_bitreverse64(m) & (~0ull >> (63 - lane));
        const int next = from ? 63 - __builtin_clzll(from) : -1;  // the same of the reversed lanes
#pragma unroll
        for (int i = 0; i < 4; ++i) back[i] = next + (1 << i) <= lane;
        back[4] = next < (lane & ~15);
        back[5] = next < 32;
    }
};

// Inclusive prefix over the 64 lanes of the pairs (P, H): H becomes
// H + P H' + P P' H'' ... over the lanes before. A DPP operand reads the
// other lane's value in the multiply-add itself; lanes without a source (the
// row's first, or rows outside row_mask) keep what they hold. VALU results
// need two wait states before a DPP read, which asm has to provide itself.
#define CC1D_SCAN_LEVEL(H, P, CTRL) "v_fmac_f32_dpp " H ", " H ", " P " " CTRL "\n\t"
#define CC1D_SCAN_DECAY(P, CTRL) "v_mul_f32_dpp " P ", " P ", " P " " CTRL "\n\t"
#define CC1D_ROW(w) "row_shr:" w " row_mask:0xf bank_mask:0xf"
#define CC1D_B15 "row_bcast:15 row_mask:0xa bank_mask:0xf"
#define CC1D_B31 "row_bcast:31 row_mask:0xc bank_mask:0xf"
__device__ __forceinline__ void wave_prefix(float& H, float& P) {
    asm("s_nop 1\n\t"
        CC1D_SCAN_LEVEL("%0", "%1", CC1D_ROW("1")) CC1D_SCAN_DECAY("%1", CC1D_ROW("1")) "s_nop 0\n\t"
        CC1D_SCAN_LEVEL("%0", "%1", CC1D_ROW("2")) CC1D_SCAN_DECAY("%1", CC1D_ROW("2")) "s_nop 0\n\t"
        CC1D_SCAN_LEVEL("%0", "%1", CC1D_ROW("4")) CC1D_SCAN_DECAY("%1", CC1D_ROW("4")) "s_nop 0\n\t"
        CC1D_SCAN_LEVEL("%0", "%1", CC1D_ROW("8")) CC1D_SCAN_DECAY("%1", CC1D_ROW("8")) "s_nop 0\n\t"
        CC1D_SCAN_LEVEL("%0", "%1", CC1D_B15) CC1D_SCAN_DECAY("%1", CC1D_B15) "s_nop 0\n\t"
        CC1D_SCAN_LEVEL("%0", "%1", CC1D_B31) "s_nop 1"
        : "+v"(H), "+v"(P));
}
// Two prefixes at once: each fills the other's wait states.
__device__ __forceinline__ void wave_prefix2(float& H0, float& P0, float& H1, float& P1) {
#define CC1D_BOTH(CTRL) \
    CC1D_SCAN_LEVEL("%0", "%1", CTRL) CC1D_SCAN_LEVEL("%2", "%3", CTRL) CC1D_SCAN_DECAY("%1", CTRL) CC1D_SCAN_DECAY("%3", CTRL)
    asm("s_nop 1\n\t"
        CC1D_BOTH(CC1D_ROW("1")) CC1D_BOTH(CC1D_ROW("2")) CC1D_BOTH(CC1D_ROW("4")) CC1D_BOTH(CC1D_ROW("8"))
        CC1D_BOTH(CC1D_B15) CC1D_SCAN_LEVEL("%0", "%1", CC1D_B31) CC1D_SCAN_LEVEL("%2", "%3", CC1D_B31) "s_nop 1"
        : "+v"(H0), "+v"(P0), "+v"(H1), "+v"(P1));
#undef CC1D_BOTH
}
template <int CTRL, int ROW_MASK> __device__ __forceinline__ float dpp_keep(float keep, float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(keep), __float_as_int(v), CTRL, ROW_MASK, 0xf, false));
}
// The prefix where lanes with cuts take in nothing from before them: selected,
// not multiplied by 0, so that a non-finite state stays with its sequence.
__device__ __forceinline__ void wave_prefix_cut(float& H, float& P, const bool (&absorb)[6]) {
#define CC1D_CUT_LEVEL(I, CTRL, MASK)                                  \
    {                                                                  \
        const float h = dpp_keep<CTRL, MASK>(0.0f, H);                 \
        const float d = dpp_keep<CTRL, MASK>(1.0f, P);                 \
        H = absorb[I] ? __builtin_fmaf(P, h, H) : H;                 \
        P *= d;                                                        \
    }
    CC1D_CUT_LEVEL(0, kDppRowShr + 1, 0xf)
    CC1D_CUT_LEVEL(1, kDppRowShr + 2, 0xf)
    CC1D_CUT_LEVEL(2, kDppRowShr + 4, 0xf)
    CC1D_CUT_LEVEL(3, kDppRowShr + 8, 0xf)
    CC1D_CUT_LEVEL(4, kDppRowBcast15, 0xa)
    CC1D_CUT_LEVEL(5, kDppRowBcast31, 0xc)
}

// Rows of at most 64 positions: a wavefront takes four channels, 16 lanes of 4
// positions each, instead of one whose positions leave most lanes idle (bf16, 16
// states, 8 x 4096 x 64: 32 us forward and 74 backward instead of 79 and 210; at
// 14 x 6016 x 11 with 64 states 128 and 335 instead of 483 and 1718). What
// is one channel's in the kernels above is 16 lanes' there: prefixes end after
// four levels, and lane l holds what belongs to state l of 16.
__device__ __forceinline__ float row_lane(float v, int n) { return __shfl(v, (threadIdx.x & 48) | n); }  // of the 16 lanes
__device__ __forceinline__ float row_reverse(float v) { return dpp_f32<0x140, 0xf>(v); }
__device__ __forceinline__ void row_prefix(float& H, float& P) {
    asm("s_nop 1\n\t"
        CC1D_SCAN_LEVEL("%0", "%1", CC1D_ROW("1")) CC1D_SCAN_DECAY("%1", CC1D_ROW("1")) "s_nop 0\n\t"
        CC1D_SCAN_LEVEL("%0", "%1", CC1D_ROW("2")) CC1D_SCAN_DECAY("%1", CC1D_ROW("2")) "s_nop 0\n\t"
        CC1D_SCAN_LEVEL("%0", "%1", CC1D_ROW("4")) CC1D_SCAN_DECAY("%1", CC1D_ROW("4")) "s_nop 0\n\t"
        CC1D_SCAN_LEVEL("%0", "%1", CC1D_ROW("8")) "s_nop 1"
        : "+v"(H), "+v"(P));
}
__device__ __forceinline__ void row_prefix2(float& H0, float& P0, float& H1, float& P1) {
#define CC1D_BOTH(CTRL) \
    CC1D_SCAN_LEVEL("%0", "%1", CTRL) CC1D_SCAN_LEVEL("%2", "%3", CTRL) CC1D_SCAN_DECAY("%1", CTRL) CC1D_SCAN_DECAY("%3", CTRL)
    asm("s_nop 1\n\t"
        CC1D_BOTH(CC1D_ROW("1")) CC1D_BOTH(CC1D_ROW("2")) CC1D_BOTH(CC1D_ROW("4"))
        CC1D_SCAN_LEVEL("%0", "%1", CC1D_ROW("8")) CC1D_SCAN_LEVEL("%2", "%3", CC1D_ROW("8")) "s_nop 1"
        : "+v"(H0), "+v"(P0), "+v"(H1), "+v"(P1));
#undef CC1D_BOTH
}
struct ShortCuts {
    bool at[kShortK], met, met_back, absorb[4], back[4];

    __device__ __forceinline__ void none() {
        met = met_back = false;
#pragma unroll
        for (int j = 0; j < kShortK; ++j) at[j] = false;
    }
    // ids of the row; t the lane's first position
    __device__ __forceinline__ void read(const int32_t* ids, int64_t stride, int t, int end, bool (&live)[kShortK]) {
        const int l = threadIdx.x & 15;
        int32_t prev = t > 0 && t < end ? ids[(t - 1) * stride] : 0;
        met = false;
#pragma unroll
        for (int j = 0; j < kShortK; ++j) {
            const int32_t id = t + j < end ? ids[(t + j) * stride] : prev;
            at[j] = t + j < end && (id != prev || t + j == 0);
            live[j] = t + j < end && id >= 0;
            met |= at[j];
            prev = id;
        }
        const uint32_t m = (uint32_t)__ballot(met) & 0xffffu, r = __builtin_bitreverse32(m) >> 16, mask = (2u << l) - 1;
        const int last = (m & mask) ? 31 - __builtin_clz(m & mask) : -1, next = (r & mask) ? 31 - __builtin_clz(r & mask) : -1;
        met_back = r >> l & 1;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            absorb[i] = last + (1 << i) <= l;
            back[i] = next + (1 << i) <= l;
        }
    }
};
__device__ __forceinline__ void row_prefix_cut(float& H, float& P, const bool (&absorb)[4]) {
    CC1D_CUT_LEVEL(0, kDppRowShr + 1, 0xf)
    CC1D_CUT_LEVEL(1, kDppRowShr + 2, 0xf)
    CC1D_CUT_LEVEL(2, kDppRowShr + 4, 0xf)
    CC1D_CUT_LEVEL(3, kDppRowShr + 8, 0xf)
}
// B and C of states n0 .. n0 + nn - 1 (nn <= 16) of a short row to LDS, [B, C][state][position], by 512 threads.
template <typename T>
__device__ __forceinline__ void short_states(float* lds, const cc1d_scan_params& p, const T* B, const T* C, int n0, int nn,
                                             const int32_t* ids, int64_t id_stride) {
    for (int i = threadIdx.x; i < 2 * nn * kShort; i += 512) {
        const int t = i % kShort, row = i / kShort, n = row < nn ? row : row - nn;
        const bool in = t < (int)p.seqlen && (ids == nullptr || ids[t * id_stride] >= 0);
        const T* at = row < nn ? B + (n0 + n) * p.B_stride[2] + t * p.B_stride[3] : C + (n0 + n) * p.C_stride[2] + t * p.C_stride[3];
        lds[((row < nn ? 0 : 16) + n) * kShort + t] = in ? to_f32(*at) : 0.0f;
    }
}
__device__ __forceinline__ void short_state(const float* lds, int n, int l, float (&v)[kShortK]) {
    const f32x4 w = *reinterpret_cast<const f32x4*>(lds + n * kShort + 4 * l);
#pragma unroll
    for (int j = 0; j < kShortK; ++j) v[j] = w[j];
}

// A block's B and C of up to 16 states of a tile, fp32 in LDS as [B, C]
// [state][K / 4][lane] of four positions: a lane reads 16 bytes, the
// wavefront's contiguous. load() issues the reads, store() waits and writes,
// so the next tile's values travel while the current ones are used. Positions
// past the sequence and of an id < 0 are 0.
//   kStateTime   unit time stride: a wavefront of W carries 32 / W of the 32 rows
//   kStateLast   unit state stride (and at least 16 bytes of states): a thread
//                carries 16 bytes of states of one position, positions along
//                the lanes
//   kStateAny    the same, one by one, any strides
enum StateMode { kStateTime = 0, kStateLast = 1, kStateAny = 2 };
constexpr int kStates = 16;
template <typename T, int K, int WAVES, StateMode MODE> struct StateRows {
    static constexpr int E = elems16<T>::value, TILE = 64 * K, Q = K / 4, OCT = kStates / E;
    static constexpr int ROWS = MODE == kStateTime ? 2 * kStates / WAVES : 2 * OCT * K / WAVES;
    Raw<T, MODE == kStateTime ? K : E> raw[ROWS];

    // kStateLast, kStateAny: which 16 bytes turn r is about (uniform), and the position in the tile
    static __device__ __forceinline__ int unit(int r, int wave) { return (r * WAVES + wave) / K; }
    static __device__ __forceinline__ int pos(int r, int wave, int lane) { return (r * WAVES + wave) % K * 64 + lane; }

    // B, C: the batch row's and group's position 0 (rows of `size` positions); a tile from t0 on of a sequence
    // that ends at end
    __device__ __forceinline__ void load(const cc1d_scan_params& p, const T* B, const T* C, int n0, int nn, int t0, int end, int size) {
        const int lane = threadIdx.x & 63, wave = (int)uniform32(threadIdx.x >> 6);
        if constexpr (MODE == kStateTime) {
            const bool isC = wave * ROWS >= kStates;
            const int64_t ns = isC ? p.C_stride[2] : p.B_stride[2];
            const T* row = (isC ? C : B) + (n0 + wave * ROWS % kStates) * ns;
#pragma unroll
            for (int r = 0; r < ROWS; ++r)
                if (wave * ROWS % kStates + r < nn) raw[r].load(row + r * ns, t0 + lane * K, size);
        } else {
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const bool isC = unit(r, wave) >= OCT;
                const int n = unit(r, wave) % OCT * E, t = t0 + pos(r, wave, lane);
                if (n >= nn) continue;
                const int64_t ns = isC ? p.C_stride[2] : p.B_stride[2], ts = isC ? p.C_stride[3] : p.B_stride[3];
                const T* at = (isC ? C : B) + (t < end ? t : end - 1) * ts;
                if constexpr (MODE == kStateLast) raw[r].load(at, n0 + n, (int)p.dstate);
                else raw[r].each(at, ns, n0 + n, (int)p.dstate);
            }
        }
    }
    // live: bit j for the lane's position j, if it counts
    __device__ __forceinline__ void store(float* lds, int n0, int nn, int dstate, int t0, int end, int size, uint32_t live) {
        const int lane = threadIdx.x & 63, wave = (int)uniform32(threadIdx.x >> 6);
        if constexpr (MODE == kStateTime) {
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                if (wave * ROWS % kStates + r >= nn) continue;
                if (end - t0 < TILE) raw[r].fix(t0 + lane * K, end, size);
                float v[K];
#pragma unroll
                for (int j = 0; j < K; ++j) v[j] = live >> j & 1 ? raw[r].get(j) : 0.0f;
#pragma unroll
                for (int q = 0; q < Q; ++q)
                    *reinterpret_cast<f32x4*>(lds + (((wave * ROWS + r) * Q + q) * 64 + lane) * 4) =
                        f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
            }
        } else {
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                const int n = unit(r, wave) % OCT * E, t = pos(r, wave, lane);
                if (n >= nn) continue;
                if (MODE == kStateLast && n0 + n + E > dstate) raw[r].fix(n0 + n, dstate, dstate);
                const bool in = (uint32_t)__shfl((int)live, t / K) >> (t % K) & 1;
#pragma unroll
                for (int e = 0; e < E; ++e)
                    lds[((((unit(r, wave) / OCT) * kStates + n + e) * Q + (t / 4) % Q) * 64 + t / K) * 4 + t % 4] =
                        in ? raw[r].get(e) : 0.0f;
            }
        }
    }
};
template <int K> __device__ __forceinline__ uint32_t live_bits(const bool (&live)[K]) {
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < K; ++j) bits |= (uint32_t)live[j] << j;
    return bits;
}
template <int K> __device__ __forceinline__ void read_state(const float* lds, int n, int lane, float (&v)[K]) {
#pragma unroll
    for (int q = 0; q < K / 4; ++q) {
        const f32x4 w = *reinterpret_cast<const f32x4*>(lds + ((n * (K / 4) + q) * 64 + lane) * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * q + j] = w[j];
    }
}

// Tiles of channel-last tensors: a block's CB channels of TILE positions pass
// through LDS, [channel][position] with PAD elements between channels, so that both
// sides are whole accesses: in memory CB contiguous channels per position, in
// registers a lane's K consecutive positions of one channel. A thread carries
// 16 bytes of channels at two neighbouring positions, which are one write of
// two positions per channel in LDS.
template <typename T, int K, int CB, int THREADS, int PAD = elems16<T>::value> struct ChannelTile {
    static constexpr int TILE = 64 * K, E = elems16<T>::value, SEGS = CB / E, PAIRS = TILE / 2 * SEGS,
                         TURNS = (PAIRS + THREADS - 1) / THREADS, ROW = TILE + PAD;
    static constexpr int BYTES = CB * ROW * (int)sizeof(T);
    Raw<T, E> r[TURNS][2];

    static __device__ __forceinline__ bool has(int i) { return i * THREADS + (int)threadIdx.x < PAIRS; }
    static __device__ __forceinline__ int seg(int i) { return (i * THREADS + (int)threadIdx.x) % SEGS * E; }   // first channel
    static __device__ __forceinline__ int pos(int i) { return (i * THREADS + (int)threadIdx.x) / SEGS * 2; }   // first position

    // base: the batch row's position 0 and channel 0; c0 the block's first channel of `dim`; positions t0 .. end - 1
    __device__ __forceinline__ void load(const T* base, int64_t t_stride, int c0, int dim, int t0, int end) {
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
            if (!has(i)) continue;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int t = t0 + pos(i) + k;
                r[i][k].load(base + (t < end ? t : end - 1) * t_stride, c0 + seg(i), dim);  // (past the end: never used)
            }
        }
    }
    __device__ __forceinline__ void to_lds(T* buf, int c0, int dim) {
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
            if (!has(i)) continue;
            if (c0 + CB > dim) {
                r[i][0].fix(c0 + seg(i), dim, dim);
                r[i][1].fix(c0 + seg(i), dim, dim);
            }
#pragma unroll
            for (int e = 0; e < E; ++e) {
                T* at = buf + (seg(i) + e) * ROW + pos(i);
                if constexpr (sizeof(T) == 4) {
                    *reinterpret_cast<u32x2*>(at) = u32x2{r[i][0].w[e], r[i][1].w[e]};
                } else {
                    const uint32_t a = r[i][0].w[e / 2], b = r[i][1].w[e / 2];
                    *reinterpret_cast<uint32_t*>(at) = (e & 1) ? (a >> 16) | (b & 0xffff0000u) : (a & 0xffffu) | (b << 16);
                }
            }
        }
    }
    // A lane's K positions of channel c.
    static __device__ __forceinline__ void row(const T* buf, int c, int lane, Raw<T, K>& v) {
        const T* at = buf + c * ROW + lane * K;
        if constexpr (Raw<T, K>::DW == 2) {
            const u32x2 w = *reinterpret_cast<const u32x2*>(at);
            v.w[0] = w[0];
            v.w[1] = w[1];
        } else {
#pragma unroll
            for (int q = 0; q < Raw<T, K>::DW / 4; ++q) {
                const u32x4 w = reinterpret_cast<const u32x4*>(at)[q];
#pragma unroll
                for (int j = 0; j < 4; ++j) v.w[4 * q + j] = w[j];
            }
        }
    }
    static __device__ __forceinline__ void put_row(T* buf, int c, int lane, const float (&v)[K]) {
        T* at = buf + c * ROW + lane * K;
        if constexpr (Raw<T, K>::DW == 2) {
            *reinterpret_cast<u32x2*>(at) = u32x2{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
        } else {
#pragma unroll
            for (int q = 0; q < Raw<T, K>::DW / 4; ++q) reinterpret_cast<u32x4*>(at)[q] = vpack<T>(v + q * E);
        }
    }
    // LDS to memory: `channels` of them from c0 on.
    static __device__ __forceinline__ void store(const T* buf, T* base, int64_t t_stride, int c0, int channels, int t0, int end) {
#pragma unroll
        for (int i = 0; i < TURNS; ++i) {
            if (!has(i)) continue;
            uint32_t a[4], b[4];
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const T* at = buf + (seg(i) + e) * ROW + pos(i);
                if constexpr (sizeof(T) == 4) {
                    const u32x2 w = *reinterpret_cast<const u32x2*>(at);
                    a[e] = w[0];
                    b[e] = w[1];
                } else {
                    const uint32_t w = *reinterpret_cast<const uint32_t*>(at);
                    a[e / 2] = (e & 1) ? a[e / 2] | (w << 16) : w & 0xffffu;
                    b[e / 2] = (e & 1) ? b[e / 2] | (w & 0xffff0000u) : w >> 16;
                }
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int t = t0 + pos(i) + k;
                if (t >= end) continue;
                T* to = base + t * t_stride + c0 + seg(i);
                const u32x4 v = k == 0 ? u32x4{a[0], a[1], a[2], a[3]} : u32x4{b[0], b[1], b[2], b[3]};
                if (seg(i) + E <= channels) {
                    *reinterpret_cast<typename AnyAddr<sizeof(T)>::v4*>(to) = v;
                } else {
#pragma unroll
                    for (int e = 0; e < E; ++e)
                        if (seg(i) + e < channels) st_elem<T>(to + e, v, e);
                }
            }
        }
    }
};

// Blocks in XCD order: the hardware deals blocks out to the 8 XCDs in turns;
// here 8 neighbours run on one XCD and share its L2: the 128-byte lines that
// hold their channels in channel-last tensors, B and C of their sequence. No
// more than 8 in a row: sequences differ in length, and each has to be spread
// over all XCDs (whole sequences on one XCD: 605 us, 380 with none of this
// order, at eight prompts of 8192 positions x 4096 channels).
__device__ __forceinline__ uint32_t xcd_block(uint32_t b, uint32_t total) {
    const uint32_t base = b & ~63u;
    if (base + 64 > total) return b;
    return base + (b & 7) * 8 + ((b >> 3) & 7);
}

// How a call's B and C lie.
template <typename T, int K> StateMode state_mode(const cc1d_scan_params& p) {
    if (p.seqlen >= K && p.B_stride[3] == 1 && p.C_stride[3] == 1) return kStateTime;
    if (p.dstate >= elems16<T>::value && p.B_stride[2] == 1 && p.C_stride[2] == 1) return kStateLast;
    return kStateAny;
}

}  // namespace cc1d
