// cc1d_attn_kernels.hpp -- linear attention with a decay for each head, on
// the matrix cores.
//
// Per sequence and head S[t] = exp(g[t]) S[t-1] + k[t] v[t]^T and out[t] =
// scale q[t]^T S[t]. Over a chunk of C positions with c the inclusive sums of
// its g and M[i][j] = exp(c_i - c_j) for i >= j, else 0,
//     O     = scale (Q K^T o M) V + diag(exp c) scale Q S_in
//     S_out = exp(c_last) S_in + (diag(exp(c_last - c)) K)^T V,
// four matrix products a chunk. No exponent is ever positive for g <= 0, so
// nothing overflows however long the chunk's decay is.
//
// The gradients are the same operator on other operands (G the gradient of S
// after a position):
//     dQ: rows dO, columns V,  values K, state S^T, forwards in time
//     dK: rows V,  columns dO, values Q, state G^T, backwards
//     dV: rows K,  columns Q,  values dO, state G,  backwards
// (run backwards the decay between two positions is the same product, so g
// comes shifted by one position). One kernel computes all of them; a job says
// which operands it reads, which way, and where the scale goes.
//
// Precision: operands are held in LDS as bf16 planes whose sum is the value:
// one for bf16, two for fp16, three for fp32 (8 bits each), and products of
// planes are summed in fp32 by the MFMAs until what is left out is below the
// result's own rounding: planes a + b <= 1 (2^-17) where only 16-bit outputs
// follow, a + b <= 2 (2^-25) in fp32 and for the states, which are fp32
// whatever the type. bf16 planes have fp32's range, so nothing overflows on
// the way that fp32 holds.
#pragma once

#include "cc1d_internal.hpp"
#include "cc1d_scan_device.hpp"

namespace cc1d {

// Pointers and strides (batch, position, head, element) of one operand; head h
// reads the operand's head h / div.
struct AttnOperand {
    const void* p;
    int64_t s[4];
    uint32_t div;
};

struct AttnState {
    float* p;
    int64_t s[4];  // (sequence or segment slot, head, row, column)
};

struct AttnJob {
    AttnOperand a, b, c;  // rows, columns, values
    AttnOperand x;        // beside the outputs, for `dots` and `over`; p null: neither
    AttnState first;      // state before the first position; p null: 0
    AttnState last;       // state after the last; p null: not wanted
    AttnState seg;        // states between segments, by AttnSpan::between(); p null: whole sequences
    float* decay;         // (the same, heads): the decay of the segment walked before it
    void* out;            // (batch * seqlen, heads, dc) contiguous
    float* mark;          // states on the way, at multiples of `piece`, by AttnSpan::between(); null: not wanted
    float* tail;          // states before the sequences' last chunks (forwards); null: not wanted. Both: see kept_rows()
    int64_t piece, pieces;  // of marks: positions, a multiple of the chunk; of a row (without cu)
    float* dots;          // (heads, batch * seqlen): x with what the state gives the outputs; null: not wanted
    float* over;          // the same: the chunk's pairs over each position; null: not wanted
    int32_t da, dc;       // sizes of rows and columns, of values
    float p_scale, in_scale, w_scale;  // on the pairs, on what the state gives, on what it takes
    int32_t reverse, out_f32;
};

constexpr int kAttnJobs = 3;

struct AttnArgs {
    AttnJob job[kAttnJobs];
    const void* g;
    int64_t g_stride[3];
    const int32_t* cu;
    int64_t batch, seqlen, num_seqs;
    int64_t seg;  // positions of a segment, a multiple of the chunk
    uint32_t heads, jobs, slots, per_row;  // slots of all sequences; of one (without cu)
    FastDiv heads_div, jobs_div, row_div;
    uint32_t blocks;
};

template <typename T> struct AttnType;
template <> struct AttnType<bf16> { static constexpr int planes = 1, order = 1; };
template <> struct AttnType<f16> { static constexpr int planes = 2, order = 1; };
template <> struct AttnType<float> { static constexpr int planes = 3, order = 2; };

// Positions of a chunk: 64 where the images of that many leave two blocks and more to a CU (both directions of 4 x 2048,
// 32 heads of 64 x 64, fp16: 350 us, with 32 positions 418; but 8164 packed positions of 128 x 64: 580, with 32 468).
// Rows and columns may change places: dq, dk and dv need the same chunks.
constexpr int kMaxChunk = 64;
template <typename T> constexpr int chunk_of(int da, int dc) { return AttnType<T>::planes * (2 * da + dc) <= 384 ? kMaxChunk : 32; }
constexpr int attn_dim_of(int64_t d) { return d <= 64 ? 64 : 128; }  // a head of d is computed as one of this

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t uint16x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f32x4 mfma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// 2 N values as P planes of bf16, two to a dword
template <int P, int N> __device__ __forceinline__ void to_planes(const float (&v)[2 * N], uint32_t (&out)[P][N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const uint32_t w = pack2<bf16>(a, b);
            out[p][i] = w;
            if (p + 1 < P) {
                a -= __uint_as_float(w << 16);
                b -= __uint_as_float(w & 0xffff0000u);
            }
        }
    }
}
__device__ __forceinline__ bf16x8 as_frag(const uint32_t (&w)[4]) { return __builtin_bit_cast(bf16x8, w); }

// LDS images: rows of BLKS 16-byte blocks, block `blk` of a row permuted so
// that the 16 rows of a fragment lie in 16 different places of the 64 banks,
// and the four rows by four blocks of a transposing read as well.
template <int BLKS> __device__ __forceinline__ int swizzle(int row, int blk) {
    if constexpr (BLKS == 16) return blk ^ (4 * (row & 3) + ((row >> 2) & 3));
    else if constexpr (BLKS == 8) return blk ^ (4 * ((row >> 1) & 1) + ((row >> 2) & 3));
    else return blk ^ ((row >> 2) & 3);
}
// Byte offsets: row 16 t + (lane & 15), block b + (what the lane adds) is a base of the lane's, xor a constant of the
// tile's (b a multiple of what the lane adds at most).
template <int BLKS> __device__ __forceinline__ uint32_t frag_base(int l16, int blk, int half) {
    return (uint32_t)(l16 * BLKS * 16 + swizzle<BLKS>(l16, blk) * 16 + half * 8);
}
template <int BLKS> __device__ __forceinline__ uint32_t frag_tile(int t, int blk) { return (uint32_t)(t * 16 * BLKS * 16 | blk * 16); }
typedef __attribute__((address_space(3))) char lds_char;
template <typename V> __device__ __forceinline__ V lds_at(const uint16_t* image, uint32_t off) {
    return *reinterpret_cast<const V*>(reinterpret_cast<const char*>(image) + off);
}

// Fragments across an image's rows (its positions are the inner index of the
// product): ds_read_b64_tr_b16 gives lane l of 16 the l-th of the 16 columns
// that lanes 4 r .. 4 r + 3 name in row r, for four rows. Two neighbouring
// tiles share 32 columns in turns of four, lane l of tile t has
// tile_col(t, l), so that the accumulators of the two tiles hold eight
// neighbours in each lane, which is what a fragment of the next product (or a
// 16-byte store) wants.
__device__ __forceinline__ int tile_col(int t, int l16) { return 32 * (t >> 1) + 4 * (t & 1) + 8 * (l16 >> 2) + (l16 & 3); }
template <int BLKS> __device__ __forceinline__ uint32_t turn_base(int l16, int g4) {
    const int row = 8 * g4 + (l16 >> 2);
    return (uint32_t)(row * BLKS * 16 + swizzle<BLKS>(row, l16 & 3) * 16);
}
// positions 32 s .. of tile t, as a fragment
template <int BLKS> __device__ __forceinline__ u32x4 turn_at(const uint16_t* image, uint32_t base, int t, int s) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    lds_char* const at = (lds_char*)image;
    u32x2 w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const uint32_t off = base ^ (uint32_t)((32 * s + 4 * h) * BLKS * 16 | ((4 * (t >> 1)) ^ h) * 16 | (t & 1) * 8);
        w[h] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(at + off)));
    }
    return u32x4{w[0][0], w[0][1], w[1][0], w[1][1]};
}

// States that the backward leaves for the decays' gradient: (places, heads, columns, rows rounded up to whole vectors).
__host__ __device__ constexpr int64_t kept_rows(int64_t rows) { return (rows + 3) / 4 * 4; }

__device__ __forceinline__ float opaque_f32(float v) { return __int_as_float(opaque(__float_as_int(v))); }

// exp2 of a sum held in two floats: the second is at most an ulp of the first
__device__ __forceinline__ float exp2_sum(float hi, float lo) {
    return __builtin_amdgcn_exp2f(hi) * __builtin_fmaf(lo, 0.69314718f, 1.0f);
}

// Inclusive prefix sums over 64 lanes, in 64 bits.
template <int CTRL, int ROW_MASK> __device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROW_MASK, 0xf, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROW_MASK, 0xf, true);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ double wave_prefix_f64(double v) {
    v += dpp_f64<0x111, 0xf>(v);  // row_shr:1, 2, 4, 8
    v += dpp_f64<0x112, 0xf>(v);
    v += dpp_f64<0x114, 0xf>(v);
    v += dpp_f64<0x118, 0xf>(v);
    v += dpp_f64<kDppRowBcast15, 0xa>(v);
    v += dpp_f64<kDppRowBcast31, 0xc>(v);
    return v;
}
__device__ __forceinline__ double lane63(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)u, 63), hi = __builtin_amdgcn_readlane((int)(uint32_t)(u >> 32), 63);
    return __builtin_bit_cast(double, ((uint64_t)hi << 32) | lo);
}

// Sum over 16 neighbouring lanes, in every one of them.
__device__ __forceinline__ float sum16(float v) {
    v += dpp_f32<kDppQuadSwap1, 0xf>(v);
    v += dpp_f32<kDppQuadSwap2, 0xf>(v);
    v += dpp_f32<kDppRowRor4, 0xf>(v);
    v += dpp_f32<kDppRowRor8, 0xf>(v);
    return v;
}

// Sum over the four lanes that are 16 apart, in every one of them, and over those of them before this one. Swaps of rows
// in the vector unit: a lane permutation through LDS takes as long as an access, and one waits for the other.
__device__ __forceinline__ float sum_rows(float v, int row, float& before) {
    typedef unsigned two __attribute__((ext_vector_type(2)));
    const unsigned u = __float_as_uint(v);
    const two a = __builtin_bit_cast(two, __builtin_amdgcn_permlane16_swap(u, u, false, false));  // rows 0 0 2 2, 1 1 3 3
    const float even = __uint_as_float(a[0]), pair = even + __uint_as_float(a[1]);
    const unsigned w = __float_as_uint(pair);
    const two b = __builtin_bit_cast(two, __builtin_amdgcn_permlane32_swap(w, w, false, false));  // the lower pair, the upper
    const float low = __uint_as_float(b[0]);
    before = (row & 1 ? even : 0.0f) + (row & 2 ? low : 0.0f);
    return low + __uint_as_float(b[1]);
}

// A log decay as the sums take it: -1e5 stands for everything below (its
// exponential is 0), so that sums of -inf have differences.
__device__ __forceinline__ double log_decay(float g) { return g < -1e5f ? -1e5 : (double)g; }
// Below this a decay is 0: its exponential is less than the least normal number, 2^-126.
constexpr float kNoDecay = -87.33655f;

// Where a block works: a sequence's segment.
struct AttnSpan {
    int64_t seq, first, len;  // the sequence; its first position and length
    int64_t slot;             // of its first segment
    int64_t segs, index;      // its segments, and which of them this is
    int64_t states;           // where its states begin
    bool live;

    // Where the state between segments p - 1 and p of the sequence lies, 1 <= p < segs. A segment that another one
    // follows has `seg` whole positions and so holds one multiple of `seg` (of the packed row, or of its own), which
    // numbers it: (seqlen - 1) / seg states at most however many sequences there are, and none for those of one segment.
    __device__ __forceinline__ int64_t between(int64_t p) const { return states + p - 1; }
    // of the state before (after) this segment in its walk
    __device__ __forceinline__ int64_t before(bool reverse) const { return between(reverse ? segs - index : index); }
    __device__ __forceinline__ int64_t after(bool reverse) const { return between(reverse ? segs - 1 - index : index + 1); }
};

__device__ __forceinline__ AttnSpan attn_span(const AttnArgs& a, uint32_t slot) {
    AttnSpan s;
    if (a.cu == nullptr) {
        s.seq = a.row_div.div(slot);
        s.first = 0;
        s.len = a.seqlen;
        s.slot = s.seq * a.per_row;
        s.states = s.seq * (a.per_row - 1);
    } else {
        // Sequence i has the slots from cu[i] / seg + i on: the last that starts at or before this one. As many sequences
        // come before it as slots, less one for each segment that may have come in between; a lane looks at every step-th.
        int64_t lo = (int64_t)slot - ((int64_t)a.slots - a.num_seqs), hi = slot < a.num_seqs ? (int64_t)slot : a.num_seqs - 1;
        lo = lo < 0 ? 0 : lo;
        while (lo < hi) {
            const int64_t step = (hi - lo + 64) >> 6, at = lo + (int64_t)(threadIdx.x & 63) * step;
            const bool before = at <= hi && (uint32_t)clamp_pos(a.cu[at < hi ? at : hi], a.seqlen) / (uint32_t)a.seg + at <= slot;
            const uint64_t all = __ballot(before);
            const int last = all ? 63 - __builtin_clzll(all) : 0;
            lo += last * step;
            hi = hi < lo + step - 1 ? hi : lo + step - 1;
        }
        s.seq = lo;
        s.first = clamp_pos(ld_uniform(a.cu + lo), a.seqlen);
        s.len = clamp_pos(ld_uniform(a.cu + lo + 1), a.seqlen) - s.first;
        if (s.len < 0) s.len = 0;
        s.states = s.first / a.seg;
        s.slot = s.states + lo;
    }
    s.segs = s.len <= a.seg ? 1 : (s.len + a.seg - 1) / a.seg;
    s.index = (int64_t)slot - s.slot;
    s.live = s.index >= 0 && s.index < s.segs;
    return s;
}

// A chunk of one operand, from HBM into its image: bf16 of whole vectors goes
// straight there (global_load_lds), else through registers, where a value
// becomes its planes.
template <typename T, int C, int D, bool QUICK> struct AttnTile {
    static constexpr int EPV = elems16<T>::value, CGS = D / EPV, UNITS = C * CGS, N = UNITS / 256, P = AttnType<T>::planes;
    static constexpr bool DIRECT = QUICK && std::is_same_v<T, bf16>;
    static_assert(UNITS % 256 == 0, "whole turns of a block");
    u32x4 v[DIRECT ? 1 : N];

    // Vector n of a thread: its row and column; neighbouring lanes take neighbouring places of the image. tid: the
    // thread's index (not a loop invariant to the compiler: a register for every address would not leave enough for the
    // state).
    static __device__ __forceinline__ void unit(int n, int tid, int& row, int& col) {
        const int u = n * 256 + tid;
        row = u / CGS;
        col = u % CGS * EPV;
        if constexpr (DIRECT) col = swizzle<CGS>(row, u % CGS) * EPV;
    }
    // `rows` positions from base on, row_stride apart. QUICK: heads of whole vectors, next to each other, and chunks
    // that span less than 2 GiB, so that a uniform base and 32-bit offsets do.
    __device__ __forceinline__ void load(const T* base, int64_t row_stride, int64_t elem_stride, int rows, int d, uint16_t* image, int tid, int wave) {
        if constexpr (QUICK) {
            // (a whole turn of the block is R rows, and a thread's column the same in each)
            constexpr int R = 256 / CGS;
            int row, col;
            unit(0, tid, row, col);
            const bool down = row_stride < 0;
            const uint32_t pitch = (uint32_t)((down ? -row_stride : row_stride) * (int64_t)sizeof(T));
            const uint32_t at = (uint32_t)(down ? R - 1 - row : row) * pitch + col * (uint32_t)sizeof(T);
            const char* low = reinterpret_cast<const char*>(base) - (down ? (uint64_t)((R - 1) * pitch) : 0);
            const int64_t turn = (int64_t)(R * sizeof(T)) * row_stride;
            if constexpr (DIRECT) {
                if (rows == C && d == D) {
#pragma unroll
                    for (int n = 0; n < N; ++n, low += turn) direct(low + at, image, n, wave);
                    return;
                }
#pragma unroll
                for (int n = 0; n < N; ++n, low += turn) {
                    if (n * R + row < rows && col < d) direct(low + at, image, n, wave);
                    else *reinterpret_cast<u32x4*>(image + (n * 256 + tid) * 8) = vzero();
                }
            } else {
                // (without a branch, so that the loads on their way are counted, and what came before them is not waited
                // for with all of them: what is not the head's is read from its first row, and dropped by store())
#pragma unroll
                for (int n = 0; n < N; ++n, low += turn)
                    v[n] = vload_any(n * R + row < rows && col < d ? reinterpret_cast<const T*>(low + at) : base);
            }
        } else {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                int row, col;
                unit(n, tid, row, col);
                v[n] = vzero();
                if (row >= rows) continue;
                const T* const at = base + row * row_stride + col * elem_stride;
                if (elem_stride == 1 && col + EPV <= d) {
                    v[n] = vload_any(at);
                    continue;
                }
#pragma unroll
                for (int e = 0; e < EPV; ++e)
                    if (col + e < d) put(v[n], e, at[e * elem_stride]);
            }
        }
    }
    // vector n of a wavefront's lanes
    static __device__ __forceinline__ void direct(const char* at, uint16_t* image, int n, int wave) {
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)at,
                                         (__attribute__((address_space(3))) void*)(image + (n * 256 + wave * 64) * 8), 16, 0, 0);
    }
    static __device__ __forceinline__ void put(u32x4& w, int e, T x) {
        if constexpr (sizeof(T) == 4) w[e] = __float_as_uint(to_f32(x));
        else w[e >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, x) << (16 * (e & 1));
    }
    __device__ __forceinline__ void none() {
        if constexpr (!DIRECT)
#pragma unroll
            for (int n = 0; n < N; ++n) v[n] = vzero();
    }
    // image[plane][position][column]
    __device__ __forceinline__ void store(uint16_t* image, int rows, int d, int tid) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            int row, col;
            unit(n, tid, row, col);
            if constexpr (QUICK)
                if (!(row < rows && col < d)) v[n] = vzero();
            uint32_t w[P][EPV / 2];
            if constexpr (std::is_same_v<T, bf16>) {
#pragma unroll
                for (int i = 0; i < 4; ++i) w[0][i] = v[n][i];
            } else {
                float f[EPV];
#pragma unroll
                for (int e = 0; e < EPV; ++e) f[e] = vget<T>(v[n], e);
                to_planes<P, EPV / 2>(f, w);
            }
#pragma unroll
            for (int p = 0; p < P; ++p) {
                uint16_t* const at = image + (p * C + row) * D + swizzle<D / 8>(row, col >> 3) * 8 + (col & 7);
                if constexpr (EPV == 8) *reinterpret_cast<u32x4*>(at) = u32x4{w[p][0], w[p][1], w[p][2], w[p][3]};
                else *reinterpret_cast<u32x2*>(at) = u32x2{w[p][0], w[p][1]};
            }
        }
    }
};

// A row's 4 NT neighbouring outputs.
template <typename T, int NT> __device__ __forceinline__ void store_outputs(char* o, const f32x4 (&O)[NT], bool f32) {
    if (sizeof(T) == 4 || f32) {
#pragma unroll
        for (int m = 0; m < NT; ++m) *reinterpret_cast<AnyAddr<4>::v4*>(o + 16 * m) = __builtin_bit_cast(u32x4, O[m]);
    } else if constexpr (sizeof(T) == 2) {
        if constexpr (NT == 2) {
            *reinterpret_cast<AnyAddr<2>::v4*>(o) = u32x4{pack2<T>(O[0][0], O[0][1]), pack2<T>(O[0][2], O[0][3]),
                                                          pack2<T>(O[1][0], O[1][1]), pack2<T>(O[1][2], O[1][3])};
        } else {
            *reinterpret_cast<AnyAddr<2>::v2*>(o) = u32x2{pack2<T>(O[0][0], O[0][1]), pack2<T>(O[0][2], O[0][3])};
        }
    }
}

// One job of one segment of one head. Four wavefronts; each holds 16 * NT of
// the state's columns with all its rows in registers (the accumulators of
// S += K^T V), where they are at once the left operand of Q S. The pairs'
// products are shared: each wavefront forms those of 16 columns and passes
// them through LDS.
// MODE: outputs; outputs and exact states, where somebody wants the last one (the third plane of what the state
// takes); or the state alone, of the segments that another one follows. QUICK: whole vectors (attn_quick()); else
// operands are read element by element.
// GRADS: jobs of a backward, with x.
enum { kAttnOut = 0, kAttnExact = 1, kAttnStates = 2 };
template <typename T, int DA, int DC, int MODE, bool QUICK, bool GRADS>
__global__ void __launch_bounds__(256, QUICK && sizeof(T) == 2 && DC == 64 ? 3 : 2) attn_kernel(const AttnArgs args) {
    typedef AttnType<T> Ty;
    constexpr bool STATES = MODE == kAttnStates;
    constexpr int SORD = MODE == kAttnOut ? Ty::order : 2, SP = SORD + 1;  // planes of what the state takes
    constexpr int C = chunk_of<T>(DA, DC), P = Ty::planes, ORD = Ty::order, PP = ORD + 1;  // PP: planes of computed operands
    constexpr int NT = DC / 64, TA = DA / 16, SC = C / 32, SA = DA / 32, IT = C / 16;
    constexpr int PT = C == 64 ? 4 : 1;  // tiles of the pairs that a wavefront forms
    // In fp32 the products of lesser planes have sums of their own, so that a large sum is rounded once for a product of
    // the first planes and once for the rest, not by each of six. 2 x 2048, 40 heads of 128 x 128: outputs and gradients
    // off by 1.7e-7 to 1.9e-7 instead of 3.4e-7 to 3.8e-7. Free in heads of 64; in those of 128 x 128 registers are
    // short and both directions take 5 % longer.
    constexpr bool LESSER = std::is_same_v<T, float>;
    constexpr int LI = LESSER ? C / 16 : 0, LP = LESSER ? PT : 0;
    constexpr int kPairs = PP * C * C, kA = STATES ? 0 : (P * C * DA > kPairs ? P * C * DA : kPairs);
    __shared__ __attribute__((aligned(16))) uint16_t lds[kA + P * C * DA + P * C * DC];
    __shared__ __attribute__((aligned(16))) float sums_hi[2][C], sums_lo[2][C], into[2][C], left[2][C];
    __shared__ float whole[2];
    __shared__ __attribute__((aligned(16))) float dot_lds[GRADS ? 4 : 1][GRADS ? C : 1], over_lds[GRADS ? 4 : 1][GRADS ? C : 4];
    uint16_t *const ldsA = lds, *const ldsB = lds + kA, *const ldsC = ldsB + P * C * DA;
    uint16_t* const ldsP = ldsA;  // the rows are dead once their products are formed

    const int tid = threadIdx.x, wave = uniform32(tid >> 6), lane = tid & 63;
    const uint32_t id = xcd_block(blockIdx.x, args.blocks);
    const uint32_t rest = args.jobs_div.div(id), jn = id - rest * args.jobs;
    const uint32_t slot = args.heads_div.div(rest), h = rest - slot * args.heads;
    const AttnJob& job = args.job[jn];
    const AttnSpan sp = attn_span(args, slot);
    if (!sp.live || (STATES && sp.index + 1 == sp.segs)) return;
    const int64_t row0 = args.cu ? 0 : sp.seq;  // batch row
    const int da = job.da, dc = job.dc;
    const bool reverse = job.reverse;
    // positions of the sequence, in the order of the walk; segments begin and end at the same ones either way
    const int64_t early = reverse ? sp.segs * args.seg - sp.len : 0, from = sp.index * args.seg - early, to = from + args.seg;
    const int r_first = from > 0 ? (int)from : 0, r_end = (int)(to < sp.len ? to : sp.len);
    const int64_t dir = reverse ? -1 : 1, p0 = reverse ? sp.first + sp.len - 1 : sp.first;

    // position r of the walk
    auto base = [&](const AttnOperand& o, int r) {
        return static_cast<const T*>(o.p) + row0 * o.s[0] + (p0 + dir * r) * o.s[1] + (int64_t)(h / o.div) * o.s[2];
    };
    const bool dots = GRADS && job.dots != nullptr, over = GRADS && job.over != nullptr, beside = dots || over;
    const float p_scale = opaque_f32(job.p_scale);
    const T* const pg = static_cast<const T*>(args.g) + row0 * args.g_stride[0] + h * args.g_stride[2];

    // ---- the state at the segment's start
    f32x4 S[TA][NT];
#pragma unroll
    for (int t = 0; t < TA; ++t)
#pragma unroll
        for (int m = 0; m < NT; ++m) S[t][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const AttnState first = sp.index > 0 ? job.seg : job.first;
    if (!STATES && first.p != nullptr) {
        const float* const at = first.p + (sp.index > 0 ? sp.before(reverse) : sp.seq) * first.s[0] + h * first.s[1];
        const int s2 = (int)first.s[2], s3 = (int)first.s[3];
#pragma unroll
        for (int t = 0; t < TA; ++t)
#pragma unroll
            for (int m = 0; m < NT; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = tile_col(t, 4 * (lane >> 4) + e), col = tile_col(wave * NT + m, lane & 15);
                    const bool in = row < da && col < dc;
                    const float v = at[in ? (uint32_t)(row * s2 + col * s3) : 0u];
                    S[t][m][e] = in ? v : 0.0f;
                }
    }

    // ---- decays of the rows from r on (by one wavefront)
    typedef std::conditional_t<sizeof(T) == 4, uint32_t, uint16_t> Bits;
    double total = 0.0;
    auto g_load = [&](int r, int n) {
        // backwards, a position's decay is the one of the position after it, and the sequence's last has none
        const T* const at = pg + (p0 + dir * r + (reverse ? 1 : 0)) * args.g_stride[1];
        uint32_t g = 0;  // (bits: converted where they are used, so that nothing waits for them here)
        if (lane < n && !(reverse && r + lane == 0)) g = *reinterpret_cast<const Bits*>(at + lane * (dir * args.g_stride[1]));
        return g;
    };
    auto decays = [&](uint32_t bits, int buf) {
        const float g = to_f32(__builtin_bit_cast(T, (Bits)(uint32_t)opaque((int)bits)));
        const double c = wave_prefix_f64(log_decay(g) * 1.4426950408889634), end = lane63(c);
        total += end;
        const float hi = (float)c, lo = (float)(c - (double)hi);
        const float ehi = (float)end, elo = (float)(end - (double)ehi);
        if (lane < C) {
            sums_hi[buf][lane] = hi;
            sums_lo[buf][lane] = lo;
            into[buf][lane] = exp2_sum(hi, lo) * job.in_scale;
            left[buf][lane] = __builtin_amdgcn_exp2f((ehi - hi) + (elo - lo)) * job.w_scale;
        }
        if (lane == 0) whole[buf] = exp2_sum(ehi, elo);
    };

    // ---- operands: where the next chunk starts, and the step from row to row
    AttnTile<T, C, DA, QUICK> ta, tb;
    AttnTile<T, C, DC, QUICK> tc;
    constexpr bool DIRECT = decltype(ta)::DIRECT;
    const T *pa = base(job.a, r_first), *pb = base(job.b, r_first), *pc = base(job.c, r_first), *px = beside ? base(job.x, r_first) : nullptr;
    const int64_t sa = dir * job.a.s[1], sb = dir * job.b.s[1], sc = dir * job.c.s[1], sx = dir * job.x.s[1];
    const int64_t ea = job.a.s[3], eb = job.b.s[3], ec = job.c.s[3], ex = job.x.s[3];
    // the next n rows, and on past them
    auto load = [&](int n, int t) {
        if constexpr (!STATES) ta.load(pa, sa, ea, n, da, ldsA, t, wave);
        tb.load(pb, sb, eb, n, da, ldsB, t, wave);
        tc.load(pc, sc, ec, n, dc, ldsC, t, wave);
        pa += n * sa;
        pb += n * sb;
        pc += n * sc;
    };
    // Chunks begin at multiples of C from the segment's first position either way: backwards, the partial one comes first.
    const int head = reverse ? (r_end - r_first) % C : 0;
    auto rows_at = [&](int r) { return r == r_first && head > 0 ? head : r_end - r < C ? r_end - r : C; };
    // A word of each 128 bytes of the next n rows, so that what goes straight into its image comes from the L2 cache when
    // its turn has come (two wavefronts to an operand). Not long before: the blocks of an XCD work on about as much as
    // its L2 holds, and lines fetched a whole chunk ahead were gone when they were wanted. 4 x 2048, 40 heads of 128 x
    // 128, bf16: forward 187 us without, 161 from the chunk's start, 165 from its middle; backward 309 (0.88 GB read),
    // 322 (1.47 GB) and 308 (0.99 GB).
    uint32_t ahead[2] = {0, 0};
    auto fetch = [&](int n, int t) {
        auto word = [&](const T* p, int64_t s, int d, int lines, uint32_t& to) {
            const int row = lines == 2 ? (t & 127) >> 1 : t & 63, at = lines == 2 ? (t & 1) * 64 : 0;
            if (row < n && at < d) to = *reinterpret_cast<const uint32_t*>(p + row * s + at);
        };
        if (wave >= 2) word(pb, sb, da, DA / 64, ahead[0]);
        else if (!STATES) word(pa, sa, da, DA / 64, ahead[0]);
        if (wave < 2) word(pc, sc, dc, DC / 64, ahead[1]);
    };

    // ---- outputs: a lane has NT * 4 neighbouring columns of row 16 it + (lane & 15)
    const int64_t tokens = args.batch * args.seqlen, t0 = row0 * args.seqlen + p0;
    const int osize = job.out_f32 ? 4 : (int)sizeof(T);
    const int64_t opitch = (int64_t)args.heads * dc * osize;  // bytes from token to token
    char* out = static_cast<char*>(job.out) + (t0 + dir * r_first) * opitch + (int64_t)h * dc * osize;
    auto dots_out = [&](int r) {
        const int64_t at = h * tokens + t0 + dir * (r + tid);
        if constexpr (GRADS) {
            if (dots) job.dots[at] = (dot_lds[0][tid] + dot_lds[1][tid]) + (dot_lds[2][tid] + dot_lds[3][tid]);
            if (over) job.over[at] = (over_lds[0][tid] + over_lds[1][tid]) + (over_lds[2][tid] + over_lds[3][tid]);
        }
    };
    // Where in the walk the state is wanted next, after `at`. (What it needs is read again each time: kept, it would take
    // scalar registers that the loop has not got.)
    auto job_again = [&]() -> const AttnJob& { return args.job[uniform32(opaque((int)jn))]; };
    auto stop_after = [&](int at) {
        const AttnJob& again = job_again();
        int stop = 0x7fffffff;
        if (again.mark != nullptr) {
            const int piece = (int)again.piece, rest = (int)sp.len % piece, base = reverse && rest > 0 ? rest : piece;
            stop = at < base ? base : base + ((at - base) / piece + 1) * piece;
        }
        const int tail = ((int)sp.len - 1) / C * C;
        return again.tail != nullptr && tail > at && tail < stop ? tail : stop;
    };
    int stop = 0x7fffffff;
    if constexpr (GRADS) stop = stop_after(r_first - 1);

    // x, in vectors of XE values: for `dots` beside the outputs, a row's NT * 4 neighbours; for `over` as a left operand
    // of NS products of 32 columns, 16 rows of x a wavefront (in chunks of 32 half of their columns). As many vectors
    // either way, and no branch between them: it would wait for the loads.
    constexpr int XE = sizeof(T) == 2 && NT == 2 ? 8 : 4, XR = NT * 4 / XE, XN = IT * XR, NS = C == 64 ? DC / 32 : DC / 64;
    static_assert(XN * XE == NS * 8, "two layouts of as many values");
    typedef uint32_t xvec __attribute__((ext_vector_type(XE * sizeof(T) / 4)));
    typedef std::conditional_t<sizeof(xvec) == 16, typename AnyAddr<sizeof(T)>::v4, typename AnyAddr<sizeof(T)>::v2> xword;
    xvec xr[GRADS ? XN : 1];
    auto x_at = [&](int unit, int e) {
        u32x4 w = vzero();
#pragma unroll
        for (int i = 0; i < (int)(XE * sizeof(T) / 4); ++i) w[i] = xr[unit][i];
        return vget<T>(w, e);
    };
    const int xt = C == 64 ? wave : wave & 1, xs = C == 64 ? 0 : (wave >> 1) * NS;
    auto load_x = [&](const T* const from, int count, int t) {
        const int l16 = t & 15, g4 = (t >> 4) & 3, col = NT == 2 ? 32 * wave + 8 * g4 : 32 * (wave >> 1) + 4 * (wave & 1) + 8 * g4;
#pragma unroll
        for (int i = 0; i < XN; ++i) {
            const int tile = dots ? i / XR : xt;
            const int c = dots ? col + XE * (i % XR) : 32 * (xs + i * XE / 8) + 8 * g4 + i * XE % 8;
            const bool in = 16 * tile + l16 < count && c < dc;
            u32x4 w = vzero();
            if constexpr (QUICK) {
                const char* const low = reinterpret_cast<const char*>(from) + ((reverse ? 15 : 0) + 16 * tile) * sx * (int64_t)sizeof(T);
                const uint32_t at = (uint32_t)(reverse ? 15 - l16 : l16) * (uint32_t)((reverse ? -sx : sx) * (int64_t)sizeof(T)) + (uint32_t)(c * (int)sizeof(T));
                xr[i] = xvec(0u);
                if (in) xr[i] = *reinterpret_cast<const xword*>(low + at);
            } else {
                const T* const p = from + (16 * tile + l16) * sx + c * ex;
                xr[i] = xvec(0u);
                if (in && ex == 1 && c + XE <= dc) {
                    xr[i] = *reinterpret_cast<const xword*>(p);
                    continue;
                }
#pragma unroll
                for (int e = 0; e < XE; ++e)  // (as AttnTile::load())
                    if (in && c + e < dc) decltype(ta)::put(w, e, p[e * ex]);
#pragma unroll
                for (int k = 0; k < (int)(XE * sizeof(T) / 4); ++k) xr[i][k] = w[k];
            }
        }
    };

    // Registers load a chunk while the block works on the one before; what goes straight into its image is waited for
    // while the CU's other blocks work. The first turn only loads (or only forms the decays).
    int r = r_first, n = 0, buf = 1;
    if constexpr (GRADS && !DIRECT)
        if (beside) load_x(px, rows_at(r_first), opaque(tid));
    ta.none();
    tb.none();
    tc.none();
    for (;;) {
        const int otid = opaque(tid), l16 = otid & 15, g4 = (otid >> 4) & 3;
        const int n_next = rows_at(r + n);
        uint32_t g_next = 0;
        // ---- the chunk into LDS
        if constexpr (DIRECT) {
            if (n > 0) load(n, otid);
            if (wave == 3 && n_next > 0) g_next = g_load(r + n, n_next);
            asm volatile("s_waitcnt vmcnt(0)" ::"v"(ahead[0]), "v"(ahead[1]) : "memory");
        } else {
            if constexpr (!STATES) ta.store(ldsA, n, da, otid);
            tb.store(ldsB, n, da, otid);
            tc.store(ldsC, n, dc, otid);
            // (x is here by now; where it is used, a wait would be for the next chunk as well)
            if constexpr (GRADS) __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
        }
        __syncthreads();
        const int col = NT == 2 ? 32 * wave + 8 * g4 : 32 * (wave >> 1) + 4 * (wave & 1) + 8 * g4;
        const bool full = n == C && dc == DC;
        if (n_next > 0) {
            if constexpr (!DIRECT) {
                if (wave == 3) g_next = g_load(r + n, n_next);
                load(n_next, otid);
            } else if (n == 0) {
                fetch(n_next, otid);
            }
        }
        if (n > 0) {
            const uint32_t fragD = frag_base<DA / 8>(l16, g4, 0);
            const uint32_t fragC = frag_base<C / 8>(l16, g4, 0), halfC = frag_base<C / 8>(l16, g4 >> 1, g4 & 1);
            const uint32_t turnB = turn_base<DA / 8>(l16, g4), turnC = turn_base<DC / 8>(l16, g4);
            f32x4 O[IT][NT];
            if constexpr (!STATES) {
                // ---- what the state gives, and the pairs, transposed (columns x rows), so that a lane gets four columns
                // of a row: both from one reading of the rows
                const int jt = C == 64 ? wave : wave & 1, it0 = C == 64 ? 0 : wave >> 1;  // this wavefront's columns; its first rows
                f32x4 acc[PT];
#pragma unroll
                for (int k = 0; k < PT; ++k) acc[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int it = 0; it < IT; ++it)
#pragma unroll
                    for (int m = 0; m < NT; ++m) O[it][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                f32x4 lesser[LI + 1][NT], few[LP + 1];
#pragma unroll
                for (int it = 0; it < LI; ++it)
#pragma unroll
                    for (int m = 0; m < NT; ++m) lesser[it][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < LP; ++k) few[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int s = 0; s < SA; ++s) {
                    bf16x8 fb[P];
#pragma unroll
                    for (int p = 0; p < P; ++p) fb[p] = lds_at<bf16x8>(ldsB + p * C * DA, fragD ^ frag_tile<DA / 8>(jt, 4 * s));
                    uint32_t sw[NT][PP][4];
#pragma unroll
                    for (int m = 0; m < NT; ++m) {
                        float f[8];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            f[e] = S[2 * s][m][e];
                            f[4 + e] = S[2 * s + 1][m][e];
                        }
                        to_planes<PP, 4>(f, sw[m]);
                    }
                    // (products that follow each other add to different sums)
#pragma unroll
                    for (int q = 0; q < P; ++q) {
                        bf16x8 fq[IT];
#pragma unroll
                        for (int it = 0; it < IT; ++it) fq[it] = lds_at<bf16x8>(ldsA + q * C * DA, fragD ^ frag_tile<DA / 8>(it, 4 * s));
#pragma unroll
                        for (int p = 0; p < PP; ++p)
#pragma unroll
                            for (int it = 0; it < IT; ++it) {
#pragma unroll
                                for (int m = 0; m < NT; ++m) {
                                    f32x4& to = LESSER && p + q > 0 ? lesser[LESSER ? it : 0][m] : O[it][m];
                                    if (p + q <= ORD) to = mfma(as_frag(sw[m][p]), fq[it], to);
                                }
                                f32x4& to = LESSER && p + q > 0 ? few[0] : acc[C == 64 ? it : 0];
                                if (p < P && p + q <= ORD && (C == 64 || it == it0)) to = mfma(fb[p < P ? p : 0], fq[it], to);
                            }
                    }
                }
#pragma unroll
                for (int it = 0; it < IT; ++it) {
                    const float e = into[buf][16 * it + l16];
#pragma unroll
                    for (int m = 0; m < NT; ++m) {
                        if constexpr (LESSER) O[it][m] += lesser[it][m];
                        O[it][m] *= e;
                    }
                }
                if constexpr (LESSER) acc[0] += few[0];
                if constexpr (GRADS && DIRECT)
                    if (beside) load_x(px, n, otid);
                uint32_t pw[PT][PP][2];
                const int j = 16 * jt + 4 * g4;
                const f32x4 jhi = *reinterpret_cast<const f32x4*>(&sums_hi[buf][j]), jlo = *reinterpret_cast<const f32x4*>(&sums_lo[buf][j]);
                auto pairs = [&](int it, const f32x4& a, uint32_t (&w)[PP][2]) {
                    const int i = 16 * it + l16;
                    const float hi = sums_hi[buf][i], lo = sums_lo[buf][i];
                    float f[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        // (opaque: a select, not a branch around each exponential)
                        const float m = opaque_f32(a[e] * (__builtin_amdgcn_exp2f((hi - jhi[e]) + (lo - jlo[e])) * p_scale));
                        f[e] = j + e <= i ? m : 0.0f;
                    }
                    to_planes<PP, 2>(f, w);
                };
                // rows before 48 have no pairs with the last 16 columns: their wavefront forms the decays instead
                if (C == 64 && wave != 3)
#pragma unroll
                    for (int k = 0; k < PT - 1; ++k) pairs(k, acc[k], pw[k]);
                if (wave == 3 && n_next > 0) decays(g_next, buf ^ 1);
                pairs(C == 64 ? 3 : it0, acc[PT - 1], pw[PT - 1]);
                __syncthreads();
                // ---- the pairs to everybody
#pragma unroll
                for (int k = 0; k < PT; ++k) {
                    if (C == 64 && k < 3 && wave == 3) continue;  // (read by nobody, but for the next to the last 16 rows)
                    const int it = it0 + k;
#pragma unroll
                    for (int p = 0; p < PP; ++p)
                        *reinterpret_cast<u32x2*>(reinterpret_cast<char*>(ldsP + p * C * C) + (halfC ^ frag_tile<C / 8>(it, 2 * jt))) =
                            u32x2{pw[k][p][0], pw[k][p][1]};
                }
                if (C == 64 && wave == 3)
#pragma unroll
                    for (int p = 0; p < PP; ++p)
                        *reinterpret_cast<u32x2*>(reinterpret_cast<char*>(ldsP + p * C * C) + (halfC ^ frag_tile<C / 8>(2, 6))) = u32x2{0u, 0u};
                __syncthreads();
                if constexpr (GRADS) if (dots) {
                    // ---- what the state gives, dotted
                    float dot[IT];
#pragma unroll
                    for (int it = 0; it < IT; ++it) {
                        dot[it] = 0.0f;
#pragma unroll
                        for (int m = 0; m < NT; ++m)
#pragma unroll
                            for (int e = 0; e < 4; ++e) dot[it] = __builtin_fmaf(O[it][m][e], x_at(it * XR + (4 * m + e) / XE, (4 * m + e) % XE), dot[it]);
                    }
#pragma unroll
                    for (int it = 0; it < IT; ++it) {
                        float unused;
                        dot[it] = sum_rows(dot[it], g4, unused);
                    }
                    if (g4 == 0)
#pragma unroll
                        for (int it = 0; it < IT; ++it) dot_lds[wave][16 * it + l16] = dot[it];
                }
                if constexpr (GRADS) if (over) {
                    // ---- The chunk's pairs over a position: of its rows on one side and its columns on the other, the pair
                    // times the product of the row of x and the column's values. A wavefront takes 16 rows (in chunks of 32
                    // half of each product: shares add up in the end). Sums along a row run up to each position, rows add
                    // up: forwards of the columns before it and the rows from it on, backwards of the columns up to it
                    // (which are the positions from it on) and the rows after it.
                    const uint32_t fragX = frag_base<DC / 8>(l16, g4, 0);
                    uint32_t xw[NS][P][4];
#pragma unroll
                    for (int s = 0; s < NS; ++s) {
                        if constexpr (std::is_same_v<T, bf16>) {
#pragma unroll
                            for (int i = 0; i < 4; ++i) xw[s][0][i] = XE == 8 ? xr[XE == 8 ? s : 0][i % (XE / 2)] : xr[XE == 8 ? 0 : 2 * s + (i >> 1)][i & 1];
                        } else {
                            float f[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) f[i] = x_at((8 * s + i) / XE, (8 * s + i) % XE);
                            to_planes<P, 4>(f, xw[s]);
                        }
                    }
                    // (every tile without a branch, so that they wait side by side; what is not the position's is dropped in
                    // the end, by a select, as it need not be finite)
                    f32x4 w[IT], less[LESSER ? IT : 1];
#pragma unroll
                    for (int jt = 0; jt < IT; ++jt) {
                        w[jt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                        less[LESSER ? jt : 0] = w[jt];
                    }
#pragma unroll
                    for (int s = 0; s < NS; ++s)
#pragma unroll
                        for (int p = 0; p < P; ++p) {
                            bf16x8 fk[IT];
#pragma unroll
                            for (int jt = 0; jt < IT; ++jt) fk[jt] = lds_at<bf16x8>(ldsC + p * C * DC, fragX ^ frag_tile<DC / 8>(jt, 4 * (xs + s)));
#pragma unroll
                            for (int q = 0; q < P; ++q)
#pragma unroll
                                for (int jt = 0; jt < IT; ++jt) {
                                    f32x4& to = LESSER && p + q > 0 ? less[LESSER ? jt : 0] : w[jt];
                                    if (p + q <= ORD) to = mfma(fk[jt], as_frag(xw[s][q]), to);
                                }
                        }
                    u32x2 pair[IT][PP];
#pragma unroll
                    for (int jt = 0; jt < IT; ++jt)
#pragma unroll
                        for (int q = 0; q < PP; ++q)
                            pair[jt][q] = *reinterpret_cast<const u32x2*>(reinterpret_cast<const char*>(ldsP + q * C * C) + (halfC ^ frag_tile<C / 8>(xt, 2 * jt)));
                    f32x4 sums[IT];
                    float tiles = 0.0f;  // of the tiles before
                    const bool in = full || 16 * xt + l16 < n;
#pragma unroll
                    for (int jt = 0; jt < IT; ++jt) {
                        if constexpr (LESSER) w[jt] += less[jt];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float f = 0.0f;
#pragma unroll
                            for (int q = PP - 1; q >= 0; --q) f += __uint_as_float(e & 1 ? pair[jt][q][e >> 1] & 0xffff0000u : pair[jt][q][e >> 1] << 16);
                            w[jt][e] *= f;
                        }
                        const float w01 = w[jt][0] + w[jt][1], w012 = w01 + w[jt][2], all = w012 + w[jt][3];
                        float lanes;
                        const float tile = sum_rows(all, g4, lanes), base = tiles + lanes;
                        tiles += tile;
                        const float upto[5] = {base, base + w[jt][0], base + w01, base + w012, base + all};
                        const int most = !in || jt > xt ? -1 : jt < xt ? C : l16 - 4 * g4 - (reverse ? 1 : 0);
#pragma unroll
                        for (int e = 0; e < 4; ++e) sums[jt][e] = sum16(e <= most ? (reverse ? upto[e + 1] : upto[e]) : 0.0f);
                    }
                    if (l16 == 0)
#pragma unroll
                        for (int jt = 0; jt < IT; ++jt) *reinterpret_cast<f32x4*>(&over_lds[wave][16 * jt + 4 * g4]) = sums[jt];
                }
            }
            // the next chunk's x, with the time until that chunk to arrive (waited for with its operands: a wait on its own
            // would be for all that is on its way)
            if constexpr (GRADS && !DIRECT)
                if (beside && n_next > 0) load_x(px + n * sx, n_next, otid);
            if constexpr (DIRECT)
                if (n_next > 0) fetch(n_next, otid);
            const float decay = whole[buf];
            bool wild = false;
#pragma unroll
            for (int t = 0; t < TA; ++t)
#pragma unroll
                for (int m = 0; m < NT; ++m) S[t][m] *= decay;
#pragma unroll
            for (int s = 0; s < SC; ++s) {
                u32x4 fc[NT][P];
                uint32_t ww[NT][SP][4];
                float w8[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) w8[e] = left[buf][32 * s + 8 * g4 + e];
#pragma unroll
                for (int m = 0; m < NT; ++m) {
                    float f[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int p = P - 1; p >= 0; --p) {
                        fc[m][p] = turn_at<DC / 8>(ldsC + p * C * DC, turnC, wave * NT + m, s);
#pragma unroll
                        for (int e = 0; e < 8; ++e) f[e] = p == P - 1 ? vget<bf16>(fc[m][p], e) : f[e] + vget<bf16>(fc[m][p], e);
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) f[e] *= w8[e];
                    to_planes<SP, 4>(f, ww[m]);
                }
                if constexpr (!STATES) {
                    // An infinite or NaN value must not meet the zeros of the pairs that come before it: it is left out
                    // here, and put on its own and the later rows below.
                    uint16x2 top = {0, 0};
#pragma unroll
                    for (int m = 0; m < NT; ++m)
#pragma unroll
                        for (int i = 0; i < 4; ++i) top = __builtin_elementwise_max(top, __builtin_bit_cast(uint16x2, fc[m][0][i] & 0x7f807f80u));
                    if (__any(top[0] == 0x7f80 || top[1] == 0x7f80)) {
                        wild = true;
#pragma unroll
                        for (int m = 0; m < NT; ++m)
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                const uint32_t x = fc[m][0][i];
                                const uint32_t keep = ((x & 0x7f80u) == 0x7f80u ? 0u : 0xffffu) | ((x & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u);
#pragma unroll
                                for (int p = 0; p < P; ++p) fc[m][p][i] &= keep;
                            }
                    }
                }
                if constexpr (!STATES) {
#pragma unroll
                    for (int q = 0; q < PP; ++q) {
                        bf16x8 fp[IT];
#pragma unroll
                        for (int it = 2 * s; it < IT; ++it) fp[it] = lds_at<bf16x8>(ldsP + q * C * C, fragC ^ frag_tile<C / 8>(it, 4 * s));
#pragma unroll
                        for (int p = 0; p < P; ++p)
#pragma unroll
                            for (int it = 2 * s; it < IT; ++it)
#pragma unroll
                                for (int m = 0; m < NT; ++m)
                                    if (p + q <= ORD) O[it][m] = mfma(__builtin_bit_cast(bf16x8, fc[m][p]), fp[it], O[it][m]);
                    }
                }
                constexpr int TG = LESSER ? 2 : TA < 4 ? TA : 4;  // tiles at once
#pragma unroll
                for (int t0 = 0; t0 < TA; t0 += TG) {
                    f32x4 lesser[LESSER ? TG : 1][NT];
                    if constexpr (LESSER)
#pragma unroll
                        for (int t = 0; t < TG; ++t)
#pragma unroll
                            for (int m = 0; m < NT; ++m) lesser[t][m] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        bf16x8 fb[TG];
#pragma unroll
                        for (int t = 0; t < TG; ++t) fb[t] = __builtin_bit_cast(bf16x8, turn_at<DA / 8>(ldsB + p * C * DA, turnB, t0 + t, s));
#pragma unroll
                        for (int q = 0; q < SP; ++q)
#pragma unroll
                            for (int t = 0; t < TG; ++t)
#pragma unroll
                                for (int m = 0; m < NT; ++m) {
                                    f32x4& to = LESSER && p + q > 0 ? lesser[LESSER ? t : 0][m] : S[t0 + t][m];
                                    if (p + q <= SORD) to = mfma(fb[t], as_frag(ww[m][q]), to);
                                }
                    }
                    if constexpr (LESSER)
#pragma unroll
                        for (int t = 0; t < TG; ++t)
#pragma unroll
                            for (int m = 0; m < NT; ++m) S[t0 + t][m] += lesser[t][m];
                    if constexpr (LESSER) __builtin_amdgcn_sched_barrier(0);  // (one group's sums at a time)
                }
            }
            if constexpr (!STATES) {
                if (wild)
                    for (int j = 0; j < n; ++j) {
#pragma unroll
                        for (int m = 0; m < NT; ++m)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int c = tile_col(wave * NT + m, 4 * g4 + e);
                                const uint32_t b = ldsC[j * DC + swizzle<DC / 8>(j, c >> 3) * 8 + (c & 7)];
                                const float nan = __uint_as_float(b << 16) * 0.0f;  // or 0
#pragma unroll
                                for (int it = 0; it < IT; ++it)
                                    if (16 * it + l16 >= j) O[it][m][e] += nan;
                            }
                    }
                // from the lowest address of the chunk, so that offsets count up in 32 bits
                char* const low = out + (reverse ? -(C - 1) * opitch : 0);
                const uint32_t pitch = (uint32_t)opitch;
                const uint32_t row = (uint32_t)(reverse ? 15 - l16 : l16);
                const uint32_t at = row * pitch + (uint32_t)(col * osize);
#pragma unroll
                for (int it = 0; it < IT; ++it) {
                    char* const o = low + (uint64_t)(uint32_t)((reverse ? C - 16 - 16 * it : 16 * it) * pitch) + at;
                    if (full) {
                        store_outputs<T, NT>(o, O[it], job.out_f32);
                    } else if (16 * it + l16 < n) {
#pragma unroll
                        for (int m = 0; m < NT; ++m) {
                            if (col + 4 * m + 4 <= dc) {
                                store_outputs<T, 1>(o + 4 * m * osize, {O[it][m]}, job.out_f32);
                                continue;
                            }
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (col + 4 * m + e < dc) {
                                    if (job.out_f32) reinterpret_cast<float*>(o)[4 * m + e] = O[it][m][e];
                                    else reinterpret_cast<T*>(o)[4 * m + e] = from_f32<T>(O[it][m][e]);
                                }
                        }
                    }
                }
                out += n * dir * opitch;
                if (beside) px += n * sx;
            }
        }
        if (n_next <= 0) break;
        if constexpr (GRADS)
            if (r + n == stop) {
                // (a lane has four neighbouring rows of a column)
                auto put = [&](float* states, int64_t place) {
                    const int ol = opaque(lane), rows = (int)kept_rows(da), row0 = 8 * (ol >> 4);
                    float* const at = states + (place * args.heads + h) * dc * rows + row0;
#pragma unroll
                    for (int m = 0; m < NT; ++m) {
                        const int col = tile_col(wave * NT + m, ol & 15);
#pragma unroll
                        for (int t = 0; t < TA; ++t)
                            if (row0 + 32 * (t >> 1) + 4 * (t & 1) < da && col < dc)
                                *reinterpret_cast<AnyAddr<4>::v4*>(at + col * rows + 32 * (t >> 1) + 4 * (t & 1)) = __builtin_bit_cast(u32x4, S[t][m]);
                    }
                };
                const AttnJob& again = job_again();
                const int64_t at = reverse ? sp.len - stop : (int64_t)stop, p = again.mark != nullptr ? at / again.piece : 0;
                if (p > 0 && p * again.piece == at) put(again.mark, (args.cu ? sp.first / again.piece : sp.seq * (again.pieces - 1)) + p - 1);
                if (again.tail != nullptr && stop == ((int)sp.len - 1) / C * C) put(again.tail, sp.seq);
                stop = stop_after(stop);
            }
        if (wave == 3 && (STATES || n == 0)) decays(g_next, buf ^ 1);
        __syncthreads();
        if constexpr (GRADS)
            if (beside && tid < n) dots_out(r);
        buf ^= 1;
        r += n;
        n = n_next;
    }
    if constexpr (GRADS) {
        __syncthreads();
        if (beside && tid < n) dots_out(r);
    }

    // ---- the state at the segment's end
    const bool ends = sp.index + 1 == sp.segs;
    const AttnState last = STATES ? job.seg : job.last;
    if (last.p != nullptr && (STATES || ends)) {
        float by = 1.0f;
        // backwards, the state before the sequence has its first decay too
        if (!STATES && reverse && sp.len > 0) by = (float)exp(log_decay(to_f32(pg[sp.first * args.g_stride[1]])));
        float* const at = last.p + (STATES ? sp.after(reverse) : sp.seq) * last.s[0] + h * last.s[1];
        const int s2 = (int)last.s[2], s3 = (int)last.s[3];
#pragma unroll
        for (int t = 0; t < TA; ++t)
#pragma unroll
            for (int m = 0; m < NT; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int row = tile_col(t, 4 * (lane >> 4) + e), col = tile_col(wave * NT + m, lane & 15);
                    if (row < da && col < dc) at[(uint32_t)(row * s2 + col * s3)] = by * S[t][m][e];
                }
    }

    if (STATES && tid == 3 * 64) job.decay[sp.after(reverse) * args.heads + h] = (float)exp2(total);
    // positions that no sequence covers
    if (!STATES && args.cu != nullptr) {
        auto zero = [&](int64_t from, int64_t to) {
            for (int64_t i = tid; i < (to - from) * dc; i += 256) {
                const int64_t at = ((from + i / dc) * args.heads + h) * dc + i % dc;
                if (job.out_f32) static_cast<float*>(job.out)[at] = 0.0f;
                else static_cast<T*>(job.out)[at] = from_f32<T>(0.0f);
            }
        };
        if (sp.seq == 0 && sp.index == 0) zero(0, sp.first);
        if (sp.seq == args.num_seqs - 1 && ends) zero(sp.first + sp.len, args.seqlen);
    }
}

// Whether every operand of every job is made of whole 16-byte vectors, and a chunk of it spans less than 2 GiB.
template <typename T> bool attn_quick(const AttnArgs& a) {
    constexpr int64_t EPV = elems16<T>::value;
    auto fits = [&](const AttnOperand& o, int d) {
        const int64_t r = o.s[1] < 0 ? -o.s[1] : o.s[1];
        return o.p == nullptr || (o.s[3] == 1 && d % EPV == 0 && r < ((int64_t)1 << 31) / (64 * (int64_t)sizeof(T)));
    };
    bool quick = true;
    for (uint32_t j = 0; j < a.jobs; ++j) {
        const AttnJob& b = a.job[j];
        quick = quick && fits(b.a, b.da) && fits(b.b, b.da) && fits(b.c, b.dc) && fits(b.x, b.dc);
    }
    return quick;
}

template <typename T, int MODE, bool QUICK, bool GRADS> int launch_attn_sizes(const AttnArgs& a, int da, int dc, hipStream_t stream) {
    const dim3 grid(a.blocks), block(256);
    if (da <= 64 && dc <= 64) return launch(attn_kernel<T, 64, 64, MODE, QUICK, GRADS>, grid, block, stream, a);
    if (da <= 64) return launch(attn_kernel<T, 64, 128, MODE, QUICK, GRADS>, grid, block, stream, a);
    if (dc <= 64) return launch(attn_kernel<T, 128, 64, MODE, QUICK, GRADS>, grid, block, stream, a);
    return launch(attn_kernel<T, 128, 128, MODE, QUICK, GRADS>, grid, block, stream, a);
}

// All jobs of `a` have rows of da and values of dc (explicitly instantiated in cc1d_attn_<dtype>[_any].hip).
template <typename T, bool QUICK> int launch_attn_modes(const AttnArgs& a, int da, int dc, bool states, hipStream_t stream);
template <typename T, bool QUICK> int launch_attn_modes_impl(const AttnArgs& a, int da, int dc, bool states, hipStream_t stream) {
    if (states) return launch_attn_sizes<T, kAttnStates, QUICK, false>(a, da, dc, stream);
    bool exact = AttnType<T>::order == 2, grads = false;
    for (uint32_t j = 0; j < a.jobs; ++j) {
        exact = exact || a.job[j].last.p != nullptr;
        grads = grads || a.job[j].x.p != nullptr;
    }
    return with_flag(grads, [&](auto gr) {
        constexpr bool GRADS = decltype(gr)::value;
        if constexpr (AttnType<T>::order < 2)
            if (!exact) return launch_attn_sizes<T, kAttnOut, QUICK, GRADS>(a, da, dc, stream);
        return launch_attn_sizes<T, kAttnExact, QUICK, GRADS>(a, da, dc, stream);
    });
}

}  // namespace cc1d
