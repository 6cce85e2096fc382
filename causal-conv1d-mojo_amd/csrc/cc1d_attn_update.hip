// cc1d_attn_update.hip -- decode step of linear attention with a decay for
// each head.
//
// Per (batch entry, head) the state's dk x dv values are read, moved by one
// step per new token (S = exp(g) S + k v^T), multiplied with q, and written
// back: 8 bytes of state a value, everything else is shared by its rows or
// columns, so HBM bounds it.
#include "cc1d_scan_device.hpp"

namespace cc1d {
namespace {

// exp(g), by a product with log2(e) in two floats: rounded to one, an exponent of -16 would cost 8 * 2^-24 of the decay.
// (-1e5 stands for everything below, as 1e5 for everything above: their second float would not be a number.)
__device__ __forceinline__ float decay_of(float g) {
    const float x = g < -1e5f ? -1e5f : g > 1e5f ? 1e5f : g, hi = x * 1.44269502f;
    const float lo = __builtin_fmaf(x, 1.44269502f, -hi) + x * 1.92596299e-8f;
    return __builtin_amdgcn_exp2f(hi) * __builtin_fmaf(lo, 0.69314718f, 1.0f);
}

struct AttnUpdateArgs {
    cc1d_attn_update_params p;
    FastDiv heads, group, quads;  // of quads: a row's groups of four columns
    int32_t row_groups;           // rows that a block's threads take at once
};

// A block holds one state in registers, four columns of R rows a thread (all
// loads in flight at once), and takes the tokens one after the other: the sum
// over its own rows, then over the threads that share columns through LDS.
template <typename T, int R, bool VEC> __global__ void __launch_bounds__(256) attn_update_kernel(const AttnUpdateArgs arg) {
    const cc1d_attn_update_params& p = arg.p;
    __shared__ float ql[2][CC1D_MAX_ATTN_DIM], kl[2][CC1D_MAX_ATTN_DIM];
    __shared__ __attribute__((aligned(16))) float vl[2][CC1D_MAX_ATTN_DIM + 4], part[256 * 4];
    __shared__ float decay[2];
    const int tid = threadIdx.x, dk = (int)p.dk, dv = (int)p.dv, tokens = (int)p.tokens;
    const uint32_t b = arg.heads.div(blockIdx.x), h = blockIdx.x - b * (uint32_t)p.heads;
    T* const out = static_cast<T*>(p.out) + ((int64_t)b * tokens * p.heads + h) * dv;
    const int64_t step = p.heads * dv;
    const int64_t row = p.attn_state_indices ? ld_uniform(p.attn_state_indices + b) : b;
    if (row < 0 || row >= p.state_rows) {
        for (int i = tid; i < tokens * dv; i += 256) out[i / dv * step + i % dv] = T{};
        return;
    }
    const int rg = (int)arg.quads.div((uint32_t)tid), quad = tid - rg * (int)arg.quads.d, col = 4 * quad;
    const bool mine = rg < arg.row_groups;
    const uint32_t kh = arg.group.div(h);
    const T* const q = static_cast<const T*>(p.q) + b * p.q_stride[0] + kh * p.q_stride[2];
    const T* const k = static_cast<const T*>(p.k) + b * p.k_stride[0] + kh * p.k_stride[2];
    const T* const v = static_cast<const T*>(p.v) + b * p.v_stride[0] + h * p.v_stride[2];
    const T* const g = static_cast<const T*>(p.g) + b * p.g_stride[0] + h * p.g_stride[2];
    const float scale = (float)p.scale;
    // One wavefront each for q, k and v, and the decay: two values a lane, asked for before and put into LDS after
    // whatever else the block asks for.
    const int lane = tid & 63, w = tid >> 6, size = w < 2 ? dk : dv;
    const T* const mine_at = w == 0 ? q : w == 1 ? k : w == 2 ? v : g;
    const int64_t by_token = w == 0 ? p.q_stride[1] : w == 1 ? p.k_stride[1] : w == 2 ? p.v_stride[1] : p.g_stride[1];
    const int64_t by_element = w == 0 ? p.q_stride[3] : w == 1 ? p.k_stride[3] : w == 2 ? p.v_stride[3] : 0;
    T next[2];
    auto ask = [&](int t) {
#pragma unroll
        for (int i = 0; i < 2; ++i) next[i] = mine_at[t * by_token + (lane + 64 * i < size ? lane + 64 * i : 0) * by_element];
    };
    auto put = [&](int buf) {
        float f[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) f[i] = lane + 64 * i < size ? to_f32(next[i]) : 0.0f;
        if (w == 3) {
            if (lane == 0) decay[buf] = decay_of(f[0]);
            return;
        }
        float* const to = w == 0 ? ql[buf] : w == 1 ? kl[buf] : vl[buf];
#pragma unroll
        for (int i = 0; i < 2; ++i) to[lane + 64 * i] = w == 0 ? f[i] * scale : f[i];
    };
    ask(0);
    float* const state = p.attn_state + row * p.attn_state_stride[0] + (int64_t)h * p.attn_state_stride[1] + col * p.attn_state_stride[3];
    float S[R][4];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int r = rg + i * arg.row_groups;
        const float* at = state + r * p.attn_state_stride[2];
        const bool here = mine && r < dk;
        if constexpr (VEC) {
            u32x4 w = vzero();
            if (here) w = vload_any_nt(at);
#pragma unroll
            for (int e = 0; e < 4; ++e) S[i][e] = __uint_as_float(w[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) S[i][e] = here && col + e < dv ? at[e * p.attn_state_stride[3]] : 0.0f;
        }
    }
    put(0);
    __syncthreads();
    auto store = [&]() {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int r = rg + i * arg.row_groups;
            float* at = state + r * p.attn_state_stride[2];
            if (!mine || r >= dk) continue;
            if constexpr (VEC) {
                vstore_any_nt(at, u32x4{__float_as_uint(S[i][0]), __float_as_uint(S[i][1]), __float_as_uint(S[i][2]), __float_as_uint(S[i][3])});
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (col + e < dv) at[e * p.attn_state_stride[3]] = S[i][e];
            }
        }
    };
    for (int t = 0; t < tokens; ++t) {
        const int buf = t & 1;
        if (t + 1 < tokens) ask(t + 1);
        const float e = decay[buf];
        float vq[4], acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < 4; ++c) vq[c] = vl[buf][(col < CC1D_MAX_ATTN_DIM ? col : 0) + c];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int r = rg + i * arg.row_groups;
            const bool here = mine && r < dk;
            const float kr = here ? kl[buf][r] : 0.0f, qr = here ? ql[buf][r] : 0.0f;
            if (!here) continue;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                S[i][c] = __builtin_fmaf(e, S[i][c], kr * vq[c]);
                acc[c] = __builtin_fmaf(qr, S[i][c], acc[c]);
            }
        }
        if (mine) *reinterpret_cast<u32x4*>(part + 4 * tid) = u32x4{__float_as_uint(acc[0]), __float_as_uint(acc[1]), __float_as_uint(acc[2]), __float_as_uint(acc[3])};
        if (t + 1 < tokens) put(buf ^ 1);
        else store();
        __syncthreads();
        const int width = 4 * (int)arg.quads.d;  // part is (row_groups, width)
        if (tid < dv) {
            float y = 0.0f;
            for (int r = 0; r < arg.row_groups; ++r) y += part[r * width + tid];
            out[t * step + tid] = from_f32<T>(y);
        }
        if (t + 1 < tokens) __syncthreads();
    }
}

}  // namespace

int launch_attn_update(const cc1d_attn_update_params& p, hipStream_t stream) {
    AttnUpdateArgs a{p, FastDiv((uint32_t)p.heads), FastDiv((uint32_t)(p.heads / p.key_heads)), FastDiv((uint32_t)ceil_div(p.dv, 4)), 0};
    a.row_groups = (int)(256 / a.quads.d);
    const int rows = (int)ceil_div(p.dk, a.row_groups);
    const dim3 grid((unsigned)(p.batch * p.heads));
    const bool vec = p.dv % 4 == 0 && p.attn_state_stride[3] == 1;
    return with_dtype(p.dtype, [&](auto t) {
        typedef decltype(t) T;
        return with_flag(vec, [&](auto vv) {
            constexpr bool VEC = decltype(vv)::value;
            if (rows <= 4) return launch(attn_update_kernel<T, 4, VEC>, grid, dim3(256), stream, a);
            if (rows <= 8) return launch(attn_update_kernel<T, 8, VEC>, grid, dim3(256), stream, a);
            return launch(attn_update_kernel<T, 16, VEC>, grid, dim3(256), stream, a);
        });
    });
}

}  // namespace cc1d
