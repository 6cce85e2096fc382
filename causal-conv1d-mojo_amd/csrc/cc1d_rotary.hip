// cc1d_rotary.hip -- norm of each query and key head with the rotation by
// position, forward and backward.
//
// Every element is read and written once; the angles belong to a token and are
// shared by all its heads, so a wavefront takes one token, forms the sines
// and cosines of the pairs that its lanes hold once, and walks over heads:
// HBM bounds it. A lane holds eight values of a head: four pairs, or eight
// values behind the rotated ones.
//
// Angles: position * inv_freq is formed and reduced to a quarter turn in 64
// bits (at a position of a million 32 bits would be off by a few hundredths of
// a turn's sixth), the sine and cosine of what is left are fp32.
#include "cc1d_internal.hpp"
#include "cc1d_scan_device.hpp"

namespace cc1d {
namespace {

struct RotaryArgs {
    cc1d_rotary_params p;
    cc1d_rotary_bwd_params b;  // the backward's own fields (fwd is p)
    FastDiv seqlen;
    int32_t share;             // wavefronts to a token: 1, 2 or 4
    uint32_t tokens, blocks;
};

// Sum over groups of LPH lanes, in every lane.
template <int LPH> __device__ __forceinline__ float group_sum(float v) {
    v += dpp_f32<kDppQuadSwap1, 0xf>(v);
    v += dpp_f32<kDppQuadSwap2, 0xf>(v);
    if constexpr (LPH >= 16) {
        v += dpp_f32<kDppRowRor4, 0xf>(v);
        v += dpp_f32<kDppRowRor8, 0xf>(v);
    } else {
        v += __shfl_xor(v, 4);
    }
    if constexpr (LPH >= 32) v += __shfl_xor(v, 16);
    if constexpr (LPH >= 64) v += __shfl_xor(v, 32);
    return v;
}

// The eight values of a head that a lane holds: two runs of up to four.
struct Unit {
    int at[2], count[2];
    int pair;      // index of the first of its four pairs
    bool turned;   // whether it has pairs (interleaved: those below `rotated`)
};

template <bool INTER> __device__ __forceinline__ Unit unit_of(int u, int dim, int rotated) {
    Unit w;
    if constexpr (INTER) {
        w.at[0] = 8 * u;
        w.at[1] = 8 * u + 4;
        w.pair = 4 * u;
        w.turned = 8 * u < rotated;
    } else {
        const int half = rotated >> 1, pairs = (half + 3) >> 2;
        w.turned = u < pairs;
        w.pair = 4 * u;
        w.at[0] = w.turned ? 4 * u : rotated + 8 * (u - pairs);
        w.at[1] = w.turned ? half + 4 * u : w.at[0] + 4;
        if (w.turned) {
            const int c = half - 4 * u < 4 ? half - 4 * u : 4;
            w.count[0] = w.count[1] = c;
            return w;
        }
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) w.count[i] = dim - w.at[i] < 4 ? (dim - w.at[i] > 0 ? dim - w.at[i] : 0) : 4;
    return w;
}

// Four values, widened to fp32 where they are used.
template <typename T> struct Four {
    uint32_t w[4 * sizeof(T) / 4];
    __device__ __forceinline__ void load(const T* at, int64_t stride, int count) {
        if (count == 4 && stride == 1) {
            if constexpr (sizeof(T) == 4) {
                const u32x4 x = vload_any(at);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = x[i];
            } else {
                const u32x2 x = *reinterpret_cast<const typename AnyAddr<2>::v2*>(at);
                w[0] = x[0];
                w[1] = x[1];
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < (int)(sizeof(w) / 4); ++i) w[i] = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i >= count) continue;
            if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(to_f32(at[i * stride]));
            else w[i >> 1] |= (uint32_t)__builtin_bit_cast(uint16_t, at[i * stride]) << (16 * (i & 1));
        }
    }
    __device__ __forceinline__ void get(float* f) const {
        u32x4 x = vzero();
#pragma unroll
        for (int i = 0; i < (int)(sizeof(w) / 4); ++i) x[i] = w[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = vget<T>(x, i);
    }
};
template <typename T> __device__ __forceinline__ void store_four(T* at, const float* f, int count) {
    if (count == 4) {
        if constexpr (sizeof(T) == 4) vstore_any_nt(at, u32x4{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])});
        else __builtin_nontemporal_store(u32x2{pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3])}, reinterpret_cast<typename AnyAddr<2>::v2*>(at));
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (i < count) at[i] = from_f32<T>(f[i]);
}

// Cosines and sines of a lane's four pairs, times the amplitude.
struct Angles {
    float c[4], s[4];
};

__device__ __forceinline__ Angles angles_of(const cc1d_rotary_params& p, int64_t b, int64_t t, const Unit& u) {
    Angles a;
    int64_t pos = t;
    if (p.positions != nullptr) {
        const int64_t at = b * p.positions_stride[0] + t * p.positions_stride[1];
        pos = p.positions_bytes == 8 ? static_cast<const int64_t*>(p.positions)[at] : static_cast<const int32_t*>(p.positions)[at];
    }
    const float amp = (float)p.amplitude;
    const int half = (int)p.rotated >> 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a.c[i] = 1.0f;
        a.s[i] = 0.0f;
        if (!u.turned || u.pair + i >= half) continue;
        const double quarters = (double)pos * (double)p.inv_freq[u.pair + i] * 0.63661977236758134308;  // of a turn
        const double whole = __builtin_rint(quarters);
        const float r = (float)(quarters - whole);
        float s, c;
        sincospif(0.5f * r, &s, &c);
        const double turn = whole - 4.0 * __builtin_floor(whole * 0.25);  // 0 .. 3
        const int q = (int)turn;
        const float s0 = (q & 1) ? c : s, c0 = (q & 1) ? s : c;
        a.s[i] = ((q & 2) ? -s0 : s0) * amp;
        a.c[i] = (q == 1 || q == 2 ? -c0 : c0) * amp;
    }
    return a;
}

// BACK: by the opposite angle.
template <bool INTER, bool BACK> __device__ __forceinline__ void turn(float (&v)[8], const Angles& a, const Unit& u, int half) {
    if (!u.turned) return;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int x = INTER ? 2 * i : i, y = INTER ? 2 * i + 1 : 4 + i;
        if (u.pair + i >= half) continue;
        const float s = BACK ? -a.s[i] : a.s[i], p = v[x], q = v[y];
        v[x] = __builtin_fmaf(p, a.c[i], -(q * s));
        v[y] = __builtin_fmaf(q, a.c[i], p * s);
    }
}

template <typename T, int LPH, bool INTER> __global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs arg) {
    const cc1d_rotary_params& p = arg.p;
    constexpr int HEADS = 64 / LPH, K = 4;  // heads a wavefront takes at once; of those, in flight
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, dim = (int)p.dim, rotated = (int)p.rotated;
    const uint32_t token = blockIdx.x * (4 / arg.share) + wave / arg.share;
    if (token >= arg.tokens) return;
    const int part = wave % arg.share;
    const uint32_t b = arg.seqlen.div(token), t = token - b * (uint32_t)p.seqlen;
    const Unit u = unit_of<INTER>(lane % LPH, dim, rotated);
    const Angles a = angles_of(p, b, t, u);
    float wq[8], wk[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const bool in = (e & 3) < u.count[e >> 2];
        wq[e] = p.q_weight && in ? p.q_weight[u.at[e >> 2] + (e & 3)] : 1.0f;
        wk[e] = p.k_weight && in ? p.k_weight[u.at[e >> 2] + (e & 3)] : 1.0f;
    }
    const float inv = 1.0f / (float)dim, eps = (float)p.eps;
    auto heads = [&](const void* src, const int64_t (&stride)[4], void* dst, int64_t count, bool norm, const float (&w)[8]) {
        const T* const base = static_cast<const T*>(src) + b * stride[0] + t * stride[1];
        T* const out = static_cast<T*>(dst) + (int64_t)token * count * dim;
        for (int64_t h0 = part * HEADS + lane / LPH; h0 < count; h0 += K * arg.share * HEADS) {
            Four<T> raw[K][2];
#pragma unroll
            for (int j = 0; j < K; ++j) {
                const int64_t h = h0 + j * arg.share * HEADS;
                if (h >= count) continue;
#pragma unroll
                for (int i = 0; i < 2; ++i) raw[j][i].load(base + h * stride[2] + u.at[i] * stride[3], stride[3], u.count[i]);
            }
#pragma unroll
            for (int j = 0; j < K; ++j) {
                const int64_t h = h0 + j * arg.share * HEADS;
                if (h >= count) continue;  // (the lanes of a head together)
                float v[8];
                raw[j][0].get(v);
                raw[j][1].get(v + 4);
                if (norm) {
                    float sum = 0.0f;
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum = __builtin_fmaf(v[e], v[e], sum);
                    const float rstd = 1.0f / sqrtf(__builtin_fmaf(group_sum<LPH>(sum), inv, eps));
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = v[e] * rstd * w[e];
                }
                turn<INTER, false>(v, a, u, rotated >> 1);
#pragma unroll
                for (int i = 0; i < 2; ++i) store_four(out + h * dim + u.at[i], v + 4 * i, u.count[i]);
            }
        }
    };
    heads(p.q, p.q_stride, p.q_out, p.q_heads, p.q_weight != nullptr, wq);
    heads(p.k, p.k_stride, p.k_out, p.k_heads, p.k_weight != nullptr, wk);
}

// Backward: with d = the gradient turned back, dweight += d x^, and dx = rstd
// (d w - x^ mean(d w x^)), x^ = x rstd. A block walks over tokens and keeps
// its lanes' shares of the weights' gradients; they are added over the block's
// heads and wavefronts at its end, and over the blocks by a second kernel.
template <typename T, int LPH, bool INTER> __global__ void __launch_bounds__(256) rotary_bwd_kernel(const RotaryArgs arg) {
    const cc1d_rotary_params& p = arg.p;
    const cc1d_rotary_bwd_params& g = arg.b;
    constexpr int HEADS = 64 / LPH, K = 2;
    __shared__ float share_lds[2][4][LPH * 8];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, dim = (int)p.dim, rotated = (int)p.rotated;
    const int part = wave % arg.share;
    const Unit u = unit_of<INTER>(lane % LPH, dim, rotated);
    float wq[8], wk[8], dwq[8], dwk[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const bool in = (e & 3) < u.count[e >> 2];
        wq[e] = p.q_weight && in ? p.q_weight[u.at[e >> 2] + (e & 3)] : 1.0f;
        wk[e] = p.k_weight && in ? p.k_weight[u.at[e >> 2] + (e & 3)] : 1.0f;
        dwq[e] = dwk[e] = 0.0f;
    }
    const float inv = 1.0f / (float)dim, eps = (float)p.eps;
    const uint32_t per = 4 / arg.share;
    for (uint32_t token = blockIdx.x * per + wave / arg.share; token < arg.tokens; token += arg.blocks * per) {
        const uint32_t b = arg.seqlen.div(token), t = token - b * (uint32_t)p.seqlen;
        const Angles a = angles_of(p, b, t, u);
        auto heads = [&](const void* src, const int64_t (&stride)[4], const void* grad, const int64_t (&gstride)[4], void* dst, int64_t count,
                         bool norm, const float (&w)[8], float (&dw)[8]) {
            const T* const base = static_cast<const T*>(src) + b * stride[0] + t * stride[1];
            const T* const gbase = static_cast<const T*>(grad) + b * gstride[0] + t * gstride[1];
            T* const out = static_cast<T*>(dst) + (int64_t)token * count * dim;
            for (int64_t h0 = part * HEADS + lane / LPH; h0 < count; h0 += K * arg.share * HEADS) {
                Four<T> raw[K][2], graw[K][2];
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    const int64_t h = h0 + j * arg.share * HEADS;
                    if (h >= count) continue;
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        graw[j][i].load(gbase + h * gstride[2] + u.at[i] * gstride[3], gstride[3], u.count[i]);
                        if (norm) raw[j][i].load(base + h * stride[2] + u.at[i] * stride[3], stride[3], u.count[i]);
                    }
                }
#pragma unroll
                for (int j = 0; j < K; ++j) {
                    const int64_t h = h0 + j * arg.share * HEADS;
                    if (h >= count) continue;
                    float d[8];
                    graw[j][0].get(d);
                    graw[j][1].get(d + 4);
                    turn<INTER, true>(d, a, u, rotated >> 1);
                    if (norm) {
                        float x[8], sum = 0.0f, along = 0.0f;
                        raw[j][0].get(x);
                        raw[j][1].get(x + 4);
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            sum = __builtin_fmaf(x[e], x[e], sum);
                            along = __builtin_fmaf(d[e] * w[e], x[e], along);
                        }
                        const float rstd = 1.0f / sqrtf(__builtin_fmaf(group_sum<LPH>(sum), inv, eps));
                        along = group_sum<LPH>(along) * inv * rstd;
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float xh = x[e] * rstd;
                            dw[e] = __builtin_fmaf(d[e], xh, dw[e]);
                            d[e] = rstd * __builtin_fmaf(-xh, along, d[e] * w[e]);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < 2; ++i) store_four(out + h * dim + u.at[i], d + 4 * i, u.count[i]);
                }
            }
        };
        heads(p.q, p.q_stride, g.dq_out, g.dq_out_stride, g.dq, p.q_heads, p.q_weight != nullptr, wq, dwq);
        heads(p.k, p.k_stride, g.dk_out, g.dk_out_stride, g.dk, p.k_heads, p.k_weight != nullptr, wk, dwk);
    }
    if (p.q_weight == nullptr && p.k_weight == nullptr) return;
    for (int e = 0; e < 8; ++e) {
#pragma unroll
        for (int m = LPH; m < 64; m *= 2) {
            dwq[e] += __shfl_xor(dwq[e], m);
            dwk[e] += __shfl_xor(dwk[e], m);
        }
        if (lane < LPH) {
            share_lds[0][wave][lane * 8 + e] = dwq[e];
            share_lds[1][wave][lane * 8 + e] = dwk[e];
        }
    }
    __syncthreads();
    // workspace: (2, blocks, dim)
    for (int i = threadIdx.x; i < 2 * LPH * 8; i += 256) {
        const int which = i / (LPH * 8), slot = i % (LPH * 8), e = slot & 7;
        const Unit w = unit_of<INTER>(slot >> 3, dim, rotated);
        if ((e & 3) >= w.count[e >> 2]) continue;
        const float* s = &share_lds[which][0][slot];
        g.workspace[((int64_t)which * arg.blocks + blockIdx.x) * dim + w.at[e >> 2] + (e & 3)] =
            (s[0] + s[LPH * 8]) + (s[2 * LPH * 8] + s[3 * LPH * 8]);
    }
}

// Sums of a column of the blocks' shares, in a fixed order: 16 columns a block.
__global__ void __launch_bounds__(256) rotary_weights_kernel(const RotaryArgs arg) {
    __shared__ float sums[16][17];
    const int c = threadIdx.x & 15, r = threadIdx.x >> 4, dim = (int)arg.p.dim;
    float* const out = blockIdx.y ? arg.b.dk_weight : arg.b.dq_weight;
    if ((blockIdx.y ? arg.p.k_weight : arg.p.q_weight) == nullptr) return;
    const int col = blockIdx.x * 16 + c;
    float s = 0.0f;
    if (col < dim) {
        const float* at = arg.b.workspace + (int64_t)blockIdx.y * arg.blocks * dim + col;
        for (uint32_t i = r; i < arg.blocks; i += 16) s += at[(int64_t)i * dim];
    }
    sums[r][c] = s;
    __syncthreads();
    if (r == 0 && col < dim) {
        for (int i = 1; i < 16; ++i) s += sums[i][c];
        out[col] = s;
    }
}

// Lanes that hold a head: a power of two.
int head_lanes(const cc1d_rotary_params& p) {
    const int units = (int)(p.interleaved ? ceil_div(p.dim, 8) : ceil_div(p.rotated / 2, 4) + ceil_div(p.dim - p.rotated, 8));
    int n = 8;
    while (n < units) n *= 2;
    return n;
}

template <typename F> int with_lanes(const cc1d_rotary_params& p, F&& f) {
    return with_flag(p.interleaved != 0, [&](auto inter) {
        switch (head_lanes(p)) {
        case 8: return f(std::integral_constant<int, 8>{}, inter);
        case 16: return f(std::integral_constant<int, 16>{}, inter);
        case 32: return f(std::integral_constant<int, 32>{}, inter);
        default: return f(std::integral_constant<int, 64>{}, inter);
        }
    });
}

int64_t bwd_blocks(const cc1d_rotary_params& p) {
    const int64_t tokens = p.batch * p.seqlen;
    return tokens < 1024 ? (tokens > 0 ? tokens : 1) : 1024;
}

RotaryArgs args_of(const cc1d_rotary_params& p, int64_t most) {
    RotaryArgs a{};
    a.p = p;
    a.tokens = (uint32_t)(p.batch * p.seqlen);
    a.seqlen = FastDiv((uint32_t)(p.seqlen > 0 ? p.seqlen : 1));
    // several wavefronts share a token where there are too few tokens to fill the chip
    a.share = p.batch * p.seqlen >= most ? 1 : 4;
    return a;
}

}  // namespace

int launch_rotary_fwd(const cc1d_rotary_params& p, hipStream_t stream) {
    const RotaryArgs a = args_of(p, 8192);
    const dim3 grid((unsigned)ceil_div(a.tokens, 4 / a.share));
    return with_dtype(p.dtype, [&](auto t) {
        return with_lanes(p, [&](auto l, auto inter) {
            return launch(rotary_kernel<decltype(t), decltype(l)::value, decltype(inter)::value>, grid, dim3(256), stream, a);
        });
    });
}

int64_t rotary_bwd_workspace_floats(const cc1d_rotary_bwd_params& b) {
    return b.fwd.q_weight || b.fwd.k_weight ? 2 * bwd_blocks(b.fwd) * b.fwd.dim : 0;
}

int launch_rotary_bwd(const cc1d_rotary_bwd_params& b, hipStream_t stream) {
    const cc1d_rotary_params& p = b.fwd;
    RotaryArgs a = args_of(p, 8192);
    a.b = b;
    a.blocks = (uint32_t)bwd_blocks(p);
    const int st = with_dtype(p.dtype, [&](auto t) {
        return with_lanes(p, [&](auto l, auto inter) {
            return launch(rotary_bwd_kernel<decltype(t), decltype(l)::value, decltype(inter)::value>, dim3(a.blocks), dim3(256), stream, a);
        });
    });
    if (st != CC1D_OK || (!p.q_weight && !p.k_weight)) return st;
    return launch(rotary_weights_kernel, dim3((unsigned)ceil_div(p.dim, 16), 2), dim3(256), stream, a);
}

}  // namespace cc1d
