// cc1d_rotary.hip -- norm of each query and key head with the rotation by
// position, forward and backward.
//
// Every element is read and written once; the angles belong to a token and are
// shared by all its heads, so a wavefront takes one token, forms the sines
// and cosines of the pairs that its lanes hold once, and walks over heads:
// HBM bounds it. A lane holds eight values of a head: four pairs, or eight
// values behind the rotated ones. The walk goes on from queries to keys and
// to the wavefront's next token, and loads one stop ahead of what it computes.
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
    int32_t share;             // wavefronts to a token: 1 or 4
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
    // four neighbours, without a branch: the loads of a stop are counted, so that only those of the stop before are waited for
    __device__ __forceinline__ void whole(const T* at) {
        if constexpr (sizeof(T) == 4) {
            const u32x4 x = vload_any(at);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = x[i];
        } else {
            const u32x2 x = *reinterpret_cast<const typename AnyAddr<2>::v2*>(at);
            w[0] = x[0];
            w[1] = x[1];
        }
    }
    __device__ __forceinline__ void get(float* f, bool some) const {
        u32x4 x = vzero();
#pragma unroll
        for (int i = 0; i < (int)(sizeof(w) / 4); ++i) x[i] = w[i];
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = some ? vget<T>(x, i) : 0.0f;
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

// A wavefront's walk: K heads a lane at each stop, from the queries (which 0) to the keys, from token to token.
template <int STEP> struct Stop {
    uint32_t token;
    int32_t which, h;
    __device__ __forceinline__ void settle(const RotaryArgs& a, int first, uint32_t tokens_a_turn) {
        while (token < a.tokens && h >= (which ? (int)a.p.k_heads : (int)a.p.q_heads)) {
            token += which ? tokens_a_turn : 0;
            which ^= 1;
            h = first;
        }
    }
    __device__ __forceinline__ Stop next(const RotaryArgs& a, int first, uint32_t tokens_a_turn) const {
        Stop s = {token, which, h + STEP * a.share};
        s.settle(a, first, tokens_a_turn);
        return s;
    }
};

// WHOLE: unit strides and runs of four (whole_runs()).
template <typename T, int LPH, bool INTER, bool WHOLE> __global__ void __launch_bounds__(256) rotary_kernel(const RotaryArgs arg) {
    const cc1d_rotary_params& p = arg.p;
    constexpr int HEADS = 64 / LPH, K = sizeof(T) == 2 ? 4 : 2;  // heads a wavefront takes at once; of those, at a stop
    typedef Stop<HEADS * K> Stop;
    const int wave = uniform32(threadIdx.x >> 6), lane = threadIdx.x & 63, dim = (int)p.dim, rotated = (int)p.rotated;
    const int first = wave % arg.share * HEADS;
    const uint32_t per = 4 / arg.share, turns = arg.blocks * per;
    const Unit u = unit_of<INTER>(lane % LPH, dim, rotated);
    Angles a;
    float wq[8], wk[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const bool in = (e & 3) < u.count[e >> 2];
        wq[e] = p.q_weight && in ? p.q_weight[u.at[e >> 2] + (e & 3)] : 1.0f;
        wk[e] = p.k_weight && in ? p.k_weight[u.at[e >> 2] + (e & 3)] : 1.0f;
    }
    const float inv = 1.0f / (float)dim, eps = (float)p.eps;
    struct Raw {
        Four<T> v[K][2];
    };
    auto load = [&](const Stop& s, Raw& r) {
        const uint32_t b = arg.seqlen.div(s.token), t = s.token - b * (uint32_t)p.seqlen;
        const int64_t (&stride)[4] = s.which ? p.k_stride : p.q_stride;
        const T* const base = static_cast<const T*>(s.which ? p.k : p.q) + b * stride[0] + t * stride[1];
        const int count = s.which ? (int)p.k_heads : (int)p.q_heads;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int h = s.h + j * arg.share * HEADS + lane / LPH;
            if constexpr (WHOLE) {
                const T* const at = base + (h < count ? h : count - 1) * stride[2];
#pragma unroll
                for (int i = 0; i < 2; ++i) r.v[j][i].whole(at + (u.count[i] ? u.at[i] : 0));
                continue;
            }
            if (h >= count) continue;
#pragma unroll
            for (int i = 0; i < 2; ++i) r.v[j][i].load(base + h * stride[2] + u.at[i] * stride[3], stride[3], u.count[i]);
        }
    };
    auto work = [&](const Stop& s, const Raw& r, T* dst, int count, bool norm, const float (&w)[8]) {
        T* const out = dst + (int64_t)s.token * count * dim;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int h = s.h + j * arg.share * HEADS + lane / LPH;
            if (h >= count) continue;  // (the lanes of a head together)
            float v[8];
            r.v[j][0].get(v, !WHOLE || u.count[0]);
            r.v[j][1].get(v + 4, !WHOLE || u.count[1]);
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
            for (int i = 0; i < 2; ++i) store_four(out + (int64_t)h * dim + u.at[i], v + 4 * i, u.count[i]);
        }
    };
    Stop here = {blockIdx.x * per + wave / arg.share, 0, first};
    here.settle(arg, first, turns);
    uint32_t angles_at = ~0u;
    // the work of a stop, with the loads of the one after it on their way
    auto at = [&](const Stop& s, const Raw& now, Raw& ahead) {
        const Stop after = s.next(arg, first, turns);
        if (WHOLE || after.token < arg.tokens) load(after.token < arg.tokens ? after : s, ahead);
        if (s.token != angles_at) {
            angles_at = s.token;
            const uint32_t b = arg.seqlen.div(s.token);
            a = angles_of(p, b, s.token - b * (uint32_t)p.seqlen, u);
        }
        if (s.which == 0) work(s, now, static_cast<T*>(p.q_out), (int)p.q_heads, p.q_weight != nullptr, wq);
        else work(s, now, static_cast<T*>(p.k_out), (int)p.k_heads, p.k_weight != nullptr, wk);
        return after;
    };
    Raw even, odd;  // (in turns: a copy would wait for the loads)
    if (here.token < arg.tokens) load(here, even);
    while (here.token < arg.tokens) {
        const Stop there = at(here, even, odd);
        if (there.token >= arg.tokens) break;
        here = at(there, odd, even);
    }
}

// Backward: with d = the gradient turned back, dweight += d x^, and dx = rstd
// (d w - x^ mean(d w x^)), x^ = x rstd. A block walks over tokens and keeps
// its lanes' shares of the weights' gradients; they are added over the block's
// heads and wavefronts at its end, and over the blocks by a second kernel.
template <typename T, int LPH, bool INTER, bool WHOLE> __global__ void __launch_bounds__(256) rotary_bwd_kernel(const RotaryArgs arg) {
    const cc1d_rotary_params& p = arg.p;
    const cc1d_rotary_bwd_params& g = arg.b;
    constexpr int HEADS = 64 / LPH, K = sizeof(T) == 2 ? 2 : 1;
    typedef Stop<HEADS * K> Stop;
    __shared__ float share_lds[2][4][LPH * 8];
    const int wave = uniform32(threadIdx.x >> 6), lane = threadIdx.x & 63, dim = (int)p.dim, rotated = (int)p.rotated;
    const int first = wave % arg.share * HEADS;
    const uint32_t per = 4 / arg.share, turns = arg.blocks * per;
    const Unit u = unit_of<INTER>(lane % LPH, dim, rotated);
    Angles a;
    float wq[8], wk[8], dwq[8], dwk[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const bool in = (e & 3) < u.count[e >> 2];
        wq[e] = p.q_weight && in ? p.q_weight[u.at[e >> 2] + (e & 3)] : 1.0f;
        wk[e] = p.k_weight && in ? p.k_weight[u.at[e >> 2] + (e & 3)] : 1.0f;
        dwq[e] = dwk[e] = 0.0f;
    }
    const float inv = 1.0f / (float)dim, eps = (float)p.eps;
    struct Raw {
        Four<T> v[K][2], d[K][2];
    };
    auto load = [&](const Stop& s, Raw& r) {
        const uint32_t b = arg.seqlen.div(s.token), t = s.token - b * (uint32_t)p.seqlen;
        const int64_t (&stride)[4] = s.which ? p.k_stride : p.q_stride;
        const int64_t (&gstride)[4] = s.which ? g.dk_out_stride : g.dq_out_stride;
        const T* const base = static_cast<const T*>(s.which ? p.k : p.q) + b * stride[0] + t * stride[1];
        const T* const gbase = static_cast<const T*>(s.which ? g.dk_out : g.dq_out) + b * gstride[0] + t * gstride[1];
        const int count = s.which ? (int)p.k_heads : (int)p.q_heads;
        const bool norm = (s.which ? p.k_weight : p.q_weight) != nullptr;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int h = s.h + j * arg.share * HEADS + lane / LPH;
            if constexpr (WHOLE) {
                const int64_t hc = h < count ? h : count - 1;
                const T* const gat = gbase + hc * gstride[2];
                const T* const at = norm ? base + hc * stride[2] : gat;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int e = u.count[i] ? u.at[i] : 0;
                    r.d[j][i].whole(gat + e);
                    r.v[j][i].whole(at + e);
                }
                continue;
            }
            if (h >= count) continue;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                r.d[j][i].load(gbase + h * gstride[2] + u.at[i] * gstride[3], gstride[3], u.count[i]);
                if (norm) r.v[j][i].load(base + h * stride[2] + u.at[i] * stride[3], stride[3], u.count[i]);
            }
        }
    };
    auto work = [&](const Stop& s, const Raw& r, T* dst, int count, bool norm, const float (&w)[8], float (&dw)[8]) {
        T* const out = dst + (int64_t)s.token * count * dim;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int h = s.h + j * arg.share * HEADS + lane / LPH;
            if (h >= count) continue;
            float d[8];
            r.d[j][0].get(d, !WHOLE || u.count[0]);
            r.d[j][1].get(d + 4, !WHOLE || u.count[1]);
            turn<INTER, true>(d, a, u, rotated >> 1);
            if (norm) {
                float x[8], sum = 0.0f, along = 0.0f;
                r.v[j][0].get(x, !WHOLE || u.count[0]);
                r.v[j][1].get(x + 4, !WHOLE || u.count[1]);
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
            for (int i = 0; i < 2; ++i) store_four(out + (int64_t)h * dim + u.at[i], d + 4 * i, u.count[i]);
        }
    };
    Stop here = {blockIdx.x * per + wave / arg.share, 0, first};
    here.settle(arg, first, turns);
    uint32_t angles_at = ~0u;
    // the work of a stop, with the loads of the one after it on their way
    auto at = [&](const Stop& s, const Raw& now, Raw& ahead) {
        const Stop after = s.next(arg, first, turns);
        if (WHOLE || after.token < arg.tokens) load(after.token < arg.tokens ? after : s, ahead);
        if (s.token != angles_at) {
            angles_at = s.token;
            const uint32_t b = arg.seqlen.div(s.token);
            a = angles_of(p, b, s.token - b * (uint32_t)p.seqlen, u);
        }
        if (s.which == 0) work(s, now, static_cast<T*>(g.dq), (int)p.q_heads, p.q_weight != nullptr, wq, dwq);
        else work(s, now, static_cast<T*>(g.dk), (int)p.k_heads, p.k_weight != nullptr, wk, dwk);
        return after;
    };
    Raw even, odd;  // (in turns: a copy would wait for the loads)
    if (here.token < arg.tokens) load(here, even);
    while (here.token < arg.tokens) {
        const Stop there = at(here, even, odd);
        if (there.token >= arg.tokens) break;
        here = at(there, odd, even);
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

// Sums of a column of the blocks' shares, in a fixed order: eight columns (32 bytes) a block, 32 rows at a time, eight
// of them on their way.
__global__ void __launch_bounds__(256) rotary_weights_kernel(const RotaryArgs arg) {
    __shared__ float sums[32][9];
    const int c = threadIdx.x & 7, r = threadIdx.x >> 3, dim = (int)arg.p.dim;
    float* const out = blockIdx.y ? arg.b.dk_weight : arg.b.dq_weight;
    if ((blockIdx.y ? arg.p.k_weight : arg.p.q_weight) == nullptr) return;
    const int col = blockIdx.x * 8 + c;
    float s = 0.0f;
    if (col < dim) {
        const float* const at = arg.b.workspace + (int64_t)blockIdx.y * arg.blocks * dim + col;
        for (uint32_t i = r; i < arg.blocks; i += 8 * 32) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = i + 32 * k < arg.blocks ? at[(int64_t)(i + 32 * k) * dim] : 0.0f;
            s += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        }
    }
    sums[r][c] = s;
    __syncthreads();
    if (r == 0 && col < dim) {
        for (int i = 1; i < 32; ++i) s += sums[i][c];
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

template <typename F> int with_lanes(const cc1d_rotary_params& p, bool whole, F&& f) {
    return with_flag(p.interleaved != 0, [&](auto inter) {
        return with_flag(whole, [&](auto w) {
            switch (head_lanes(p)) {
            case 8: return f(std::integral_constant<int, 8>{}, inter, w);
            case 16: return f(std::integral_constant<int, 16>{}, inter, w);
            case 32: return f(std::integral_constant<int, 32>{}, inter, w);
            default: return f(std::integral_constant<int, 64>{}, inter, w);
            }
        });
    });
}

// Whether every run of a lane is four neighbours or none.
bool whole_runs(const cc1d_rotary_params& p) {
    const bool fours = p.dim % 4 == 0 && (p.interleaved || p.rotated % 8 == 0);
    return fours && (p.q_heads == 0 || p.q_stride[3] == 1) && (p.k_heads == 0 || p.k_stride[3] == 1);
}

// Several wavefronts share a token where there are too few tokens to fill the chip, and heads enough for each.
int share_of(const cc1d_rotary_params& p) {
    const int64_t heads = p.q_heads > p.k_heads ? p.q_heads : p.k_heads;
    return p.batch * p.seqlen < 8192 && heads * head_lanes(p) > 2 * 64 ? 4 : 1;
}

int64_t blocks_of(const cc1d_rotary_params& p, int64_t most) {
    const int64_t n = ceil_div(p.batch * p.seqlen, 4 / share_of(p));
    return n < 1 ? 1 : n < most ? n : most;
}

RotaryArgs args_of(const cc1d_rotary_params& p, int64_t most) {
    RotaryArgs a{};
    a.p = p;
    a.tokens = (uint32_t)(p.batch * p.seqlen);
    a.seqlen = FastDiv((uint32_t)(p.seqlen > 0 ? p.seqlen : 1));
    a.share = share_of(p);
    a.blocks = (uint32_t)blocks_of(p, most);
    return a;
}

constexpr int64_t kFwdBlocks = 1024, kBwdBlocks = 768;

}  // namespace

int launch_rotary_fwd(const cc1d_rotary_params& p, hipStream_t stream) {
    const RotaryArgs a = args_of(p, kFwdBlocks);
    const dim3 grid(a.blocks);
    return with_dtype(p.dtype, [&](auto t) {
        return with_lanes(p, whole_runs(p), [&](auto l, auto inter, auto w) {
            return launch(rotary_kernel<decltype(t), decltype(l)::value, decltype(inter)::value, decltype(w)::value>, grid, dim3(256), stream, a);
        });
    });
}

int64_t rotary_bwd_workspace_floats(const cc1d_rotary_bwd_params& b) {
    return b.fwd.q_weight || b.fwd.k_weight ? 2 * blocks_of(b.fwd, kBwdBlocks) * b.fwd.dim : 0;
}

int launch_rotary_bwd(const cc1d_rotary_bwd_params& b, hipStream_t stream) {
    const cc1d_rotary_params& p = b.fwd;
    RotaryArgs a = args_of(p, kBwdBlocks);
    a.b = b;
    const bool whole = whole_runs(p) && (p.q_heads == 0 || b.dq_out_stride[3] == 1) && (p.k_heads == 0 || b.dk_out_stride[3] == 1);
    const int st = with_dtype(p.dtype, [&](auto t) {
        return with_lanes(p, whole, [&](auto l, auto inter, auto w) {
            return launch(rotary_bwd_kernel<decltype(t), decltype(l)::value, decltype(inter)::value, decltype(w)::value>, dim3(a.blocks), dim3(256), stream, a);
        });
    });
    if (st != CC1D_OK || (!p.q_weight && !p.k_weight)) return st;
    return launch(rotary_weights_kernel, dim3((unsigned)ceil_div(p.dim, 8), 2), dim3(256), stream, a);
}

}  // namespace cc1d
