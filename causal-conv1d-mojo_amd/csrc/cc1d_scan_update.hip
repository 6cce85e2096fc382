// cc1d_scan_update.hip -- decode step of the selective state space scan.
//
// Per (batch entry, channel) the state's dstate values are read, moved by one
// step per new token (h = exp(dt A) h + dt u B), multiplied with C, and
// written back: 8 bytes of state per value, everything else shared by the
// dstate values of a channel or the channels of a group, so HBM bounds it: 38
// us at 256 x 5120 x 16 (4.6 TB/s; a copy of these bytes 28). Four tokens at 31
// x 4096 x 64 take 28 us, of which the bytes are 11: there the steps themselves
// (an exponential and three more per state and token) bound it.
#include "cc1d_scan_device.hpp"

namespace cc1d {
namespace {

struct UpdateArgs {
    cc1d_scan_update_params p;
    uint32_t blocks;  // per batch entry
    FastDiv blocks_div, group;  // of blocks; of a group's channels
};

// Element `i` (units of stride) past a wave-uniform base. WIDE: the tensor's
// extent of channels and states does not fit 32-bit byte offsets.
template <bool WIDE, typename P> __device__ __forceinline__ P* past(P* base, uint32_t i, int64_t stride) {
    if constexpr (WIDE) return base + (int64_t)i * stride;
    else return reinterpret_cast<P*>(reinterpret_cast<uintptr_t>(base) + i * (uint32_t)(stride * (int64_t)sizeof(P)));
}

// Four of a channel's states from n on. VEC: unit stride, and dstate a
// multiple of 4 (lanes past it read its last four and count for nothing);
// else one by one, those there are.
template <bool VEC> struct Quad {
    float v[4];
    template <bool NT = false, typename P> __device__ __forceinline__ void load(const P* base, int64_t stride, int n, int N) {
        if constexpr (VEC) {
            const P* at = base + (n < N ? n : N - 4);
            if constexpr (sizeof(P) == 4) {
                const u32x4 w = NT ? vload_any_nt(at) : vload_any(at);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(w[j]);
            } else {
                const u32x2 w = *reinterpret_cast<const typename AnyAddr<2>::v2*>(at);
                const u32x4 w4 = {w[0], w[1], 0u, 0u};
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = vget<P>(w4, j);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = n + j < N ? to_f32(base[(n + j) * stride]) : 0.0f;
        }
    }
    __device__ __forceinline__ void store(float* base, int64_t stride, int n, int N) const {
        if constexpr (VEC) {
            if (n < N)
                vstore_any_nt(base + n, u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])});
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (n + j < N) base[(n + j) * stride] = v[j];
        }
    }
};

template <int T> __device__ __forceinline__ float quad_lane(float v) {  // lane T of each quad's value
    return dpp_f32<T * 0x55, 0xf>(v);
}

// LPC lanes hold a channel's states, four each; a block takes 256 / LPC
// channels of a batch entry (two or four entries per block, to share A, were
// slower: 60 and 64 us against 53 at 256 x 5120 x 16, fewer wavefronts fitting
// beside each other). Tokens go by four: a lane of a quad forms the step, the
// gate and the output of its own one, which the quad's others take over.
// TOK: tokens at a time, 1 or 4.
template <typename T, int LPC, bool WIDE, bool VEC, int TOK> __global__ void __launch_bounds__(256) scan_update_kernel(const UpdateArgs arg) {
    const cc1d_scan_update_params& p = arg.p;
    constexpr uint32_t PER = 256 / LPC;
    const int sub = threadIdx.x % LPC, n = 4 * sub, N = (int)p.dstate, tokens = (int)p.seqlen;
    const uint32_t b = arg.blocks_div.div(blockIdx.x);
    const uint32_t d = (blockIdx.x - b * arg.blocks) * PER + threadIdx.x / LPC;
    if (d >= (uint32_t)p.dim) return;  // (a channel's lanes leave together)
    T* const out_row = static_cast<T*>(p.out) + b * p.out_stride[0];
    const int64_t row = p.ssm_state_indices ? ld_uniform(p.ssm_state_indices + b) : b;
    if (row < 0 || row >= p.state_rows) {
        for (int t = sub; t < tokens; t += LPC) past<WIDE>(out_row, d, p.out_stride[1])[t * p.out_stride[2]] = T{};
        return;
    }
    const uint32_t g = arg.group.div(d);
    float* const state = past<WIDE>(p.ssm_state + row * p.ssm_state_stride[0], d, p.ssm_state_stride[1]);
    Quad<VEC> h, A;
    h.template load<true>(state, p.ssm_state_stride[2], n, N);
    A.load(past<WIDE>(p.A, d, p.A_stride[0]), p.A_stride[1], n, N);
    const T* u = past<WIDE>(static_cast<const T*>(p.u) + b * p.u_stride[0], d, p.u_stride[1]);
    const T* delta = past<WIDE>(static_cast<const T*>(p.delta) + b * p.delta_stride[0], d, p.delta_stride[1]);
    const T* z = p.z ? past<WIDE>(static_cast<const T*>(p.z) + b * p.z_stride[0], d, p.z_stride[1]) : nullptr;
    const T* B = past<WIDE>(static_cast<const T*>(p.B) + b * p.B_stride[0], g, p.B_stride[1]);
    const T* C = past<WIDE>(static_cast<const T*>(p.C) + b * p.C_stride[0], g, p.C_stride[1]);
    T* out = past<WIDE>(out_row, d, p.out_stride[1]);
    const float bias = p.delta_bias ? *past<WIDE>(p.delta_bias, d, p.delta_bias_stride) : 0.0f;
    const float skip = p.D ? *past<WIDE>(p.D, d, p.D_stride) : 0.0f;

    for (int t0 = 0; t0 < tokens; t0 += TOK) {
        const int last = TOK == 1 ? 0 : tokens - 1 - t0, mine = (sub & 3) < last ? (sub & 3) : last;  // the quad's tokens: 0 .. min(3, last)
        const int64_t t = t0 + mine;
        const float uv = to_f32(u[t * p.u_stride[2]]);
        const float raw = to_f32(delta[t * p.delta_stride[2]]) + bias;
        const float zv = z ? to_f32(z[t * p.z_stride[2]]) : 0.0f;
        Quad<VEC> Bq[TOK], Cq[TOK];
#pragma unroll
        for (int i = 0; i < TOK; ++i) {
            if (i > last) continue;
            Bq[i].load(B + (t0 + i) * p.B_stride[3], p.B_stride[2], n, N);
            Cq[i].load(C + (t0 + i) * p.C_stride[3], p.C_stride[2], n, N);
        }
        if (t0 == 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j) A.v[j] *= kLog2e;
        }
        const float dt = p.delta_softplus ? softplus(raw) : raw;
        const float du = dt * uv;
        float y = 0.0f;
        auto token = [&](auto which) {
            constexpr int i = decltype(which)::value;
            if (i > last) return;
            const float ds = TOK == 1 ? dt : quad_lane<i>(dt), us = TOK == 1 ? du : quad_lane<i>(du);
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                h.v[j] = __builtin_fmaf(__builtin_amdgcn_exp2f(ds * A.v[j]), h.v[j], us * Bq[i].v[j]);
                if (VEC || n + j < N) sum = __builtin_fmaf(Cq[i].v[j], h.v[j], sum);
            }
            if (VEC && n >= N) sum = 0.0f;
            sum = lanes_sum<LPC>(sum);
            if (mine == i) y = sum;
        };
        token(std::integral_constant<int, 0>{});
        if constexpr (TOK > 1) {
            token(std::integral_constant<int, 1>{});
            token(std::integral_constant<int, 2>{});
            token(std::integral_constant<int, 3>{});
        }
        y = __builtin_fmaf(skip, uv, y);
        if (z) y *= silu(zv);
        if (sub <= (last < TOK - 1 ? last : TOK - 1)) out[t * p.out_stride[2]] = from_f32<T>(y);
    }
    h.store(state, p.ssm_state_stride[2], n, N);
}

}  // namespace

int launch_scan_update(const cc1d_scan_update_params& p, hipStream_t stream) {
    int lpc = 4;
    while (4 * lpc < p.dstate) lpc *= 2;
    const uint32_t blocks = (uint32_t)ceil_div(p.dim, 256 / lpc);
    const UpdateArgs a{p, blocks, FastDiv(blocks), FastDiv((uint32_t)(p.dim / p.groups))};
    const dim3 grid((unsigned)(blocks * p.batch));
    // byte offsets of the last channel (and group) from the batch entry's base
    bool wide = false;
    auto reach = [&](int64_t count, int64_t stride, int64_t size) {
        wide = wide || stride < 0 || (double)count * (double)stride * (double)size >= (double)((int64_t)1 << 32);
    };
    const int es = p.dtype == CC1D_DTYPE_FP32 ? 4 : 2;
    for (const int64_t* s : {p.u_stride, p.delta_stride, p.z_stride, p.out_stride}) reach(p.dim, s[1], es);
    reach(p.dim, p.ssm_state_stride[1], 4);
    reach(p.dim, p.A_stride[0], 4);
    reach(p.dim, p.D_stride, 4);
    reach(p.dim, p.delta_bias_stride, 4);
    reach(p.groups, p.B_stride[1], es);
    reach(p.groups, p.C_stride[1], es);
    const bool vec = p.dstate % 4 == 0 && p.ssm_state_stride[2] == 1 && p.A_stride[1] == 1 && p.B_stride[2] == 1 &&
                     p.C_stride[2] == 1 && !wide;
    return with_dtype(p.dtype, [&](auto t) {
        auto go = [&](auto l) {
            typedef decltype(t) T;
            constexpr int LPC = decltype(l)::value;
            if (vec && p.seqlen == 1) return launch(scan_update_kernel<T, LPC, false, true, 1>, grid, dim3(256), stream, a);
            if (vec) return launch(scan_update_kernel<T, LPC, false, true, 4>, grid, dim3(256), stream, a);
            return launch(scan_update_kernel<T, LPC, true, false, 4>, grid, dim3(256), stream, a);
        };
        switch (lpc) {
        case 4: return go(std::integral_constant<int, 4>{});
        case 8: return go(std::integral_constant<int, 8>{});
        case 16: return go(std::integral_constant<int, 16>{});
        case 32: return go(std::integral_constant<int, 32>{});
        default: return go(std::integral_constant<int, 64>{});
        }
    });
}

}  // namespace cc1d
