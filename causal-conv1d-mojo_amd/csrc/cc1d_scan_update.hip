// cc1d_scan_update.hip -- decode step of the selective state space scan.
//
// Per (batch entry, channel) the state's dstate values are read, moved by one
// step per new token (h = exp(dt A) h + dt u B), multiplied with C, and
// written back: 8 bytes of state per value, everything else shared by the
// dstate values of a channel or the channels of a group, so HBM bounds it.
#include "cc1d_scan_device.hpp"

namespace cc1d {
namespace {

// One thread per (batch entry, channel, state): LPC lanes of a wavefront (the
// next power of two, or 64 lanes in turns) hold a channel's states.
template <typename T> __global__ void __launch_bounds__(256) scan_update_kernel(const cc1d_scan_update_params p, int lpc) {
    const int per = 256 / lpc;
    const int64_t blocks = (p.dim + per - 1) / per, b = blockIdx.x / blocks;
    const int sub = threadIdx.x % lpc;
    const int64_t d = blockIdx.x % blocks * per + threadIdx.x / lpc;
    if (d >= p.dim) return;
    T* out = static_cast<T*>(p.out) + b * p.out_stride[0] + d * p.out_stride[1];
    const int64_t row = p.ssm_state_indices ? p.ssm_state_indices[b] : b;
    if (row < 0 || row >= p.state_rows) {
        if (sub == 0)
            for (int64_t t = 0; t < p.seqlen; ++t) out[t * p.out_stride[2]] = T{};
        return;
    }
    const T* u = static_cast<const T*>(p.u) + b * p.u_stride[0] + d * p.u_stride[1];
    const T* delta = static_cast<const T*>(p.delta) + b * p.delta_stride[0] + d * p.delta_stride[1];
    const T* z = p.z ? static_cast<const T*>(p.z) + b * p.z_stride[0] + d * p.z_stride[1] : nullptr;
    const int64_t g = d / (p.dim / p.groups);
    const T* Bp = static_cast<const T*>(p.B) + b * p.B_stride[0] + g * p.B_stride[1];
    const T* Cp = static_cast<const T*>(p.C) + b * p.C_stride[0] + g * p.C_stride[1];
    float* state = p.ssm_state + row * p.ssm_state_stride[0] + d * p.ssm_state_stride[1];
    const float bias = p.delta_bias ? p.delta_bias[d * p.delta_bias_stride] : 0.0f;
    const float skip = p.D ? p.D[d * p.D_stride] : 0.0f;
    for (int64_t t = 0; t < p.seqlen; ++t) {
        const float uu = to_f32(u[t * p.u_stride[2]]);
        const float raw = to_f32(delta[t * p.delta_stride[2]]) + bias;
        const float dt = p.delta_softplus ? softplus(raw) : raw;
        float y = 0.0f;
        for (int64_t n = sub; n < p.dstate; n += lpc) {
            const float a = __builtin_amdgcn_exp2f(dt * (p.A[d * p.A_stride[0] + n * p.A_stride[1]] * kLog2e));
            const float h = __builtin_fmaf(a, state[n * p.ssm_state_stride[2]],
                                           dt * uu * to_f32(Bp[n * p.B_stride[2] + t * p.B_stride[3]]));
            state[n * p.ssm_state_stride[2]] = h;
            y = __builtin_fmaf(h, to_f32(Cp[n * p.C_stride[2] + t * p.C_stride[3]]), y);
        }
        for (int w = lpc / 2; w > 0; w /= 2) y += __shfl_xor(y, w);
        y = __builtin_fmaf(skip, uu, y);
        if (z) y *= silu(to_f32(z[t * p.z_stride[2]]));
        if (sub == 0) out[t * p.out_stride[2]] = from_f32<T>(y);
    }
}

}  // namespace

int launch_scan_update(const cc1d_scan_update_params& p, hipStream_t stream) {
    int lpc = 1;
    while (lpc < 64 && lpc < p.dstate) lpc *= 2;
    return with_dtype(p.dtype, [&](auto t) {
        const dim3 grid((unsigned)(ceil_div(p.dim, 256 / lpc) * p.batch));
        return launch(scan_update_kernel<decltype(t)>, grid, dim3(256), stream, p, lpc);
    });
}

}  // namespace cc1d
