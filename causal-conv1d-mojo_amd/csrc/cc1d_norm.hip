// cc1d_norm.hip -- residual add and layer / rms norm, forward and backward.
#include "cc1d_internal.hpp"

namespace cc1d {
namespace {

__device__ __forceinline__ float block_sum(float v, float* lds) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}

template <typename T, typename R>
__device__ __forceinline__ float row_value(const T* x, const R* res, int64_t i) {
    const float v = x ? to_f32(x[i]) : 0.0f;
    return res ? v + to_f32(res[i]) : v;
}

// One block per row, three passes over it.
template <typename T, typename R> __global__ void __launch_bounds__(256) norm_fwd_kernel(const cc1d_norm_params p) {
    __shared__ float lds[4];
    const int64_t row = blockIdx.x;
    const T* x = static_cast<const T*>(p.x) + row * p.x_stride;
    const R* res = p.residual ? static_cast<const R*>(p.residual) + row * p.residual_stride : nullptr;
    float mean = 0.0f, var = 0.0f;
    if (!p.rms) {
        for (int64_t i = threadIdx.x; i < p.dim; i += 256) mean += row_value(x, res, i);
        mean = block_sum(mean, lds) / (float)p.dim;
    }
    for (int64_t i = threadIdx.x; i < p.dim; i += 256) {
        const float o = row_value(x, res, i) - mean;
        var = __builtin_fmaf(o, o, var);
    }
    var = block_sum(var, lds) / (float)p.dim;
    const float rstd = 1.0f / __builtin_sqrtf(var + (float)p.eps);
    for (int64_t i = threadIdx.x; i < p.dim; i += 256) {
        const float r = row_value(x, res, i);
        const float y = __builtin_fmaf((r - mean) * rstd, p.weight[i * p.weight_stride],
                                       p.bias ? p.bias[i * p.bias_stride] : 0.0f);
        static_cast<T*>(p.y)[row * p.y_stride + i] = from_f32<T>(y);
        if (p.sum) static_cast<R*>(p.sum)[row * p.sum_stride + i] = from_f32<R>(r);
    }
    if (p.stats && threadIdx.x == 0) {
        p.stats[2 * row] = mean;
        p.stats[2 * row + 1] = rstd;
    }
}

template <typename T, typename R> __global__ void __launch_bounds__(256) norm_bwd_kernel(const cc1d_norm_bwd_params b) {
    __shared__ float lds[4];
    const cc1d_norm_params& p = b.fwd;
    const int64_t row = blockIdx.x;
    const T* x = p.x ? static_cast<const T*>(p.x) + row * p.x_stride : nullptr;
    const R* res = p.residual ? static_cast<const R*>(p.residual) + row * p.residual_stride : nullptr;
    const T* dy = static_cast<const T*>(b.dy) + row * b.dy_stride;
    const float mean = p.stats[2 * row], rstd = p.stats[2 * row + 1];
    float level = 0.0f, along = 0.0f;
    for (int64_t i = threadIdx.x; i < p.dim; i += 256) {
        const float xh = (row_value(x, res, i) - mean) * rstd;
        const float d = to_f32(dy[i]) * p.weight[i * p.weight_stride];
        level += d;
        along = __builtin_fmaf(d, xh, along);
    }
    level = p.rms ? 0.0f : block_sum(level, lds) / (float)p.dim;
    along = block_sum(along, lds) / (float)p.dim;
    for (int64_t i = threadIdx.x; i < p.dim; i += 256) {
        const float xh = (row_value(x, res, i) - mean) * rstd;
        float d = (to_f32(dy[i]) * p.weight[i * p.weight_stride] - level - xh * along) * rstd;
        if (b.dsum) d += to_f32(static_cast<const R*>(b.dsum)[row * b.dsum_stride + i]);
        static_cast<T*>(b.dx)[row * b.dx_stride + i] = from_f32<T>(d);
        if (b.dresidual) static_cast<R*>(b.dresidual)[row * b.dresidual_stride + i] = from_f32<R>(d);
    }
}

// Partial sums of a share of the rows, one thread per column.
template <typename T, typename R>
__global__ void __launch_bounds__(256) norm_bwd_columns(const cc1d_norm_bwd_params b, int64_t share) {
    const cc1d_norm_params& p = b.fwd;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= p.dim) return;
    const int64_t from = blockIdx.y * share, to = from + share < p.rows ? from + share : p.rows;
    float dw = 0.0f, db = 0.0f;
    for (int64_t row = from; row < to; ++row) {
        const T* x = p.x ? static_cast<const T*>(p.x) + row * p.x_stride : nullptr;
        const R* res = p.residual ? static_cast<const R*>(p.residual) + row * p.residual_stride : nullptr;
        const float dy = to_f32(static_cast<const T*>(b.dy)[row * b.dy_stride + i]);
        dw = __builtin_fmaf(dy, (row_value(x, res, i) - p.stats[2 * row]) * p.stats[2 * row + 1], dw);
        db += dy;
    }
    b.workspace[(2 * blockIdx.y) * p.dim + i] = dw;
    b.workspace[(2 * blockIdx.y + 1) * p.dim + i] = db;
}

__global__ void __launch_bounds__(256) norm_bwd_reduce(const cc1d_norm_bwd_params b, int64_t parts) {
    const int64_t dim = b.fwd.dim, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= dim) return;
    float dw = 0.0f, db = 0.0f;
    for (int64_t k = 0; k < parts; ++k) {
        dw += b.workspace[2 * k * dim + i];
        db += b.workspace[(2 * k + 1) * dim + i];
    }
    b.dweight[i] = dw;
    if (b.dbias) b.dbias[i] = db;
}

constexpr int64_t kShare = 64;  // rows of a partial sum

template <typename F> int with_norm_types(const cc1d_norm_params& p, F&& f) {
    return with_dtype(p.dtype, [&](auto t) {
        return p.residual_dtype == p.dtype ? f(t, t) : f(t, float{});
    });
}

}  // namespace

int64_t norm_bwd_workspace_floats(const cc1d_norm_bwd_params& b) {
    return 2 * ceil_div(b.fwd.rows, kShare) * b.fwd.dim;
}

int launch_norm_fwd(const cc1d_norm_params& p, hipStream_t stream) {
    return with_norm_types(p, [&](auto t, auto r) {
        return launch(norm_fwd_kernel<decltype(t), decltype(r)>, dim3((unsigned)p.rows), dim3(256), stream, p);
    });
}

int launch_norm_bwd(const cc1d_norm_bwd_params& b, hipStream_t stream) {
    const cc1d_norm_params& p = b.fwd;
    const int64_t parts = ceil_div(p.rows, kShare);
    return with_norm_types(p, [&](auto t, auto r) {
        typedef decltype(t) T;
        typedef decltype(r) R;
        const unsigned cols = (unsigned)ceil_div(p.dim, 256);
        int st = CC1D_OK;
        if (p.rows > 0) st = launch(norm_bwd_kernel<T, R>, dim3((unsigned)p.rows), dim3(256), stream, b);
        if (st == CC1D_OK && p.rows > 0)
            st = launch(norm_bwd_columns<T, R>, dim3(cols, (unsigned)parts), dim3(256), stream, b, kShare);
        if (st == CC1D_OK) st = launch(norm_bwd_reduce, dim3(cols), dim3(256), stream, b, parts);
        return st;
    });
}

}  // namespace cc1d
