// cc1d_norm.hip -- residual add and layer / rms norm, forward and backward.
//
// Bandwidth kernels: every value is read once and stays on the chip, 8 per
// lane and step, while its row's sums are formed (the mean first, then the
// spread around it), so rows go through the card once each way. At 8192 x 2560
// bf16 with an fp32 residual: forward 56 us (4.5 TB/s), backward 77 (4.4) and its
// reduction 9; a copy reaches 6.3 with non-temporal accesses, 5.0 without.
//
// Rows of up to 8192 columns (one step a lane) fit in registers. Wider ones
// have 2 to 4 steps a lane in blocks of up to 16 wavefronts, whose 128 registers
// a lane do not hold them: the backward spills 216, 652 and 980 bytes a lane at
// 2, 3 and 4 steps (forward 0, 68, 256, or 188 to 844 where the width is no
// multiple of 8). Same bytes, bf16 with an fp32 residual: 2048 x 8192 takes 54
// and 67 us, 2048 x 12288 (half as much again) 78 and 198, 1024 x 32768 (twice)
// 213 and 636.
#include "cc1d_internal.hpp"
#include "cc1d_steps.hpp"

namespace cc1d {
namespace {

constexpr int E = 8;              // values per lane and step

// Where a lane stands: LPR lanes of a wavefront (64 / LPR rows at a time), or
// `wpr` whole wavefronts, share a row. At step i a lane has positions
// at(i) .. at(i) + 7. EVEN: dim is a multiple of 8 and the parameters lie
// together, so a lane has all 8 or none (and reads the row's last 8 instead);
// else a row's last lane has some of them, moved into place after loading.
template <int LPR, bool EVEN> struct Place {
    static constexpr int CHUNK = LPR * E;
    int lane, wave, sub, wpr, dim;
    __device__ __forceinline__ int at(int i) const { return ((i * wpr + sub) * LPR + lane) * E; }
    __device__ __forceinline__ bool any(int i) const { return (i * wpr + sub) * CHUNK < dim; }       // wave-uniform
    __device__ __forceinline__ bool full(int i) const { return (i * wpr + sub + 1) * CHUNK <= dim; }  // wave-uniform
    __device__ __forceinline__ bool in(int i, int j) const { return EVEN ? at(i) < dim : at(i) + j < dim; }
    template <typename T> __device__ __forceinline__ void load(Raw<T, E>& r, const T* row, int i) const {
        if (EVEN || LPR > 8 || dim >= E) r.template load<true>(row, at(i), dim);
        else r.each(row, 1, at(i), dim);
    }
    template <typename T> __device__ __forceinline__ void fix(Raw<T, E>& r, int i) const {
        if (full(i)) return;
        if constexpr (EVEN) {
#pragma unroll
            for (int k = 0; k < Raw<T, E>::DW; ++k) r.w[k] = at(i) < dim ? r.w[k] : 0u;
        } else {
            if (LPR > 8 || dim >= E) r.fix(at(i), dim, dim);
        }
    }
    template <typename T> __device__ __forceinline__ void store(T* row, int i, const float (&v)[E]) const {
        if constexpr (EVEN) {
            if (at(i) < dim) {
#pragma unroll
                for (int q = 0; q < E / elems16<T>::value; ++q)
                    vstore_any_nt(row + at(i) + q * elems16<T>::value, vpack<T>(v + q * elems16<T>::value));
            }
        } else {
            store_steps<T, E, true>(row, 1, at(i), dim, v);
        }
    }
    // parameters
    __device__ __forceinline__ void params(const float* w, int64_t stride, int i, float (&v)[E]) const {
        if constexpr (EVEN) {
            const int from = at(i) < dim ? at(i) : dim - E;
#pragma unroll
            for (int q = 0; q < E / 4; ++q) {
                const u32x4 x = vload_any(w + from + 4 * q);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[4 * q + j] = __uint_as_float(x[j]);
            }
        } else if (stride == 1 && dim >= E) {
            Raw<float, E> r;
            r.load(w, at(i), dim);
            if (!full(i)) r.fix(at(i), dim, dim);
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] = r.get(j);
        } else {
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] = at(i) + j < dim ? w[(at(i) + j) * stride] : 0.0f;
        }
    }
    // Sum of a row; lds: a float per wavefront of the block.
    __device__ __forceinline__ float row_sum(float v, float* lds) const {
        v = lanes_sum<LPR>(v);
        if (LPR < 64 || wpr == 1) return v;
        __syncthreads();
        if (lane == 0) lds[wave] = v;
        __syncthreads();
        const float* row = lds + wave - sub;
        float sum = 0.0f;
        for (int w = 0; w < wpr; ++w) sum += row[w];
        return sum;
    }
};
template <int LPR, bool EVEN> __device__ __forceinline__ Place<LPR, EVEN> place(int64_t dim, int wpr) {
    const int wave = (int)uniform32(threadIdx.x >> 6);
    return {(int)threadIdx.x % LPR, wave, wave % wpr, wpr, (int)dim};
}

// T: x and y; R: the residual and the sum. A block's rows go on in steps of
// the grid. Values and parameters are asked for at once, before the sums.
template <typename T, typename R, int STEPS, int LPR, bool EVEN>
__global__ void __launch_bounds__(STEPS == 1 && LPR == 64 ? 1024 : (STEPS == 1 ? 256 : 1024))
norm_fwd_kernel(const cc1d_norm_params p, int wpr) {
    __shared__ float lds[16];
    const Place<LPR, EVEN> at = place<LPR, EVEN>(p.dim, wpr);
    const int slots = (int)(blockDim.x / LPR) / wpr, slot = LPR == 64 ? at.wave / wpr : (int)threadIdx.x / LPR;
    const float inv = 1.0f / (float)p.dim;
    for (int64_t first = (int64_t)blockIdx.x * slots; first < p.rows; first += (int64_t)gridDim.x * slots) {
        const int64_t want = first + slot, row = want < p.rows ? want : p.rows - 1;  // (the barriers are the block's)
        Raw<T, E> rx[STEPS];
        Raw<R, E> rr[STEPS];
        float w[STEPS][E], c[STEPS][E];
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            if (!at.any(i)) continue;
            at.load(rx[i], static_cast<const T*>(p.x) + row * p.x_stride, i);
            if (p.residual) at.load(rr[i], static_cast<const R*>(p.residual) + row * p.residual_stride, i);
            at.params(p.weight, p.weight_stride, i, w[i]);
            if (p.bias) at.params(p.bias, p.bias_stride, i, c[i]);
        }
        float v[STEPS][E], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            if (!at.any(i)) continue;
            at.fix(rx[i], i);
            if (p.residual) at.fix(rr[i], i);
#pragma unroll
            for (int j = 0; j < E; ++j) {
                v[i][j] = rx[i].get(j);
                if (p.residual) v[i][j] += rr[i].get(j);
                sum += v[i][j];
            }
            if (p.sum && want < p.rows)
                at.store(static_cast<R*>(p.sum) + row * p.sum_stride, i, v[i]);
        }
        const float mean = p.rms ? 0.0f : at.row_sum(sum, lds) * inv;
        float var = 0.0f;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            if (!at.any(i)) continue;
#pragma unroll
            for (int j = 0; j < E; ++j) {
                v[i][j] -= mean;
                if (!at.full(i)) v[i][j] = at.in(i, j) ? v[i][j] : 0.0f;
                var = __builtin_fmaf(v[i][j], v[i][j], var);
            }
        }
        const float rstd = 1.0f / __builtin_sqrtf(__builtin_fmaf(at.row_sum(var, lds), inv, (float)p.eps));
        if (want >= p.rows) continue;  // (only in the block's last turn)
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            if (!at.any(i)) continue;
#pragma unroll
            for (int j = 0; j < E; ++j) {
                v[i][j] *= rstd;
                v[i][j] = p.bias ? __builtin_fmaf(v[i][j], w[i][j], c[i][j]) : v[i][j] * w[i][j];
            }
            at.store(static_cast<T*>(p.y) + row * p.y_stride, i, v[i]);
        }
        if (p.stats && at.sub == 0 && at.lane == 0) {
            p.stats[2 * row] = mean;
            p.stats[2 * row + 1] = rstd;
        }
    }
}

// dx = rstd (dy w - mean(dy w) - xh mean(dy w xh)) + dsum, and the block's sums
// of dy xh and dy: a lane's columns are the same in every row it takes. A row's
// values are asked for while the one before is worked on, all of them, dsum
// too: loads return in order, so one asked for later would wait for the next row.
template <typename T, typename R, int STEPS, int LPR, bool EVEN>
__global__ void __launch_bounds__(STEPS == 1 && LPR == 64 ? 1024 : (STEPS == 1 ? 256 : 1024))
norm_bwd_kernel(const cc1d_norm_bwd_params b, int wpr) {
    constexpr int CHUNK = LPR * E;
    __shared__ float lds[16];
    __shared__ __attribute__((aligned(16))) float share[4 * STEPS * CHUNK];  // for blocks of several rows at a time (wpr 1 or 2)
    const cc1d_norm_params& p = b.fwd;
    const Place<LPR, EVEN> at = place<LPR, EVEN>(p.dim, wpr);
    const int slots = (int)(blockDim.x / LPR) / wpr, slot = LPR == 64 ? at.wave / wpr : (int)threadIdx.x / LPR;
    const float inv = 1.0f / (float)p.dim;
    float dw[STEPS][E], db[STEPS][E], w[STEPS][E];
#pragma unroll
    for (int i = 0; i < STEPS; ++i) {
#pragma unroll
        for (int j = 0; j < E; ++j) dw[i][j] = db[i][j] = 0.0f;
        if (at.any(i)) at.params(p.weight, p.weight_stride, i, w[i]);
    }
    Raw<T, E> rx[STEPS], rdy[STEPS];
    Raw<R, E> rr[STEPS], rs[STEPS];
    float mean, rstd;
    auto fetch = [&](int64_t row) {
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            if (!at.any(i)) continue;
            if (p.x) at.load(rx[i], static_cast<const T*>(p.x) + row * p.x_stride, i);
            if (p.residual) at.load(rr[i], static_cast<const R*>(p.residual) + row * p.residual_stride, i);
            at.load(rdy[i], static_cast<const T*>(b.dy) + row * b.dy_stride, i);
            if (b.dsum) at.load(rs[i], static_cast<const R*>(b.dsum) + row * b.dsum_stride, i);
        }
        mean = p.stats[2 * row];
        rstd = p.stats[2 * row + 1];
    };
    const int64_t turn = (int64_t)gridDim.x * slots;
    auto row_of = [&](int64_t first) { return first + slot < p.rows ? first + slot : p.rows - 1; };
    fetch(row_of((int64_t)blockIdx.x * slots));
    for (int64_t first = (int64_t)blockIdx.x * slots; first < p.rows; first += turn) {
        const bool mine = first + slot < p.rows;
        const int64_t row = row_of(first);
        float xh[STEPS][E], d[STEPS][E], s[STEPS][E], level = 0.0f, along = 0.0f;
        const float r1 = rstd;
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            if (!at.any(i)) continue;
            if (p.x) at.fix(rx[i], i);
            if (p.residual) at.fix(rr[i], i);
            at.fix(rdy[i], i);
            if (b.dsum) at.fix(rs[i], i);
#pragma unroll
            for (int j = 0; j < E; ++j) {
                float r = p.x ? rx[i].get(j) : 0.0f;
                if (p.residual) r += rr[i].get(j);
                xh[i][j] = (r - mean) * rstd;
                if (!at.full(i)) xh[i][j] = at.in(i, j) ? xh[i][j] : 0.0f;
                const float g = rdy[i].get(j);
                d[i][j] = g * w[i][j];
                level += d[i][j];
                along = __builtin_fmaf(d[i][j], xh[i][j], along);
                if (mine) {
                    dw[i][j] = __builtin_fmaf(g, xh[i][j], dw[i][j]);
                    db[i][j] += g;
                }
                s[i][j] = b.dsum ? rs[i].get(j) : 0.0f;
            }
        }
        if (first + turn < p.rows) fetch(row_of(first + turn));
        level = p.rms ? 0.0f : at.row_sum(level, lds) * inv;
        along = at.row_sum(along, lds) * inv;
        if (!mine) continue;  // (only in the block's last turn)
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
            if (!at.any(i)) continue;
#pragma unroll
            for (int j = 0; j < E; ++j) d[i][j] = __builtin_fmaf(d[i][j] - level - xh[i][j] * along, r1, s[i][j]);
            at.store(static_cast<T*>(b.dx) + row * b.dx_stride, i, d[i]);
            if (b.dresidual) at.store(static_cast<R*>(b.dresidual) + row * b.dresidual_stride, i, d[i]);
        }
    }
    // the slots' sums one after the other, the last one writes the block's
    for (int k = 0; k < slots; ++k) {
        if (k == slot) {
#pragma unroll
            for (int i = 0; i < STEPS; ++i) {
                if (!at.any(i)) continue;
                float* mw = share + at.at(i);
                float* mb = share + 2 * STEPS * CHUNK + at.at(i);
                if (k > 0) {
#pragma unroll
                    for (int j = 0; j < E; ++j) {
                        dw[i][j] += mw[j];
                        db[i][j] += mb[j];
                    }
                }
                if (k < slots - 1) {
#pragma unroll
                    for (int j = 0; j < E; ++j) {
                        mw[j] = dw[i][j];
                        mb[j] = db[i][j];
                    }
                } else {
                    float* to = b.workspace + 2 * (int64_t)blockIdx.x * p.dim;
                    at.store(to, i, dw[i]);
                    at.store(to + p.dim, i, db[i]);
                }
            }
        }
        if (slots > 1) __syncthreads();
    }
}

// Adds the blocks' sums: 64 columns of dweight, then of dbias, per block; its 8
// wavefronts take every eighth share and are added in their order.
__global__ void __launch_bounds__(512) norm_bwd_reduce(const cc1d_norm_bwd_params b, int64_t parts) {
    __shared__ float lds[8][64];
    const int64_t dim = b.fwd.dim, i = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    const int wave = threadIdx.x >> 6;
    float sum = 0.0f;
    if (i < 2 * dim) {
#pragma unroll 8
        for (int64_t k = wave; k < parts; k += 8) sum += b.workspace[2 * k * dim + i];
    }
    lds[wave][threadIdx.x & 63] = sum;
    __syncthreads();
    if (wave != 0 || i >= 2 * dim) return;
    for (int w = 1; w < 8; ++w) sum += lds[w][threadIdx.x];
    if (i < dim) b.dweight[i] = sum;
    else if (b.dbias) b.dbias[i - dim] = sum;
}

// Lanes or wavefronts per row and their steps, by dim alone (a row's result
// does not depend on the rows beside it): 8 values a lane, up to 16 wavefronts,
// so that a row's way through the card is short and a lane holds few values,
// then more steps. Narrow rows share a block of 4 wavefronts.
struct NormPlan {
    int lpr, wpr, steps, waves;
    int slots() const { return 64 / lpr * waves / wpr; }  // rows of a block at a time
};
NormPlan norm_plan(int64_t dim) {
    int lpr = 8;
    while (lpr < 64 && lpr * E < dim) lpr *= 2;
    const int64_t chunks = ceil_div(dim, lpr * E);
    const int steps = (int)ceil_div(chunks, 16), wpr = (int)ceil_div(chunks, steps);
    return {lpr, wpr, steps, wpr <= 2 ? 4 : wpr};
}
// Shares of the parameter gradients: three blocks a CU (15 wavefronts at 2560
// columns; a fourth would not fit beside them and run alone at the end). With
// two, three and four a CU, kernel and reduction in a row of launches, us:
// 8192 x 2560 bf16 + fp32 74, 86, 92; 2048 x 8192 70, 79, 89; 4099 x 1533 fp32
// 35, 36, 39; 16384 x 1024 bf16 43, 38, 38; 32768 x 256 bf16 22, 22, 24.
constexpr int64_t kBwdBlocks = 768;

int64_t bwd_blocks(const cc1d_norm_params& p, const NormPlan& n) {
    const int64_t all = ceil_div(p.rows, n.slots());
    return all < kBwdBlocks ? all : kBwdBlocks;
}

template <typename F> int with_norm_types(const cc1d_norm_params& p, F&& f) {
    return with_dtype(p.dtype, [&](auto t) {
        return p.residual_dtype == p.dtype ? f(t, t) : f(t, float{});
    });
}
// g(steps, lanes per row, even): rows of 64 lanes or more have 1 .. 4 steps, narrower ones one
template <typename F> int with_plan(const cc1d_norm_params& p, const NormPlan& n, F&& g) {
    using std::integral_constant;
    const bool even = p.dim % E == 0 && p.weight_stride == 1 && (p.bias == nullptr || p.bias_stride == 1);
    auto f = [&](auto steps, auto lpr) { return with_flag(even, [&](auto e) { return g(steps, lpr, e); }); };
    if (n.lpr == 8) return f(integral_constant<int, 1>{}, integral_constant<int, 8>{});
    if (n.lpr == 16) return f(integral_constant<int, 1>{}, integral_constant<int, 16>{});
    if (n.lpr == 32) return f(integral_constant<int, 1>{}, integral_constant<int, 32>{});
    switch (n.steps) {
    case 1: return f(integral_constant<int, 1>{}, integral_constant<int, 64>{});
    case 2: return f(integral_constant<int, 2>{}, integral_constant<int, 64>{});
    case 3: return f(integral_constant<int, 3>{}, integral_constant<int, 64>{});
    default: return f(integral_constant<int, 4>{}, integral_constant<int, 64>{});
    }
}

}  // namespace

int64_t norm_bwd_workspace_floats(const cc1d_norm_bwd_params& b) {
    return 2 * bwd_blocks(b.fwd, norm_plan(b.fwd.dim)) * b.fwd.dim;
}

int launch_norm_fwd(const cc1d_norm_params& p, hipStream_t stream) {
    const NormPlan n = norm_plan(p.dim);
    // a turn for all rows, or as many of them as a launch has threads for
    const int64_t blocks = ceil_div(p.rows, n.slots()), most = UINT32_MAX / (64 * n.waves);
    const dim3 grid((unsigned)(blocks < most ? blocks : most)), block(64 * n.waves);
    return with_norm_types(p, [&](auto t, auto r) {
        return with_plan(p, n, [&](auto steps, auto lpr, auto even) {
            return launch(norm_fwd_kernel<decltype(t), decltype(r), decltype(steps)::value, decltype(lpr)::value,
                                          decltype(even)::value>, grid, block, stream, p, n.wpr);
        });
    });
}

int launch_norm_bwd(const cc1d_norm_bwd_params& b, hipStream_t stream) {
    const cc1d_norm_params& p = b.fwd;
    const NormPlan n = norm_plan(p.dim);
    const int64_t blocks = bwd_blocks(p, n);
    int st = CC1D_OK;
    if (p.rows > 0)
        st = with_norm_types(p, [&](auto t, auto r) {
            return with_plan(p, n, [&](auto steps, auto lpr, auto even) {
                return launch(norm_bwd_kernel<decltype(t), decltype(r), decltype(steps)::value, decltype(lpr)::value,
                                              decltype(even)::value>, dim3((unsigned)blocks), dim3(64 * n.waves), stream, b, n.wpr);
            });
        });
    if (st != CC1D_OK) return st;
    return launch(norm_bwd_reduce, dim3((unsigned)ceil_div(2 * p.dim, 64)), dim3(512), stream, b, p.rows > 0 ? blocks : 0);
}

}  // namespace cc1d
