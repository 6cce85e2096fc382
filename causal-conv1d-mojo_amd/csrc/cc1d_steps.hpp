// cc1d_steps.hpp -- K consecutive elements of a row per lane, for rows that
// start and end anywhere: what the scan and the norm kernels read and write.
#pragma once

#include "cc1d_device.hpp"

namespace cc1d {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// K consecutive positions of a row as they lie in memory.
template <typename T, int K> struct Raw {
    static constexpr int DW = K * (int)sizeof(T) / 4;  // dwords: 2 (four 16-bit positions), 4 or 8
    uint32_t w[DW];

    // NT: data that the call touches once
    template <bool NT = false> __device__ __forceinline__ void vector(const T* p) {
        if constexpr (DW == 2) {
            const u32x2 v = *reinterpret_cast<const typename AnyAddr<sizeof(T)>::v2*>(p);
            w[0] = v[0];
            w[1] = v[1];
        } else {
#pragma unroll
            for (int q = 0; q < DW / 4; ++q) {
                const u32x4 v = NT ? vload_any_nt(p + q * elems16<T>::value) : vload_any(p + q * elems16<T>::value);
#pragma unroll
                for (int i = 0; i < 4; ++i) w[4 * q + i] = v[i];
            }
        }
    }
    // Positions t .. t + K - 1 of a row of `size` >= K positions with unit
    // stride. Lanes that would read past the row read its last K positions
    // instead, for fix() to put in place.
    template <bool NT = false> __device__ __forceinline__ void load(const T* row, int t, int size) {
        vector<NT>(row + (t + K <= size ? t : size - K));
    }
    // After load(): positions from `end` on are 0.
    __device__ __forceinline__ void fix(int t, int end, int size) {
        shift(t + K <= size ? 0 : (t < size ? t + K - size : K));
        constexpr int PER = 4 / (int)sizeof(T);
#pragma unroll
        for (int i = 0; i < DW; ++i) {
            if constexpr (PER == 1) w[i] = t + i < end ? w[i] : 0u;
            else w[i] &= t + 2 * i + 1 < end ? ~0u : (t + 2 * i < end ? 0xffffu : 0u);
        }
    }
    // drops the first s positions (0 .. K), the others move up, zeros follow
    __device__ __forceinline__ void shift(int s) {
        constexpr int PER = 4 / (int)sizeof(T);
        if constexpr (PER == 2) {
            const bool odd = (s & 1) != 0;
#pragma unroll
            for (int i = 0; i < DW; ++i) {
                const uint32_t up = i + 1 < DW ? w[i + 1] : 0u;
                w[i] = odd ? (w[i] >> 16) | (up << 16) : w[i];
            }
        }
        const int d = s / PER;
#pragma unroll
        for (int b = 1; b <= DW; b *= 2) {
            const bool on = (d & b) != 0;
#pragma unroll
            for (int i = 0; i < DW; ++i) w[i] = on ? (i + b < DW ? w[i + b < DW ? i + b : 0] : 0u) : w[i];
        }
    }
    // One by one, any stride; positions from `end` on are 0. Not unrolled: the
    // vector forms are the ones to be fast, and share their registers with it.
    __device__ __forceinline__ void each(const T* row, int64_t stride, int t, int end) {
        constexpr int PER = 4 / (int)sizeof(T);
#pragma unroll 1
        for (int j = K - 1; j >= 0; --j) {
            uint32_t v = 0u;
            if (t + j < end) {
                if constexpr (PER == 1) v = __builtin_bit_cast(uint32_t, row[(t + j) * stride]);
                else v = row[(t + j) * stride].bits;
            }
#pragma unroll
            for (int i = DW - 1; i >= 0; --i) {
                const uint32_t low = i > 0 ? w[i > 0 ? i - 1 : 0] : 0u;
                if constexpr (PER == 1) w[i] = i > 0 ? low : v;
                else w[i] = (w[i] << 16) | (i > 0 ? low >> 16 : v);
            }
        }
    }
    __device__ __forceinline__ float get(int j) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
        else if constexpr (__is_same(T, bf16)) return (j & 1) ? __uint_as_float(w[j / 2] & 0xffff0000u) : __uint_as_float(w[j / 2] << 16);
        else return to_f32(f16{(uint16_t)((j & 1) ? w[j / 2] >> 16 : w[j / 2] & 0xffffu)});
    }
};
template <typename T, int K, bool NT = false>
__device__ __forceinline__ void store_steps(T* row, int64_t stride, int t, int end, const float (&v)[K]) {
    if (stride == 1 && t + K <= end) {
        if constexpr (sizeof(T) == 2 && K == 4) {
            *reinterpret_cast<typename AnyAddr<2>::v2*>(row + t) = u32x2{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
        } else {
            constexpr int E = elems16<T>::value;
#pragma unroll
            for (int q = 0; q < K / E; ++q) {
                if (NT) vstore_any_nt(row + t + q * E, vpack<T>(v + q * E));
                else *reinterpret_cast<typename AnyAddr<sizeof(T)>::v4*>(row + t + q * E) = vpack<T>(v + q * E);
            }
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < K; ++j)
        if (t + j < end) row[(t + j) * stride] = from_f32<T>(v[j]);
}

// Sum over aligned groups of LPC lanes (a power of two), to all of them.
template <int LPC> __device__ __forceinline__ float lanes_sum(float v) {
    if constexpr (LPC == 64) return wave_sum(v);
    if constexpr (LPC >= 2) v += dpp_f32<kDppQuadSwap1, 0xf>(v);
    if constexpr (LPC >= 4) v += dpp_f32<kDppQuadSwap2, 0xf>(v);
    if constexpr (LPC == 8) v += dpp_f32<0x141, 0xf>(v);  // row_half_mirror: the other four lanes
    if constexpr (LPC >= 16) {
        v += dpp_f32<kDppRowRor4, 0xf>(v);
        v += dpp_f32<kDppRowRor8, 0xf>(v);
    }
    if constexpr (LPC >= 32) v += __shfl_xor(v, 16);
    return v;
}

}  // namespace cc1d
