// Values in 8-bit codes: what a code stands for.
#pragma once

#include "common.h"

namespace rch {

// Types that codes stand for.
template <int DT>
struct Coded;
template <>
struct Coded<RCH_DT_F16> {
    typedef _Float16 type;
    typedef h8 vec8;
};
template <>
struct Coded<RCH_DT_BF16> {
    typedef __bf16 type;
    typedef bf8 vec8;
};

// The four codes of a word as numbers.
template <int FMT>
__device__ __forceinline__ f4 code_numbers(uint32_t word) {
    if constexpr (FMT == RCH_CODES_INT8) {
        const int w = static_cast<int>(word);
        return f4{static_cast<float>(w << 24 >> 24), static_cast<float>(w << 16 >> 24), static_cast<float>(w << 8 >> 24),
                  static_cast<float>(w >> 24)};
    } else {
        const f2 low = __builtin_bit_cast(f2, __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(word), false));
        const f2 high = __builtin_bit_cast(f2, __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(word), true));
        return f4{low[0], low[1], high[0], high[1]};
    }
}

// The scale that counts: of 8-bit floats its power of two.
template <int FMT>
__device__ __forceinline__ float code_scale(float scale) {
    if constexpr (FMT == RCH_CODES_INT8) return scale;
    const uint32_t bits = __float_as_uint(scale);
    return (bits & 0x7f800000u) == 0x7f800000u ? __builtin_nanf("") : __uint_as_float(bits & 0x7f800000u);
}

// What eight codes of one scale stand for: the fp32 product, rounded to the cache's type.  8-bit floats with a power of two
// are converted by one instruction for two (exact in bf16; half a step in fp16 where they are subnormal).
template <int DT, int FMT>
__device__ __forceinline__ typename Coded<DT>::vec8 code_values(uint32_t low, uint32_t high, float scale) {
    typedef typename Coded<DT>::type T;
    typename Coded<DT>::vec8 x;
    if constexpr (FMT == RCH_CODES_INT8) {
        const f4 a = code_numbers<FMT>(low), b = code_numbers<FMT>(high);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = static_cast<T>(a[i] * scale), x[4 + i] = static_cast<T>(b[i] * scale);
    } else {
        const int w[2] = {static_cast<int>(low), static_cast<int>(high)};
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (DT == RCH_DT_BF16) {
                const auto p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], scale, false), q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[i], scale, true);
                x[4 * i] = p[0], x[4 * i + 1] = p[1], x[4 * i + 2] = q[0], x[4 * i + 3] = q[1];
            } else {
                const auto p = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], scale, false), q = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w[i], scale, true);
                x[4 * i] = p[0], x[4 * i + 1] = p[1], x[4 * i + 2] = q[0], x[4 * i + 3] = q[1];
            }
        }
    }
    return x;
}
// The same of eight codes with a scale each.
template <int DT, int FMT>
__device__ __forceinline__ typename Coded<DT>::vec8 code_values(uint32_t low, uint32_t high, f4 scale_low, f4 scale_high) {
    typedef typename Coded<DT>::type T;
    typename Coded<DT>::vec8 x;
    const f4 a = code_numbers<FMT>(low), b = code_numbers<FMT>(high);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = static_cast<T>(a[i] * scale_low[i]), x[4 + i] = static_cast<T>(b[i] * scale_high[i]);
    return x;
}
// Eight codes as numbers (exact).
template <int DT, int FMT>
__device__ __forceinline__ typename Coded<DT>::vec8 code_values(uint32_t low, uint32_t high) {
    if constexpr (FMT == RCH_CODES_E4M3) {
        return code_values<DT, FMT>(low, high, 1.0f);
    } else {
        typedef typename Coded<DT>::type T;
        typename Coded<DT>::vec8 x;
        const f4 a = code_numbers<FMT>(low), b = code_numbers<FMT>(high);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = static_cast<T>(a[i]), x[4 + i] = static_cast<T>(b[i]);
        return x;
    }
}
template <int DT, int FMT>
__device__ __forceinline__ typename Coded<DT>::type code_value(uint8_t code, float scale) {
    return code_values<DT, FMT>(code, 0, scale)[0];
}

}  // namespace rch
