// Values in 8-bit codes: what a code stands for.
#pragma once

#include "common.h"

namespace rch {

typedef unsigned int u1 __attribute__((ext_vector_type(1)));

// The four codes of a word as numbers.
template <int FMT>
__device__ __forceinline__ f4 code_numbers(uint32_t word) {
    if constexpr (FMT == RCH_CODES_INT8) {
        return f4{static_cast<float>(static_cast<int8_t>(word)), static_cast<float>(static_cast<int8_t>(word >> 8)),
                  static_cast<float>(static_cast<int8_t>(word >> 16)), static_cast<float>(static_cast<int8_t>(word >> 24))};
    } else {
        const f2 low = __builtin_bit_cast(f2, __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(word), false));
        const f2 high = __builtin_bit_cast(f2, __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(word), true));
        return f4{low[0], low[1], high[0], high[1]};
    }
}

// One code's value, rounded to the cache's type.
template <int FMT, typename T>
__device__ __forceinline__ T code_value(uint8_t code, float scale) {
    return static_cast<T>(code_numbers<FMT>(code)[0] * scale);
}

}  // namespace rch
