// What the attention kernels share: items of a plan, the mask, element types, partial results.
#pragma once

#include "common.h"

namespace rch {

// One item of a plan (rch_attend in reelcache_hip.h).
struct AttendItem {
    int table, length, q_row, queries, row_begin, row_end, kv_head, key_begin, key_end, part;
};

__device__ __forceinline__ AttendItem attend_item(const rch_attend& A, int index) {
    const RCH_GLOBAL int32_t* w = gin<int32_t>(A.plan_ptr) + A.items + static_cast<int64_t>(index) * RCH_ATTEND_ITEM;
    return {w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7], w[8], w[9]};
}

// Keys [first, last) that query token i of a sequence sees (apart from holes).
__device__ __forceinline__ void attend_range(const rch_attend& A, const AttendItem& I, int token, int& first, int& last) {
    const int place = I.length - I.queries + token;
    first = 0;
    last = I.length;
    if (A.block) {
        const int block = static_cast<int>(A.block);
        // floor((place) / block): a place before the first key has no block.
        const int64_t end = place < 0 ? 0 : (static_cast<int64_t>(place / block) + 1) * block;
        last = end < last ? static_cast<int>(end) : last;
    }
    if (A.window) {
        const int64_t begin = static_cast<int64_t>(place) - A.window + 1;
        first = begin > 0 ? (begin < I.length ? static_cast<int>(begin) : I.length) : 0;
    }
}

template <int DT>
struct AttendType;
template <>
struct AttendType<RCH_DT_F32> {
    typedef float type;
};
template <>
struct AttendType<RCH_DT_F16> {
    typedef _Float16 type;
};
template <>
struct AttendType<RCH_DT_BF16> {
    typedef __bf16 type;
};

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }

// A reference exponent that no score lies below (the lowest fp32): a row that has seen nothing keeps it, and its sum
// stays 0.
constexpr float kNoReference = -3.402823466e38f;
constexpr float kLn2 = 0.693147180559945309f;

__device__ __forceinline__ float row_lse(float reference, float sum) {
    return sum == 0.0f ? -INFINITY : __fmul_rn(reference + __builtin_amdgcn_logf(sum), kLn2);
}

// What a row's weighted sums are multiplied by.  Without a weight: 0 where the row sees no key; where it sees some
// (blank), every score is -inf, and the quotient has no value.
__device__ __forceinline__ float row_factor(float sum, bool blank) {
    return sum != 0.0f ? 1.0f / sum : blank ? __builtin_nanf("") : 0.0f;
}
// The reference that a part without a weight leaves: kNoReference, or -inf where it is blank.
__device__ __forceinline__ float part_reference(float reference, float sum, bool blank) {
    return sum == 0.0f && blank ? -INFINITY : reference;
}
__device__ __forceinline__ bool part_blank(float reference, float sum) { return sum == 0.0f && reference == -INFINITY; }

// Whether a row sees a key of an item's (for rows without a weight).
__device__ __forceinline__ bool sees_any(const rch_attend& A, const AttendItem& I, int first, int last) {
    first = first > I.key_begin ? first : I.key_begin;
    last = last < I.key_end ? last : I.key_end;
    if (first >= last || !A.holes) return first < last;
    const int size = static_cast<int>(A.page_tokens);
    const RCH_GLOBAL int32_t* table = gin<int32_t>(A.plan_ptr) + I.table;
    for (int page = first / size; page <= (last - 1) / size; ++page)
        if (table[page] >= 0 && table[page] < A.pages) return true;
    return false;
}

__device__ __forceinline__ int64_t partial_sums(const rch_attend& A, int64_t row) {
    return A.partial_ptr + row * A.head_dim * 4;
}
__device__ __forceinline__ int64_t partial_stats(const rch_attend& A, int64_t row) {
    return A.partial_ptr + (A.partial_rows * A.head_dim + 1) / 2 * 8 + row * 8;
}

// Launches the items of the tiled form.
int launch_attend_rows(const rch_attend& A, int dtype, hipStream_t stream);

}  // namespace rch
