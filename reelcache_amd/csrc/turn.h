// Where tokens stand and how their pairs turn (rch_rotary_job and rch_codes have the same place fields).
#pragma once

#include "common.h"

namespace rch {

// The products are rounded apart (no FMA), as in the restore kernels.
__device__ __forceinline__ void rotate_pair(float& e, float& o, float c, float s) {
    const float re = __fsub_rn(__fmul_rn(e, c), __fmul_rn(o, s));
    const float ro = __fadd_rn(__fmul_rn(e, s), __fmul_rn(o, c));
    e = re;
    o = ro;
}

// The token's place on each axis.
template <typename Job>
__device__ __forceinline__ void turning_rows(const Job& J, int64_t batch, int64_t token, int (&row)[3]) {
    if (J.rows_ptr) {
        const RCH_GLOBAL int32_t* r = gin<int32_t>(J.rows_ptr) + batch * J.rows_batch_stride + token * J.rows_token_stride;
#pragma unroll
        for (int a = 0; a < 3; ++a) row[a] = a < J.axes ? r[a * J.rows_axis_stride] : 0;
    } else if (J.axes == 3) {
        const int t = static_cast<int>(token), plane = static_cast<int>(J.grid_h * J.grid_w), w = static_cast<int>(J.grid_w);
        const int f = t / plane, y = (t - f * plane) / w;
        row[0] = static_cast<int>(J.row_t) + f;
        row[1] = static_cast<int>(J.row_h) + y;
        row[2] = static_cast<int>(J.row_w) + t - f * plane - y * w;
    } else {
        row[0] = static_cast<int>(J.row_t + token);
        row[1] = row[2] = 0;
    }
}

// (cos, sin) of pair j; a row outside its axis turns to NaN (nothing is read there).
template <typename Job>
__device__ __forceinline__ f2 turning_angle(const Job& J, const int (&row)[3], int j) {
    const int bound1 = static_cast<int>(J.sec_t), bound2 = bound1 + static_cast<int>(J.sec_h);
    const int axis = J.axes == 1 ? 0 : (j < bound1 ? 0 : (j < bound2 ? 1 : 2));
    const int r = axis == 0 ? row[0] : (axis == 1 ? row[1] : row[2]);
    const int64_t limit = axis == 0 ? J.limit_t : (axis == 1 ? J.limit_h : J.limit_w);
    f2 pair = {__builtin_nanf(""), __builtin_nanf("")};
    if (r >= 0 && r < limit) pair = gin<f2>(J.pairs_ptr)[static_cast<int64_t>(r) * static_cast<int>(J.pairs) + j];
    return pair;
}

}  // namespace rch
