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

// The token's place on each axis.  (By value: an array that this wrote to stayed in scratch memory, and rotations of
// 4680 tokens and stores took 1 to 2 % more.)
struct TurningRows {
    int t, h, w;
};
template <typename Job>
__device__ __forceinline__ TurningRows turning_rows(const Job& J, int64_t batch, int64_t token) {
    if (J.rows_ptr) {
        const RCH_GLOBAL int32_t* r = gin<int32_t>(J.rows_ptr) + batch * J.rows_batch_stride + token * J.rows_token_stride;
        const int first = r[0], second = 1 < J.axes ? r[J.rows_axis_stride] : 0, third = 2 < J.axes ? r[2 * J.rows_axis_stride] : 0;
        return {first, second, third};
    }
    if (J.axes == 3) {
        const int t = static_cast<int>(token), plane = static_cast<int>(J.grid_h * J.grid_w), w = static_cast<int>(J.grid_w);
        const int f = t / plane, y = (t - f * plane) / w;
        return {static_cast<int>(J.row_t) + f, static_cast<int>(J.row_h) + y, static_cast<int>(J.row_w) + t - f * plane - y * w};
    }
    return {static_cast<int>(J.row_t + token), 0, 0};
}

// (cos, sin) of pair j; a row outside its axis turns to NaN (nothing is read there).
template <typename Job>
__device__ __forceinline__ f2 turning_angle(const Job& J, const TurningRows& row, int j, int pairs) {
    const int bound1 = static_cast<int>(J.sec_t), bound2 = bound1 + static_cast<int>(J.sec_h);
    const int axis = J.axes == 1 ? 0 : (j < bound1 ? 0 : (j < bound2 ? 1 : 2));
    const int r = axis == 0 ? row.t : (axis == 1 ? row.h : row.w);
    const int64_t limit = axis == 0 ? J.limit_t : (axis == 1 ? J.limit_h : J.limit_w);
    f2 pair = {__builtin_nanf(""), __builtin_nanf("")};
    if (r >= 0 && r < limit) pair = gin<f2>(J.pairs_ptr)[static_cast<int64_t>(r) * pairs + j];
    return pair;
}

}  // namespace rch
