// Attention to chosen blocks of keys: each item walks a list of blocks of its sequence, in tiles that start over at each.
#include "attend_rows.h"

namespace rch {

namespace {

template <int DT>
void launch_dim(const rch_attend& A, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(A.n_rows));
    if (A.head_dim <= 64) hipLaunchKernelGGL((attend_rows_kernel<DT, 2, kList, RCH_CODES_NONE>), grid, dim3(256), 0, stream, A);
    else if (A.head_dim <= 96) hipLaunchKernelGGL((attend_rows_kernel<DT, 3, kList, RCH_CODES_NONE>), grid, dim3(256), 0, stream, A);
    else if (A.head_dim <= 128) hipLaunchKernelGGL((attend_rows_kernel<DT, 4, kList, RCH_CODES_NONE>), grid, dim3(256), 0, stream, A);
    else if (A.head_dim <= 192) hipLaunchKernelGGL((attend_rows_kernel<DT, 6, kList, RCH_CODES_NONE>), grid, dim3(256), 0, stream, A);
    else hipLaunchKernelGGL((attend_rows_kernel<DT, 8, kList, RCH_CODES_NONE>), grid, dim3(256), 0, stream, A);
}

}  // namespace

int launch_attend_lists(const rch_attend& A, int dtype, hipStream_t stream) {
    if (dtype == RCH_DT_F16) launch_dim<RCH_DT_F16>(A, stream);
    else if (dtype == RCH_DT_F32) launch_dim<RCH_DT_F32>(A, stream);
    else launch_dim<RCH_DT_BF16>(A, stream);
    return check_launch("rch_attend_run (lists)");
}

}  // namespace rch
