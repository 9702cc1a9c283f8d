// Attention to chosen blocks of keys: each item walks a list of blocks of its sequence, in tiles that start over at each
// or run on over them (blocks of a multiple of 16 keys that is none of 64; fp32: 8 and 32).
#include "attend_rows.h"

namespace rch {

namespace {

template <int DT, int NB>
void launch(const rch_attend& A, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(A.n_rows));
    if (A.tile_unit == A.block_tokens) hipLaunchKernelGGL((attend_rows_kernel<DT, NB, kList, RCH_CODES_NONE>), grid, dim3(256), 0, stream, A);
    else hipLaunchKernelGGL((attend_rows_kernel<DT, NB, kPack, RCH_CODES_NONE>), grid, dim3(256), 0, stream, A);
}

template <int DT>
void launch_dim(const rch_attend& A, hipStream_t stream) {
    if (A.head_dim <= 64) launch<DT, 2>(A, stream);
    else if (A.head_dim <= 96) launch<DT, 3>(A, stream);
    else if (A.head_dim <= 128) launch<DT, 4>(A, stream);
    else if (A.head_dim <= 192) launch<DT, 6>(A, stream);
    else launch<DT, 8>(A, stream);
}

}  // namespace

int launch_attend_lists(const rch_attend& A, int dtype, hipStream_t stream) {
    if (dtype == RCH_DT_F16) launch_dim<RCH_DT_F16>(A, stream);
    else if (dtype == RCH_DT_F32) launch_dim<RCH_DT_F32>(A, stream);
    else launch_dim<RCH_DT_BF16>(A, stream);
    return check_launch("rch_attend_run (lists)");
}

}  // namespace rch
