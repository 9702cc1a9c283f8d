// The launches of the attention over pools in codes of one format (FMT).
#pragma once

#include "attend_rows.h"
#include "attend_single.h"

namespace rch {

template <int DT, int NB, int FMT>
void launch_codes(const rch_attend& A, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(A.n_rows));
    if (A.lists_ptr && A.tile_unit == A.block_tokens) hipLaunchKernelGGL((attend_rows_kernel<DT, NB, kList, FMT>), grid, dim3(256), 0, stream, A);
    else if (A.lists_ptr) hipLaunchKernelGGL((attend_rows_kernel<DT, NB, kPack, FMT>), grid, dim3(256), 0, stream, A);
    else if (A.tile_unit == A.page_tokens) hipLaunchKernelGGL((attend_rows_kernel<DT, NB, kPage, FMT>), grid, dim3(256), 0, stream, A);
    else if (A.page_tokens % 16 == 0) hipLaunchKernelGGL((attend_rows_kernel<DT, NB, kShare, FMT>), grid, dim3(256), 0, stream, A);
    else hipLaunchKernelGGL((attend_rows_kernel<DT, NB, kRow, FMT>), grid, dim3(256), 0, stream, A);
}

template <int DT, int FMT>
void launch_codes_dim(const rch_attend& A, hipStream_t stream) {
    if (A.head_dim <= 64) launch_codes<DT, 2, FMT>(A, stream);
    else if (A.head_dim <= 96) launch_codes<DT, 3, FMT>(A, stream);
    else if (A.head_dim <= 128) launch_codes<DT, 4, FMT>(A, stream);
    else if (A.head_dim <= 192) launch_codes<DT, 6, FMT>(A, stream);
    else launch_codes<DT, 8, FMT>(A, stream);
}

// Single tokens: heads of 96 and 192 channels take the tiles of 128 and 256.
template <int DT, int NB, int FMT>
void launch_single(const rch_attend& A, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(A.n_rows));
    if (A.lists_ptr) hipLaunchKernelGGL((attend_single_kernel<DT, NB, kList, FMT>), grid, dim3(64), 0, stream, A);
    else if (A.tile_unit == A.page_tokens) hipLaunchKernelGGL((attend_single_kernel<DT, NB, kPage, FMT>), grid, dim3(64), 0, stream, A);
    else hipLaunchKernelGGL((attend_single_kernel<DT, NB, kRow, FMT>), grid, dim3(64), 0, stream, A);
}

template <int DT, int FMT>
void launch_single_dim(const rch_attend& A, hipStream_t stream) {
    if (A.head_dim <= 64) launch_single<DT, 2, FMT>(A, stream);
    else if (A.head_dim <= 128) launch_single<DT, 4, FMT>(A, stream);
    else launch_single<DT, 8, FMT>(A, stream);
}

template <int FMT>
int launch_codes_rows(const rch_attend& A, int dtype, hipStream_t stream) {
    if (A.single) {
        if (dtype == RCH_DT_F16) launch_single_dim<RCH_DT_F16, FMT>(A, stream);
        else launch_single_dim<RCH_DT_BF16, FMT>(A, stream);
        return check_launch("rch_attend_run (single tokens of codes)");
    }
    if (dtype == RCH_DT_F16) launch_codes_dim<RCH_DT_F16, FMT>(A, stream);
    else launch_codes_dim<RCH_DT_BF16, FMT>(A, stream);
    return check_launch("rch_attend_run (codes)");
}

}  // namespace rch
