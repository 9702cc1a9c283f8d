// Attention to chosen blocks of keys: each item walks a list of blocks of its sequence, in tiles that start over at each
// or run on over them (blocks of a multiple of 16 keys that is none of 64; fp32: 8 and 32).
//
// Bound: a chunk of 39 runs of 120 queries over 26 of 273 blocks of 120 (12 heads of 128) takes 130-142 us, 600 TFLOP/s: 468
// row blocks on 512 places, tiles of 64 and 56 keys, and runs that choose apart read 431 MB past the L2 for 201 MB of pools.
// Single tokens over 31 blocks of 64: 11.8 us, latency.  Blocks of 32 over int8 pages (prompts of up to 1500 queries, heads of
// 80): 56 us in tiles that run on; choice, attention and join take 75 us so and 99 in tiles that start over, half empty, at each.
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
