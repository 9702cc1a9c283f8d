// Attention of many query rows: 128 rows (tokens x heads of a key head) to a workgroup of four waves,
// each over all keys of the item.
//
// Bound: the matrix cores (4 * D operations for every row and key) with the exponentials beside them.
// A tile of 64 (fp32: 32) keys and values is fetched into one half of LDS while the waves work on the other half;
// one barrier to a tile.  Two workgroups (heads of up to 64 channels: three, of more than 128: one) fill a CU's
// registers and LDS, so one's products cover the other's softmax.  bf16, a chunk's 4680 queries x 32760 keys, 12
// heads of 128: 931 us, 1012 TFLOP/s, the matrix cores busy 48 % of the time at the 2.0 GHz that the power limit
// leaves (2.2 GHz with less even work).  Without the fetches it would take 927 of then 1013 us, without the LDS
// reads 930, without the softmax 855.  Long single tokens (652 MB of keys and values) take 122 us, 5.4 TB/s.
// Other shapes measured on the chunk: 256 rows in 8 waves with three stages 1095 against 938 us; 64 rows to a wave
// 1404 against 949; four stages 220 against 175 us (2340 queries x 9360 keys).  For 24 heads of 64, 4680 x 20000:
// three workgroups to a CU 640 us, two 730, four (128 registers, spilled) 844.
// Heads of 256 reach 552 TFLOP/s (one workgroup: softmax and products in turn), of 192 638; fp32 120 to 133 (64 and
// 128 channels) of the 153 that a large product reaches, of 256 85 (spilled).
#include "attend_rows.h"

namespace rch {

namespace {

template <int DT, int NB>
void launch(const rch_attend& A, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(A.n_rows));
    constexpr int kShareRows = RowTile<DT, NB, DT == RCH_DT_F32 ? 1 : 2>::KT / 4;
    if (A.tile_unit == A.page_tokens) hipLaunchKernelGGL((attend_rows_kernel<DT, NB, kPage, RCH_CODES_NONE>), grid, dim3(256), 0, stream, A);
    else if (A.page_tokens % kShareRows == 0) hipLaunchKernelGGL((attend_rows_kernel<DT, NB, kShare, RCH_CODES_NONE>), grid, dim3(256), 0, stream, A);
    else hipLaunchKernelGGL((attend_rows_kernel<DT, NB, kRow, RCH_CODES_NONE>), grid, dim3(256), 0, stream, A);
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

int launch_attend_rows(const rch_attend& A, int dtype, hipStream_t stream) {
    if (dtype == RCH_DT_F16) launch_dim<RCH_DT_F16>(A, stream);
    else if (dtype == RCH_DT_F32) launch_dim<RCH_DT_F32>(A, stream);
    else launch_dim<RCH_DT_BF16>(A, stream);
    return check_launch("rch_attend_run (rows)");
}

}  // namespace rch
