// Attention of many query rows: 128 rows (tokens x heads of a key head) to a workgroup of four waves,
// each over all keys of the item.
//
// Bound: the matrix cores (4 * D operations for every row and key) with the exponentials beside them.
// A tile of 64 (fp32: 32) keys and values is fetched into one half of LDS while the waves work on the other half;
// one barrier to a tile.  Two workgroups fit a CU, so one's products cover the other's softmax.
#include "attend_tile.h"

namespace rch {

namespace {

template <int DT, int NB, bool PAGED>
__global__ void __launch_bounds__(256, 2) attend_rows_kernel(const rch_attend A, int first_item) {
    typedef RowTile<DT, NB, DT == RCH_DT_F32 ? 1 : 2> Tile;
    constexpr int RB = Tile::RB, KT = Tile::KT, ES = Tile::ES, kTileBytes = KT * RB, NI = kTileBytes / 1024 / 4;
    __shared__ __attribute__((aligned(1024))) char lds[4 * kTileBytes];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const AttendItem I = attend_item(A, first_item + blockIdx.x);
    const QueryRow R = query_row(A, I, I.row_begin + 32 * wave + (lane & 31));
    const float scale = __int_as_float(static_cast<int>(A.scale_bits));
    Tile tile;
    tile.init(A, I, R, lane);

    KeyWalk<KT, PAGED> walk;
    walk.table = (const const_int*)(uintptr_t)(A.plan_ptr + 4 * static_cast<int64_t>(I.table));
    walk.unit = static_cast<int>(A.tile_unit);
    walk.end = I.key_end;
    walk.pages = static_cast<int>(A.pages);
    walk.begin(I.key_begin);
    Fetch<Tile, NI, PAGED> fetch;
    fetch.init(A, wave * NI, lane);
    const int64_t k_head = A.k_ptr + ES * I.kv_head * A.k_head_stride, v_head = A.v_ptr + ES * I.kv_head * A.v_head_stride;
    lds_char* const tiles = (lds_char*)lds;
    const uint32_t lds_base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(tiles)) + wave * NI * 1024;

    if (!walk.done()) fetch.issue(A, walk, k_head, v_head, lds_base, lds_base + kTileBytes);
    int stage = 2 * kTileBytes, first = 0, last = 0;
    uint64_t held = ~uint64_t{0};
    // Waits for the next tile, fetches the one after it, and finds what the wave's rows see of it.
    auto advance = [&]() {
        const int base = walk.base(), count = walk.count();
        walk.next();
        const int other = stage;
        stage = 2 * kTileBytes - stage;
        // The tile has landed in every wave's share, and no wave reads the other half any more.
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (!walk.done()) fetch.issue(A, walk, k_head, v_head, lds_base + other, lds_base + other + kTileBytes);
        first = R.first - base;
        last = min(R.last - base, count);
        if constexpr (!PAGED) {
            if (A.holes) {
                const int key = min(base + lane, I.key_end - 1);
                const int id = page_entry(walk.table, key / static_cast<int>(A.page_tokens));
                held = __ballot(id >= 0 && id < A.pages);
            }
        }
        return __any(first < KT && last > 0 && last > first);
    };
    auto masked = [&]() { return __any(first > 0 || last < KT) || held != ~uint64_t{0}; };
    bool rare = false;
    while (!walk.done()) {
        if (!advance()) continue;
        const bool some = masked();
        if (some && Tile::any_infinite(tiles + stage + kTileBytes, lane)) {
            rare = true;
            break;
        }
        tile.template step<false>(tiles + stage, tiles + stage + kTileBytes, scale, first, last, held, some, lane);
    }
    if (rare) {
        for (bool seen = true;; seen = advance()) {
            if (seen)
                tile.template step<true>(tiles + stage, tiles + stage + kTileBytes, scale, first, last, held, masked(), lane);
            if (walk.done()) break;
        }
    }

    if (!R.valid) return;
    const int h = lane >> 5, row = I.row_begin + 32 * wave + (lane & 31);
    const float sum = row_sum(tile.sum);
    if (I.part >= 0) {
        const int64_t at = I.part + row - I.row_begin;
        const int64_t to = partial_sums(A, at);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int d = Tile::channel_of(b, i, h);
                if (d < A.head_dim) *gout<f4>(to + 4 * d) = f4{tile.o[b][i], tile.o[b][i + 1], tile.o[b][i + 2], tile.o[b][i + 3]};
            }
        if (h == 0) *gout<f2>(partial_stats(A, at)) = f2{tile.reference, sum};
        return;
    }
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int64_t to = A.out_ptr + ES * ((I.q_row + R.token) * A.out_token_stride + R.head * A.out_head_stride);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int d = Tile::channel_of(b, i, h);
            if (d < A.head_dim)
                Tile::store4(to + ES * d, f4{tile.o[b][i] * inverse, tile.o[b][i + 1] * inverse, tile.o[b][i + 2] * inverse,
                                             tile.o[b][i + 3] * inverse});
        }
    if (h == 0 && A.lse_ptr) gout<float>(A.lse_ptr)[(I.q_row + R.token) * A.heads + R.head] = row_lse(tile.reference, sum);
}

template <int DT, int NB>
void launch(const rch_attend& A, int first, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(A.n_rows));
    if (A.tile_unit == A.page_tokens) hipLaunchKernelGGL((attend_rows_kernel<DT, NB, true>), grid, dim3(256), 0, stream, A, first);
    else hipLaunchKernelGGL((attend_rows_kernel<DT, NB, false>), grid, dim3(256), 0, stream, A, first);
}

template <int DT>
void launch_dim(const rch_attend& A, int first, hipStream_t stream) {
    if (A.head_dim <= 64) launch<DT, 2>(A, first, stream);
    else if (A.head_dim <= 96) launch<DT, 3>(A, first, stream);
    else launch<DT, 4>(A, first, stream);
}

}  // namespace

int launch_attend_rows(const rch_attend& A, int dtype, int first, hipStream_t stream) {
    if (dtype == RCH_DT_F16) launch_dim<RCH_DT_F16>(A, first, stream);
    else if (dtype == RCH_DT_F32) launch_dim<RCH_DT_F32>(A, first, stream);
    else launch_dim<RCH_DT_BF16>(A, first, stream);
    return check_launch("rch_attend_run (rows)");
}

}  // namespace rch
