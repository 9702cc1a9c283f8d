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
#include "attend_tile.h"

namespace rch {

namespace {

template <int DT, int NB, int MODE>
__global__ void __launch_bounds__(256, NB <= 2 ? 3 : NB <= 4 ? 2 : 1) attend_rows_kernel(const rch_attend A) {
    typedef RowTile<DT, NB, DT == RCH_DT_F32 ? 1 : 2> Tile;
    constexpr int KT = Tile::KT, ES = Tile::ES, kTileBytes = KT * Tile::RB;
    constexpr int kStageBytes = 2 * kTileBytes;
    __shared__ __attribute__((aligned(1024))) char lds[2 * kStageBytes];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const AttendItem I = attend_item(A, blockIdx.x);
    if (I.row_begin >= I.row_end) return;  // a plan's filling
    const QueryRow R = query_row(A, I, I.row_begin + 32 * wave + (lane & 31));
    const float scale = __int_as_float(static_cast<int>(A.scale_bits));
    Tile tile;
    tile.init(A, I, R, lane);
    const bool active = I.row_begin + 32 * wave < I.row_end;  // a wave without rows only fetches
    WaveRange range;
    range.init(R);

    KeyWalk<KT, MODE> walk;
    walk.begin(A, I, ES);
    Fetch<Tile, MODE> fetch;
    fetch.init(A, wave, lane);
    lds_char* const tiles = (lds_char*)lds;
    const uint32_t mine = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(tiles)) + wave * (kTileBytes / 4);

    // The tile on its way: its first key and keys; `walk` is the one after it.
    bool coming = false;
    int next_key = 0, next_keys = 0, at = kStageBytes, key = 0, keys = 0, first = 0, last = 0;
    uint64_t held = ~uint64_t{0};
    auto send = [&](int to) {
        coming = !walk.done();
        if (!coming) return;
        next_key = walk.base;
        next_keys = walk.count();
        fetch.issue(A, walk, mine + to, mine + to + kTileBytes);
        walk.next();
        fetch.look_up(walk);
    };
    fetch.look_up(walk);
    send(0);
    // Waits for the tile on its way, fetches another one, and tells whether the wave's rows see any of it.
    auto advance = [&]() {
        // The tile has landed in every wave's share, and no wave reads the other half any more.
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        key = next_key;
        keys = next_keys;
        const int other = at;
        at = kStageBytes - at;
        send(other);
        if constexpr (MODE != kPage) {
            if (A.holes) {
                const int id = page_entry(walk.table, min(key + lane, I.key_end - 1) / static_cast<int>(A.page_tokens));
                held = __ballot(id >= 0 && id < A.pages);
            }
        }
        return active && range.sees(key, keys);
    };
    auto masked = [&]() {
        first = R.first - key;
        last = min(R.last - key, keys);
        return range.masked(key, keys, KT) || held != ~uint64_t{0};
    };
    bool rare = false;
    while (coming) {
        if (!advance()) continue;
        const bool some = masked();
        if (some && Tile::any_infinite(tiles + at + kTileBytes, lane)) {
            rare = true;
            break;
        }
        tile.template step<false>(tiles + at, tiles + at + kTileBytes, scale, first, last, held, some, lane);
    }
    if (rare) {
        for (bool seen = true;; seen = advance()) {
            if (seen) {
                const bool some = masked();
                tile.template step<true>(tiles + at, tiles + at + kTileBytes, scale, first, last, held, some, lane);
            }
            if (!coming) break;
        }
    }

    if (!R.valid) return;
    const int h = lane >> 5, row = I.row_begin + 32 * wave + (lane & 31);
    const float sum = row_sum(tile.sum);
    const bool blank = sum == 0.0f && sees_any(A, I, R.first, R.last);
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
        if (h == 0) *gout<f2>(partial_stats(A, at)) = f2{part_reference(tile.reference.whole(scale), sum, blank), sum};
        return;
    }
    const float inverse = row_factor(sum, blank);
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
    if (h == 0 && A.lse_ptr) gout<float>(A.lse_ptr)[(I.q_row + R.token) * A.heads + R.head] = row_lse(tile.reference.whole(scale), sum);
}

template <int DT, int NB>
void launch(const rch_attend& A, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(A.n_rows));
    constexpr int kShareRows = RowTile<DT, NB, DT == RCH_DT_F32 ? 1 : 2>::KT / 4;
    if (A.tile_unit == A.page_tokens) hipLaunchKernelGGL((attend_rows_kernel<DT, NB, kPage>), grid, dim3(256), 0, stream, A);
    else if (A.page_tokens % kShareRows == 0) hipLaunchKernelGGL((attend_rows_kernel<DT, NB, kShare>), grid, dim3(256), 0, stream, A);
    else hipLaunchKernelGGL((attend_rows_kernel<DT, NB, kRow>), grid, dim3(256), 0, stream, A);
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
