// The kernel of the attention on the matrix cores: 128 query rows (tokens x heads of a key head) to a workgroup of four
// waves, each over all keys of the item.  What bounds it and what it measured stands with its instances.
#pragma once

#include "attend_codes.h"

namespace rch {

// FMT: what the pools hold (RCH_CODES_*).
template <int DT, int NB, int MODE, int FMT>
__global__ void __launch_bounds__(256, NB <= 2 ? 3 : NB <= 4 ? 2 : 1) attend_rows_kernel(const rch_attend A) {
    constexpr bool kCodes = FMT != RCH_CODES_NONE;
    typedef RowTile<DT, NB, DT == RCH_DT_F32 ? 1 : 2, kCodes && NB != 3 && NB != 6, kCodes> Tile;
    constexpr int KT = Tile::KT, ES = Tile::ES, kTileBytes = KT * Tile::RB;
    constexpr int kStageBytes = 2 * kTileBytes;
    typedef typename std::conditional_t<kCodes, std::common_type<CodeFetch<DT == RCH_DT_F32 ? RCH_DT_BF16 : DT, Tile, MODE, kCodes ? FMT : RCH_CODES_INT8>>,
                                        std::common_type<Fetch<Tile, MODE>>>::type Fetcher;
    __shared__ __attribute__((aligned(1024))) char lds[2 * kStageBytes + (kCodes ? 4 * kTileBytes / 4 : 0)];  // codes: half as many bytes
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

    if constexpr (kCodes) wait_vector_memory();  // the queries, so that no tile's wait is for them
    KeyWalk<KT, MODE, kCodes> walk;
    if constexpr (MODE == kPack) walk.wave = wave;
    walk.begin(A, I, kCodes ? 1 : ES);
    Fetcher fetch;
    if constexpr (kCodes) fetch.init(A, I, wave, lane);
    else fetch.init(A, wave, lane);
    lds_char* const tiles = (lds_char*)lds;
    const uint32_t mine = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(tiles)) + wave * (kTileBytes / 4);

    lds_char* const codes = tiles + 2 * kStageBytes + wave * (kTileBytes / 4);
    const uint32_t own_codes = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(codes));

    // The tile on its way: its first key and keys; `walk` is the one after it.
    bool coming = false;
    int next_key = 0, next_keys = 0, at = kStageBytes, key = 0, keys = 0, first = 0, last = 0;
    uint64_t held = ~uint64_t{0};
    int next_shares[4], shares[4];  // kPack: first keys of the tiles' shares
    ShareView<KT / 4> view;
    auto send = [&](int to) {
        coming = !walk.done();
        if (!coming) return;
        if constexpr (MODE == kPack) {
#pragma unroll
            for (int s = 0; s < 4; ++s) next_shares[s] = walk.first_key(s);
        } else {
            next_key = walk.base;
            next_keys = walk.count();
        }
        if constexpr (kCodes) fetch.issue(A, walk, own_codes);
        else fetch.issue(A, walk, mine + to, mine + to + kTileBytes);
        walk.next();
        fetch.look_up(walk);
    };
    fetch.look_up(walk);
    send(0);
    auto copy_shares = [&]() {
        if constexpr (MODE == kPack)
#pragma unroll
            for (int s = 0; s < 4; ++s) shares[s] = next_shares[s];
    };
    // Waits for the tile on its way, fetches another one, and tells whether the wave's rows see any of it.
    auto advance = [&]() {
        if constexpr (kCodes) {
            // The wave's codes have landed; their values go into the half that no wave reads since the last barrier, and the
            // next codes into their place.
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            at = kStageBytes - at;
            fetch.commit(codes, tiles + at, tiles + at + kTileBytes, lane);
            key = next_key;
            keys = next_keys;
            copy_shares();
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            send(0);
            asm volatile("s_barrier" ::: "memory");
        } else {
            // The tile has landed in every wave's share, and no wave reads the other half any more.
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            key = next_key;
            keys = next_keys;
            copy_shares();
            const int other = at;
            at = kStageBytes - at;
            send(other);
        }
        if constexpr (MODE == kPack) {
            view.look(walk, range, shares);
            return active && view.sees;
        }
        if constexpr (MODE == kShare || MODE == kRow) {
            if (A.holes) {
                const int id = page_entry(walk.table, min(key + lane, I.key_end - 1) / static_cast<int>(A.page_tokens));
                held = __ballot(id >= 0 && id < A.pages);
            }
        }
        return active && range.sees(key, keys);
    };
    auto masked = [&]() {
        if constexpr (MODE == kPack) {
            first = 0;
            last = KT;
            if (view.masked) held = ShareView<KT / 4>::bits(walk, shares, R.first, R.last);
            return view.masked;
        }
        first = R.first - key;
        last = min(R.last - key, keys);
        return range.masked(key, keys, KT) || held != ~uint64_t{0};
    };
    bool rare = false;
    while (coming) {
        if (!advance()) continue;
        const bool some = masked();
        // (Rows behind the last key, and those of a hole, are zeros: only keys that a row does not see may be anything.)
        if (some && (MODE == kPack ? view.hides : range.hides(key, keys)) && Tile::any_infinite(tiles + at + kTileBytes, lane)) {
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
    bool blank = false;
    if (sum == 0.0f) {
        const int unit = max(static_cast<int>(A.block_tokens), 1), per = (unit + KT - 1) / KT;
        if constexpr (MODE == kList) blank = sees_any_listed(A, I, R.first, R.last, I.key_begin / per, (I.key_end + per - 1) / per);
        else if constexpr (MODE == kPack) blank = sees_any_listed(A, I, R.first, R.last, I.key_begin * KT / unit, min(I.entries, (I.key_end * KT + unit - 1) / unit));
        else blank = sees_any(A, I, R.first, R.last);
    }
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

}  // namespace rch
