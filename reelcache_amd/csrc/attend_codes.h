// Tiles of keys and values from pools in 8-bit codes.
//
// A wave fetches its quarter of a K and a V tile as codes a tile ahead, straight into a part of LDS that is its own, with
// the rows' scales in registers.  Once they are there it writes the values that they stand for, rounded to the cache's type,
// into the LDS tile where native pools' rows are fetched to (attend_tile.h): the arithmetic on it is the same, so attention
// over codes has the bits of attention over the values read back.  (Codes on their way in registers, 16 of them, spilled the
// queries, and each tile waited for their reloads and so for the next tile's loads: a chunk of 4680 queries x 32760 keys
// in e4m3 took 1177 us so.)
//
// Bound: the products and what stands beside them.  That chunk takes 1015-1090 us where native pools take 915-945 on the same
// cards: 7.9 vector instructions to a matrix instruction instead of 6.5, and 61 LDS instructions to a wave's tile instead of
// 49, as the waves write it.
#pragma once

#include "attend_tile.h"
#include "codes.h"

namespace rch {

template <int DT, typename Tile, int MODE, int FMT>
struct CodeFetch {
    typedef typename Tile::vec8 vec8;
    static constexpr int KT = Tile::KT, RB = Tile::RB, kLanes = RB / 32, kRows = 64 / kLanes, kShareRows = KT / 4;
    static constexpr int NI = kShareRows / kRows;  // loads of a wave's quarter of K, or of V
    static constexpr int kWaveBytes = 2 * NI * 1024;
    float k_scale[NI], v_scale[NI];
    // Tiles whose shares are found one by one: a wave's rows lie in one page, and so do those of a page's or block's tile.
    static constexpr bool kShares = MODE == kShare || MODE == kPack;
    int share, row0, piece, pieces;  // the share's first row, the lane's first one, its 16 channels, such pieces of a head
    uint32_t k_at[MODE == kRow ? 1 : NI], v_at[MODE == kRow ? 1 : NI];  // byte offsets in a tile of one page
    uint32_t size, magic, dim, k_row, v_row;
    int64_t ks_head, vs_head, ks_page, vs_page;  // scales of the item's head in page 0; bytes of a page
    int ids[MODE == kRow ? NI : 1];
    int count;  // rows of the tile (or share) on its way

    __device__ __forceinline__ void init(const rch_attend& A, const AttendItem& I, int wave, int lane) {
        pieces = static_cast<int>(A.head_dim) / 16;
        share = wave * kShareRows;
        row0 = share + lane / kLanes;
        piece = lane % kLanes;
        k_row = static_cast<uint32_t>(A.k_token_stride);
        v_row = static_cast<uint32_t>(A.v_token_stride);
        ks_head = A.k_scale_ptr + 4 * I.kv_head * A.k_scale_head_stride;
        vs_head = A.v_scale_ptr + 4 * I.kv_head * A.v_scale_head_stride;
        ks_page = 4 * A.k_scale_page_stride;
        vs_page = 4 * A.v_scale_page_stride;
        size = static_cast<uint32_t>(A.page_tokens);
        magic = (65536u + size - 1) / size;  // x / size for x < 128, size <= 64
        dim = static_cast<uint32_t>(A.head_dim);
        if constexpr (MODE != kRow) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int row = row0 + i * kRows - (kShares ? share : 0);
                k_at[i] = piece < pieces ? row * k_row + piece * 16 : kOutOfRange;
                v_at[i] = piece < pieces ? row * v_row + piece * 16 : kOutOfRange;
            }
        }
    }
    __device__ __forceinline__ int page_of(uint32_t x) const {
        return size < 64 ? static_cast<int>((x * magic) >> 16) : (x >= size ? 1 : 0);
    }
    __device__ __forceinline__ void look_up(const KeyWalk<KT, MODE, true>& W) {
        if constexpr (MODE == kShare || MODE == kRow) {
            if (W.done()) return;
            const int keys = W.end - W.base, page0 = W.base / static_cast<int>(size);
            const int off0 = W.base - page0 * static_cast<int>(size);
            if constexpr (MODE == kShare) ids[0] = W.table[page0 + page_of(off0 + min(share, keys - 1))];
            else
#pragma unroll
            for (int i = 0; i < NI; ++i) ids[i] = page_entry(W.table, page0 + page_of(off0 + min(row0 + i * kRows, keys - 1)));
        }
    }

    // Sends the walk's tile on its way to the wave's LDS at `lds`.  Rows without a key have codes 0.
    __device__ __forceinline__ void issue(const rch_attend& A, const KeyWalk<KT, MODE, true>& W, uint32_t lds) {
        if constexpr (MODE != kRow) {
            int64_t k, v;
            int id, in_page;
            if constexpr (kShares) {
                if constexpr (MODE == kPack) {
                    W.own(id, in_page, count);
                } else {
                    const int x = W.base % static_cast<int>(size) + share;
                    in_page = x - page_of(x) * static_cast<int>(size);
                    id = ids[0];
                    count = id >= 0 && id < W.pages ? max(0, min(W.count() - share, kShareRows)) : 0;
                }
                if (count == 0) id = in_page = 0;  // nothing is in its range
                k = W.k_head + id * W.k_page + in_page * static_cast<int64_t>(k_row);
                v = W.v_head + id * W.v_page + in_page * static_cast<int64_t>(v_row);
            } else {
                id = W.id, in_page = W.in_page, k = W.k, v = W.v;
                count = W.count();
            }
            const u4 kr = tile_rsrc(k, count > 0 ? (count - 1) * k_row + dim : 0), vr = tile_rsrc(v, count > 0 ? (count - 1) * v_row + dim : 0);
            const int64_t ks = ks_head + id * ks_page + 4 * static_cast<int64_t>(in_page), vs = vs_head + id * vs_page + 4 * static_cast<int64_t>(in_page);
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                fetch_buffer(kr, k_at[i], lds + i * 1024);
                fetch_buffer(vr, v_at[i], lds + (NI + i) * 1024);
            }
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int row = max(0, min(row0 + i * kRows - (kShares ? share : 0), count - 1));
                k_scale[i] = gin<float>(ks)[row];
                v_scale[i] = gin<float>(vs)[row];
            }
        } else {
            count = W.count();
            const int off0 = W.base % static_cast<int>(size);
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int row = row0 + i * kRows, x = off0 + row, in_page = x - page_of(x) * static_cast<int>(size);
                const int id = row < count ? ids[i] : -1;
                const bool held = id >= 0 && id < W.pages, in = held && piece < pieces;
                const int64_t page = held ? id : 0;
                const int64_t ka = W.k_head + page * W.k_page + in_page * static_cast<int64_t>(k_row) + piece * 16;
                const int64_t va = W.v_head + page * W.v_page + in_page * static_cast<int64_t>(v_row) + piece * 16;
                fetch_global(in ? ka : A.plan_ptr, lds + i * 1024);  // or zeros
                fetch_global(in ? va : A.plan_ptr, lds + (NI + i) * 1024);
                k_scale[i] = *gin<float>(held ? ks_head + page * ks_page + 4 * static_cast<int64_t>(in_page) : A.plan_ptr);
                v_scale[i] = *gin<float>(held ? vs_head + page * vs_page + 4 * static_cast<int64_t>(in_page) : A.plan_ptr);
            }
        }
    }

    // 16 codes' values: two pieces of eight, at `place` and `apart` from there.
    static __device__ __forceinline__ void put(lds_char* row, int place, int apart, u4 codes, float scale) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
            *reinterpret_cast<__attribute__((address_space(3))) vec8*>(row + (half ? place ^ apart : place) * 16) =
                code_values<DT, FMT>(codes[2 * half], codes[2 * half + 1], scale);
    }
    // Writes the values of the codes that have landed at `raw`.
    __device__ __forceinline__ void commit(const lds_char* raw, lds_char* k_tile, lds_char* v_tile, int lane) const {
        typedef __attribute__((address_space(3))) const u4 lds_u4;
        u4 k[NI], v[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            k[i] = *(lds_u4*)(raw + i * 1024 + lane * 16);
            v[i] = *(lds_u4*)(raw + (NI + i) * 1024 + lane * 16);
        }
        __builtin_amdgcn_sched_barrier(0);  // all on their way before one is waited for
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int row = row0 + i * kRows;
            // (codes behind the last row are 0, their scales another row's)
            const bool none = MODE != kRow && row - (kShares ? share : 0) >= count;
            put(k_tile + row * RB, Tile::k_place(2 * piece) ^ Tile::k_swizzle(row), Tile::k_place(1), k[i], none ? 0.0f : k_scale[i]);
            put(v_tile + row * RB, Tile::v_place(2 * piece) ^ Tile::v_swizzle(row), Tile::v_place(1), v[i], none ? 0.0f : v_scale[i]);
        }
    }
};

}  // namespace rch
