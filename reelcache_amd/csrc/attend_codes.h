// Tiles of keys and values from pools in 8-bit codes.
//
// A wave loads its quarter of a K and a V tile a tile ahead, 16 codes and a row's scale to a lane, into registers, and
// writes the values that they stand for, rounded to the cache's type, into the LDS tile where native pools' rows are
// fetched to (attend_tile.h): the arithmetic on it is the same, so attention over codes has the bits of attention over
// the values read back.
#pragma once

#include "attend_tile.h"
#include "codes.h"

namespace rch {

template <int DT, typename Tile, int MODE, int FMT>
struct CodeFetch {
    typedef typename Tile::vec8 vec8;
    static constexpr int KT = Tile::KT, RB = Tile::RB, kLanes = RB / 32, kRows = 64 / kLanes, kShareRows = KT / 4;
    static constexpr int NI = kShareRows / kRows;
    u4 k[NI], v[NI];
    float k_scale[NI], v_scale[NI];
    int row0, piece, pieces;  // the lane's first row, its 16 channels, such pieces of a head
    uint32_t size, magic, k_row, v_row;
    int64_t ks_head, vs_head, ks_page, vs_page;  // scales of the item's head in page 0; bytes of a page
    int ids[MODE == kRow ? NI : 1];

    __device__ __forceinline__ void init(const rch_attend& A, const AttendItem& I, int wave, int lane) {
        pieces = static_cast<int>(A.head_dim) / 16;
        row0 = wave * kShareRows + lane / kLanes;
        piece = lane % kLanes;
        k_row = static_cast<uint32_t>(A.k_token_stride);
        v_row = static_cast<uint32_t>(A.v_token_stride);
        ks_head = A.k_scale_ptr + 4 * I.kv_head * A.k_scale_head_stride;
        vs_head = A.v_scale_ptr + 4 * I.kv_head * A.v_scale_head_stride;
        ks_page = 4 * A.k_scale_page_stride;
        vs_page = 4 * A.v_scale_page_stride;
        size = static_cast<uint32_t>(A.page_tokens);
        magic = (65536u + size - 1) / size;  // x / size for x < 128, size <= 64
    }
    __device__ __forceinline__ int page_of(uint32_t x) const {
        return size < 64 ? static_cast<int>((x * magic) >> 16) : (x >= size ? 1 : 0);
    }
    __device__ __forceinline__ void look_up(const KeyWalk<KT, MODE, true>& W) {
        if constexpr (MODE == kRow) {
            if (W.done()) return;
            const int keys = W.end - W.base, page0 = W.base / static_cast<int>(size);
            const int off0 = W.base - page0 * static_cast<int>(size);
#pragma unroll
            for (int i = 0; i < NI; ++i) ids[i] = page_entry(W.table, page0 + page_of(off0 + min(row0 + i * kRows, keys - 1)));
        }
    }
    static __device__ __forceinline__ __amdgpu_buffer_rsrc_t uniform(int64_t base, uint32_t bytes) {
        const uint32_t low = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(base));
        const uint32_t high = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(base >> 32));
        return make_rsrc(static_cast<int64_t>(static_cast<uint64_t>(high) << 32 | low), __builtin_amdgcn_readfirstlane(bytes));
    }

    // The walk's tile on its way into registers.  Rows without a key have code and scale 0.
    __device__ __forceinline__ void load(const rch_attend& A, const KeyWalk<KT, MODE, true>& W) {
        if constexpr (MODE != kRow) {
            const int rows = W.count();
            const uint32_t dim = static_cast<uint32_t>(A.head_dim), last = static_cast<uint32_t>(rows - 1);
            const auto kr = uniform(W.k, last * k_row + dim), vr = uniform(W.v, last * v_row + dim);
            const auto ksr = uniform(ks_head + W.id * ks_page + 4 * static_cast<int64_t>(W.in_page), 4 * rows);
            const auto vsr = uniform(vs_head + W.id * vs_page + 4 * static_cast<int64_t>(W.in_page), 4 * rows);
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int row = row0 + i * kRows;
                const bool in = piece < pieces && row < rows;
                k[i] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(kr, in ? row * k_row + piece * 16 : kOutOfRange, 0, 0));
                v[i] = __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(vr, in ? row * v_row + piece * 16 : kOutOfRange, 0, 0));
                k_scale[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(ksr, row < rows ? 4 * row : kOutOfRange, 0, 0));
                v_scale[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(vsr, row < rows ? 4 * row : kOutOfRange, 0, 0));
            }
        } else {
            const int keys = W.end - W.base, off0 = W.base % static_cast<int>(size);
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int row = row0 + i * kRows, x = off0 + row, in_page = x - page_of(x) * static_cast<int>(size);
                const int id = row < keys ? ids[i] : -1;
                const bool held = id >= 0 && id < W.pages, in = held && piece < pieces;
                const int64_t page = held ? id : 0;
                const int64_t ka = W.k_head + page * W.k_page + in_page * static_cast<int64_t>(k_row) + piece * 16;
                const int64_t va = W.v_head + page * W.v_page + in_page * static_cast<int64_t>(v_row) + piece * 16;
                k[i] = *gin<u4>(in ? ka : A.plan_ptr);
                v[i] = *gin<u4>(in ? va : A.plan_ptr);
                k_scale[i] = *gin<float>(held ? ks_head + page * ks_page + 4 * static_cast<int64_t>(in_page) : A.plan_ptr);
                v_scale[i] = *gin<float>(held ? vs_head + page * vs_page + 4 * static_cast<int64_t>(in_page) : A.plan_ptr);
            }
        }
    }

    // 16 codes' values: two pieces of eight.
    static __device__ __forceinline__ void put(lds_char* row, int first, int swizzle, u4 codes, float scale) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
            *reinterpret_cast<__attribute__((address_space(3))) vec8*>(row + ((first + half) ^ swizzle) * 16) =
                code_values<DT, FMT>(codes[2 * half], codes[2 * half + 1], scale);
    }
    __device__ __forceinline__ void commit(lds_char* k_tile, lds_char* v_tile) const {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int row = row0 + i * kRows;
            put(k_tile + row * RB, 2 * piece, Tile::k_swizzle(row), k[i], k_scale[i]);
            put(v_tile + row * RB, 2 * piece, Tile::v_swizzle(row), v[i], v_scale[i]);
        }
    }
};

}  // namespace rch
