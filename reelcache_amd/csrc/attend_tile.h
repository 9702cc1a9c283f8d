// Tiles of keys and values for the attention on the matrix cores.
//
// A wave works on 32 query rows, as the columns of the products:
//   S^T [32 keys x 32 rows] = K [keys x D] Q^T    (v_mfma_f32_32x32x16: A = K from LDS, B = Q in registers)
//   O^T [32 channels x 32 rows] += V^T [channels x keys] P^T
// The lane of column n (lane % 32, half h = lane / 32) holds, of S^T, keys 8 (i / 4) + 4 h + i % 4 of its
// row n for i = 0..15.  A product's inner index may run over the keys in any order that both operands
// share, so registers 8 q .. 8 q + 7, rounded to 16 bits, are the B operand of keys 16 q .. 16 q + 15 as
// they are, and the A operand V^T takes the same order: two transposed LDS reads of four keys each.
// Everything a row's softmax needs lies in two lanes: maxima meet by one half-wave swap per tile, and
// the sums only at the end.
//
// K and V rows travel from memory to LDS directly (buffer / global loads to LDS), 16 bytes a lane; the
// lane order is the LDS order, so the bank swizzle is applied to the channel piece that a lane fetches:
// piece c of row r lies at piece c ^ (r % pieces) in K (rows are read 8 at a time at one c) and at
// c ^ 4 (r % 4) in V (rows are read 4 at a time, 64 bytes of each).
#pragma once

#include <type_traits>

#include "attend.h"

namespace rch {

typedef __attribute__((address_space(3))) char lds_char;

template <int DT>
struct Half;
template <>
struct Half<RCH_DT_BF16> {
    typedef __bf16 type;
    typedef bf8 vec8;
    typedef __bf16 vec4 __attribute__((ext_vector_type(4)));
    // Weights are rounded to bf16 for the second product: relative 2**-8 each, averaged over the keys.
    static constexpr float kBias = 0.0f;
    static constexpr uint32_t kExponent = 0x7f80u;
    static __device__ __forceinline__ f16v mfma(vec8 a, vec8 b, f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};
template <>
struct Half<RCH_DT_F16> {
    typedef _Float16 type;
    typedef h8 vec8;
    typedef _Float16 vec4 __attribute__((ext_vector_type(4)));
    // fp16 weights carry a factor 2**7 (divided out with the sum): the largest is 2**15, and small ones stay
    // above the subnormals down to 2**-21.
    static constexpr float kBias = 7.0f;
    static constexpr uint32_t kExponent = 0x7c00u;
    static __device__ __forceinline__ f16v mfma(vec8 a, vec8 b, f16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};

// The running reference of a row's exponents moves when a score passes it by more than 2**kSlack: any
// reference gives the same quotient, and the sums are rarely multiplied.
constexpr float kSlack = 8.0f;

// A weight's exponent is the score times the scale less the reference, rounded once; the reference is such a product
// rounded by itself.  The two differ by the product's rounding: 2**-5 at most up to this size.  Farther out that
// rounding alone would be whole powers of two (32 at 2**30), so a row's scores are taken less their largest first (an
// exact difference for those that count): every tile of such a row takes the branch that moves references.
constexpr float kFarScore = 1048576.0f;

// What a row's exponents refer to: (score - shift) * scale - value.  The shift is 0 but for rows far out.
struct Reference {
    float value, shift, limit;  // limit: a largest score (scaled, less the bias) above it moves the reference

    __device__ __forceinline__ void init() {
        value = limit = kNoReference;
        shift = 0.0f;
    }
    // Moves it to a tile's largest score (top: scaled, less the bias), where that is larger.  Returns the factor of the
    // row's sums.
    template <typename Scores>
    __device__ __forceinline__ float move(float largest, float top, float scale, float bias, Scores& s) {
        float next = fmaxf(value, top), fade = exp2_of(value - next);
        limit = next + kSlack;
        const bool out = shift != 0.0f || (__builtin_fabsf(top) > kFarScore && top > value);
        if (__builtin_expect(__any(out), 0)) {
            const float to = shift != 0.0f ? fmaxf(shift, largest) : largest;
            const float far = value == kNoReference ? 1.0f : exp2_of((shift - to) * scale + (value + bias));
            fade = out ? far : fade;
            next = out ? -bias : next;
            limit = out ? -INFINITY : limit;
            shift = out ? to : 0.0f;
#pragma unroll
            for (auto& block : s)
#pragma unroll
                for (int i = 0; i < 16; ++i) block[i] -= shift;
        }
        value = next;
        return fade;
    }
    // As one number, for a part's partial results and the logarithm of the sum.
    __device__ __forceinline__ float whole(float scale) const { return shift * scale + value; }
};

// The larger of the two lanes of a row.
__device__ __forceinline__ float row_max(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto both = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}
__device__ __forceinline__ float row_sum(float x) {
    const uint32_t u = __float_as_uint(x);
    const auto both = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __uint_as_float(both[0]) + __uint_as_float(both[1]);
}

// 16 bytes a lane from memory to LDS at `lds` (wave-uniform) + 16 * lane, not waited for.  In assembly, so
// that the compiler does not wait for them before every LDS read: the callers' own waits and barriers
// order them.  Nothing is written but LDS.  The compiler counts no wait states into an assembly block: m0 needs one
// before the load, and a resource's registers five after a vector instruction (v_readfirstlane) wrote them.
__device__ __forceinline__ void fetch_buffer(u4 rsrc, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(rsrc)
                 : "memory", "m0");
}
__device__ __forceinline__ void fetch_global(int64_t address, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(address) : "memory", "m0");
}

__device__ __forceinline__ u4 tile_rsrc(int64_t base, uint32_t bytes) {
    u4 r;
    r[0] = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(base));
    r[1] = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(base >> 32) & 0xffffu);
    r[2] = __builtin_amdgcn_readfirstlane(bytes);
    r[3] = kBufferWord3;
    return r;
}

// Where a row of queries stands: its token and head, the keys it sees.
struct QueryRow {
    int token, head, first, last;
    bool valid;
};

__device__ __forceinline__ QueryRow query_row(const rch_attend& A, const AttendItem& I, int row) {
    QueryRow R;
    const int group = static_cast<int>(A.group);
    R.valid = row < I.row_end;
    const int r = R.valid ? row : I.row_end - 1;
    R.token = r / group;
    R.head = I.kv_head * group + r - R.token * group;
    attend_range(A, I, R.token, R.first, R.last);
    return R;
}

// A table entry by a per-lane index.
__device__ __forceinline__ int page_entry(const const_int* table, int index) {
    return gin<int32_t>(static_cast<int64_t>(reinterpret_cast<uintptr_t>(table)))[index];
}

// How a tile's rows are found: kPage: tiles start over at each page and lie in one page; kShare: a tile is KT
// consecutive keys, and the KT / 4 rows that a wave fetches lie in one page (its size is a multiple of that);
// kRow: any page size.  The first two take a scalar base to a fetch, the last an address to a lane.
// kList: chosen blocks of keys, one after the other; a block lies in one page and tiles start over at each.
// kPack: chosen blocks whose size is a multiple of KT / 4: tiles run on over them, each wave's rows lie in one.
enum TileMode { kPage, kShare, kRow, kList, kPack };

// Quotients of numbers below 2^31 by one divisor: the reciprocal is rounded down, so a product is one too few at most.
struct Divider {
    uint32_t by, reciprocal;
    __device__ __forceinline__ void init(uint32_t d) { by = d, reciprocal = 0xffffffffu / d; }
    __device__ __forceinline__ int quotient(int x) const {
        const uint32_t q = __umulhi(static_cast<uint32_t>(x), reciprocal);
        return static_cast<int>(q + (static_cast<uint32_t>(x) - q * by >= by ? 1 : 0));
    }
};

// The page of a walk's tile and the tile's first row there, for those who ask (pools in codes find the rows' scales by it).
template <bool KEPT>
struct TilePlace {
    __device__ __forceinline__ void stand(int, int) {}
    __device__ __forceinline__ void step(int) {}
};
template <>
struct TilePlace<true> {
    int id, in_page;
    __device__ __forceinline__ void stand(int page, int row) { id = page, in_page = row; }
    __device__ __forceinline__ void step(int rows) { in_page += rows; }
};

// The walk over an item's key tiles.
template <int KT, int MODE, bool KEPT = false>
struct KeyWalk : TilePlace<KEPT> {
    const const_int* table;
    int unit, end, pages;     // tokens that tiles start over at, last key, pages of the pool
    int base, left, page;     // current tile: first key, keys from it to the unit's end, page index (kPage)
    int64_t k, v;             // kPage: addresses of the tile's first K and V row
    int64_t k_head, v_head, k_page, v_page;  // of the item's head in page 0; bytes of a page
    int k_tile, v_tile;       // bytes of KT rows

    __device__ __forceinline__ bool done() const { return base >= end; }
    // Enters the page of `base` (at row `off`), skipping dropped ones.
    __device__ __forceinline__ void enter(int off) {
        while (!done()) {
            const int id = table[page];
            if (id >= 0 && id < pages) {
                k = k_head + id * k_page + static_cast<int64_t>(off / KT) * k_tile;
                v = v_head + id * v_page + static_cast<int64_t>(off / KT) * v_tile;
                this->stand(id, off);
                return;
            }
            base += left;
            left = unit;
            ++page;
            off = 0;
        }
    }
    __device__ __forceinline__ void begin(const rch_attend& A, const AttendItem& I, int es) {
        table = (const const_int*)(uintptr_t)(A.plan_ptr + 4 * static_cast<int64_t>(I.table));
        unit = static_cast<int>(A.tile_unit);
        end = I.key_end;
        pages = static_cast<int>(A.pages);
        k_head = A.k_ptr + es * I.kv_head * A.k_head_stride;
        v_head = A.v_ptr + es * I.kv_head * A.v_head_stride;
        k_page = es * A.k_page_stride;
        v_page = es * A.v_page_stride;
        k_tile = static_cast<int>(es * KT * A.k_token_stride);
        v_tile = static_cast<int>(es * KT * A.v_token_stride);
        page = I.key_begin / unit;
        const int off = (I.key_begin - page * unit) / KT * KT;
        base = page * unit + off;
        left = unit - off;
        if constexpr (MODE == kPage) enter(off);
    }
    __device__ __forceinline__ void next() {
        if constexpr (MODE == kPage) {
            if (left > KT) {
                base += KT;
                left -= KT;
                k += k_tile;
                v += v_tile;
                this->step(KT);
                return;
            }
            base += left;
            left = unit;
            ++page;
            enter(0);
        } else {
            base += KT;
        }
    }
    // Keys of the current tile.
    __device__ __forceinline__ int count() const { return min(end - base, MODE == kPage ? min(left, KT) : KT); }
};

// The walk over the tiles of an item's chosen blocks.  An entry's page is looked up a block before it is entered, and the
// entry itself two before, so that no tile waits for either.
template <int KT, bool KEPT>
struct KeyWalk<KT, kList, KEPT> : TilePlace<KEPT> {
    const const_int *table, *entry;
    int unit, end, pages, blocks;   // tokens of a block, keys and blocks of the sequence
    Divider per_page;               // blocks of a page
    int tiles;                      // of the item, the current one among them
    int entries;                    // of the list that are left to read
    int base, left;                 // current tile: first key, keys from it to the block's end
    int block1, page1, off1, block2;  // the next block, its page and place there; the one behind it
    int64_t k, v, k_head, v_head, k_page, v_page;
    int k_tile, v_tile, k_row, v_row;

    __device__ __forceinline__ bool done() const { return tiles <= 0; }
    __device__ __forceinline__ int read() {
        if (entries <= 0) return -1;
        --entries;
        return *entry++;
    }
    // Moves the entries up by one.
    __device__ __forceinline__ void shift() {
        block1 = block2;
        page1 = -1;
        if (block1 >= 0 && block1 < blocks) {
            const int index = per_page.quotient(block1);
            off1 = (block1 - index * static_cast<int>(per_page.by)) * unit;
            page1 = table[index];
        }
        block2 = read();
    }
    // Enters the next block at its tile `sub`, skipping entries without keys.
    __device__ __forceinline__ void enter(int sub) {
        while (tiles > 0) {
            const int block = block1, id = page1, first = off1 + sub * KT;
            shift();
            // (a tile behind the sequence's last key has none either)
            if (id >= 0 && id < pages && block * unit + sub * KT < end) {
                this->stand(id, first);
                k = k_head + id * k_page + first * static_cast<int64_t>(k_row);
                v = v_head + id * v_page + first * static_cast<int64_t>(v_row);
                base = block * unit + sub * KT;
                left = unit - sub * KT;
                return;
            }
            tiles -= (unit + KT - 1) / KT - sub;
            sub = 0;
        }
    }
    __device__ __forceinline__ void begin(const rch_attend& A, const AttendItem& I, int es) {
        table = (const const_int*)(uintptr_t)(A.plan_ptr + 4 * static_cast<int64_t>(I.table));
        unit = static_cast<int>(A.block_tokens);
        per_page.init(static_cast<uint32_t>(A.page_tokens) / static_cast<uint32_t>(unit));
        end = I.length;
        blocks = (end + unit - 1) / unit;
        pages = static_cast<int>(A.pages);
        k_head = A.k_ptr + es * I.kv_head * A.k_head_stride;
        v_head = A.v_ptr + es * I.kv_head * A.v_head_stride;
        k_page = es * A.k_page_stride;
        v_page = es * A.v_page_stride;
        k_row = static_cast<int>(es * A.k_token_stride);
        v_row = static_cast<int>(es * A.v_token_stride);
        k_tile = KT * k_row;
        v_tile = KT * v_row;
        const int per = (unit + KT - 1) / KT, at = I.key_begin / per;
        entry = (const const_int*)(uintptr_t)(A.lists_ptr + 4 * static_cast<int64_t>(I.list)) + at;
        tiles = I.key_end - I.key_begin;
        entries = tiles > 0 ? (I.key_end + per - 1) / per - at : 0;
        off1 = 0;
        block2 = read();
        shift();
        enter(I.key_begin - at * per);
    }
    __device__ __forceinline__ void next() {
        --tiles;
        if (left > KT && base + KT < end) {
            base += KT;
            left -= KT;
            k += k_tile;
            v += v_tile;
            this->step(KT);
            return;
        }
        tiles -= (left - 1) / KT;  // tiles of the block behind the sequence's last key
        enter(0);
    }
    __device__ __forceinline__ int count() const { return min(end - base, min(left, KT)); }
};

// The walk over tiles that run on over chosen blocks.  A tile is four shares of KT / 4 rows, each of one block; a wave
// fetches its own and knows the place of all, for the masks.  Entries are read two tiles ahead, their pages one.
template <int KT, bool KEPT>
struct KeyWalk<KT, kPack, KEPT> {
    static constexpr int S = KT / 4;
    const const_int *table, *list;
    int unit, end, pages, blocks;
    Divider per_block, per_page;  // keys of a block, blocks of a page
    int wave, at, stop;           // the wave; keys of the list before the current tile, and before the end
    int block[4], page[4];        // of the current tile's shares: entries and pages (-1: no key)
    int ahead[4];                 // entries of the next tile
    int64_t k_head, v_head, k_page, v_page;
    int k_row, v_row;

    __device__ __forceinline__ bool done() const { return at >= stop; }
    __device__ __forceinline__ int offset(int s) const {
        const int x = at + s * S;
        return x - per_block.quotient(x) * unit;
    }
    __device__ __forceinline__ void read(int from) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int x = from + s * S;
            ahead[s] = -1;
            if (x < stop) ahead[s] = list[per_block.quotient(x)];
        }
    }
    // The tile at `at` becomes the current one.
    __device__ __forceinline__ void look_up() {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            block[s] = ahead[s] < blocks ? ahead[s] : -1;
            page[s] = -1;
            if (block[s] >= 0) page[s] = table[per_page.quotient(block[s])];
        }
        read(at + KT);
    }
    __device__ __forceinline__ void begin(const rch_attend& A, const AttendItem& I, int es) {
        table = (const const_int*)(uintptr_t)(A.plan_ptr + 4 * static_cast<int64_t>(I.table));
        list = (const const_int*)(uintptr_t)(A.lists_ptr + 4 * static_cast<int64_t>(I.list));
        unit = static_cast<int>(A.block_tokens);
        per_block.init(static_cast<uint32_t>(unit));
        per_page.init(static_cast<uint32_t>(A.page_tokens) / static_cast<uint32_t>(unit));
        end = I.length;
        blocks = (end + unit - 1) / unit;
        pages = static_cast<int>(A.pages);
        k_head = A.k_ptr + es * I.kv_head * A.k_head_stride;
        v_head = A.v_ptr + es * I.kv_head * A.v_head_stride;
        k_page = es * A.k_page_stride;
        v_page = es * A.v_page_stride;
        k_row = static_cast<int>(es * A.k_token_stride);
        v_row = static_cast<int>(es * A.v_token_stride);
        at = __builtin_amdgcn_readfirstlane(I.key_begin * KT);
        stop = __builtin_amdgcn_readfirstlane(min(I.key_end * KT, I.entries * unit));
        read(at);
        look_up();
    }
    __device__ __forceinline__ void next() {
        at += KT;
        look_up();
    }
    // First key and keys of share s of the current tile (0 keys: -1).
    __device__ __forceinline__ int first_key(int s) const { return page[s] >= 0 && page[s] < pages ? block[s] * unit + offset(s) : -1; }
    __device__ __forceinline__ int keys(int first) const { return first < 0 ? 0 : max(0, min(end - first, S)); }
    // (by values: a choice of places would put the four into memory)
    __device__ __forceinline__ int own(const int (&x)[4]) const {
        const int a = x[0], b = x[1], c = x[2], d = x[3], low = wave & 1 ? b : a, high = wave & 1 ? d : c;
        return wave & 2 ? high : low;
    }
    // The wave's own share: its page (or -1), the first row there, and its keys.
    __device__ __forceinline__ void own(int& id, int& in_page, int& rows) const {
        const int b = own(block), x = offset(wave);
        id = own(page);
        if (id >= pages) id = -1;
        rows = id < 0 ? 0 : keys(b * unit + x);
        in_page = (b - per_page.quotient(max(b, 0)) * static_cast<int>(per_page.by)) * unit + x;
    }
};

// What a wave's rows see of a tile of four shares whose first keys are `key` (-1: none).
template <int S>
struct ShareView {
    bool sees, masked, hides;
    template <typename Walk, typename Range>
    __device__ __forceinline__ void look(const Walk& W, const Range& R, const int (&key)[4]) {
        sees = masked = hides = false;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int n = W.keys(key[s]);
            masked = masked || n < S;
            sees = sees || (n > 0 && key[s] + n > R.first_low && key[s] < R.last_high);
            hides = hides || (n > 0 && (key[s] < R.first_high || key[s] + n > R.last_low));
        }
        masked = masked || hides;
    }
    // Bits of the keys that one row sees.
    template <typename Walk>
    static __device__ __forceinline__ uint64_t bits(const Walk& W, const int (&key)[4], int first, int last) {
        uint64_t all = 0;
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const int n = W.keys(key[s]), from = max(first - key[s], 0), to = min(last - key[s], n);
            const uint32_t mask = to > from ? ((1u << to) - 1) & ~((1u << from) - 1) : 0;  // to <= 16
            all |= static_cast<uint64_t>(mask) << (s * S);
        }
        return all;
    }
};

// Fetches the calling wave's quarter of a K and a V tile: NI instructions of 1024 bytes each.  Tile: the
// arithmetic's layout (ES: bytes of an element, RB: LDS bytes of a row, the swizzles).
template <typename Tile, int MODE>
struct Fetch {
    static constexpr int KT = Tile::KT, RB = Tile::RB, ES = Tile::ES, kRows = 1024 / RB, kPieces = RB / 16, kShareRows = KT / 4;
    static constexpr int NI = kShareRows / kRows;
    uint32_t k_at[MODE == kRow ? 1 : NI], v_at[MODE == kRow ? 1 : NI];  // byte offsets from the scalar base
    int share, row0, piece, pieces;  // the share's first row, the lane's first one, its piece, pieces of a head
    uint32_t size, magic, row_bytes, k_row, v_row;
    int ids[MODE == kRow ? NI : 1];  // pages of the walk's tile

    __device__ __forceinline__ void init(const rch_attend& A, int wave, int lane) {
        pieces = static_cast<int>(A.head_dim) * ES / 16;
        share = wave * kShareRows;
        row0 = share + lane / kPieces;
        piece = lane % kPieces;
        row_bytes = static_cast<uint32_t>(A.head_dim) * ES;
        k_row = static_cast<uint32_t>(A.k_token_stride * ES);
        v_row = static_cast<uint32_t>(A.v_token_stride * ES);
        size = static_cast<uint32_t>(A.page_tokens);
        magic = (65536u + size - 1) / size;  // x / size for x < 128, size <= 64
        if constexpr (MODE != kRow) {
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int row = row0 + i * kRows, from = MODE == kShare || MODE == kPack ? row - share : row;
                const int kc = piece ^ Tile::k_swizzle(row), vc = piece ^ Tile::v_swizzle(row);
                k_at[i] = kc < pieces ? from * k_row + kc * 16 : kOutOfRange;
                v_at[i] = vc < pieces ? from * v_row + vc * 16 : kOutOfRange;
            }
        }
    }
    // Pages from the first key's that row x (counted from that page's start) lies in.
    __device__ __forceinline__ int page_of(uint32_t x) const {
        return size < 64 ? static_cast<int>((x * magic) >> 16) : (x >= size ? 1 : 0);
    }

    // Looks up the pages of the walk's tile (called when the walk arrives there, a tile before its fetch, so that
    // the fetch waits for no table).
    __device__ __forceinline__ void look_up(const KeyWalk<KT, MODE>& W) {
        if constexpr (MODE == kShare || MODE == kRow) {
            if (W.done()) return;
            const int keys = W.end - W.base, page0 = W.base / static_cast<int>(size);
            const int off0 = W.base - page0 * static_cast<int>(size);
            // Rows behind the last key: its page.
            if constexpr (MODE == kShare) {
                ids[0] = W.table[page0 + page_of(off0 + min(share, keys - 1))];
            } else {
#pragma unroll
                for (int i = 0; i < NI; ++i) ids[i] = page_entry(W.table, page0 + page_of(off0 + min(row0 + i * kRows, keys - 1)));
            }
        }
    }

    __device__ __forceinline__ void issue(const rch_attend& A, const KeyWalk<KT, MODE>& W, uint32_t k_lds, uint32_t v_lds) const {
        if constexpr (MODE != kRow) {
            int64_t k, v;
            int rows;
            if constexpr (MODE == kPack) {
                k_lds = __builtin_amdgcn_readfirstlane(k_lds), v_lds = __builtin_amdgcn_readfirstlane(v_lds);  // (of wide heads, out of a vector register)
                int id, in_page;
                W.own(id, in_page, rows);
                k = rows > 0 ? W.k_head + id * W.k_page + in_page * static_cast<int64_t>(k_row) : A.plan_ptr;
                v = rows > 0 ? W.v_head + id * W.v_page + in_page * static_cast<int64_t>(v_row) : A.plan_ptr;
            } else {
                k = W.k, v = W.v;
                rows = W.count();
            }
            if constexpr (MODE == kShare) {
                // Rows behind the last key, and those of a dropped page, are out of the buffer's range: zeros.
                const int x = W.base % static_cast<int>(size) + share, in_page = x - page_of(x) * static_cast<int>(size);
                rows = ids[0] >= 0 && ids[0] < W.pages ? min(rows - share, kShareRows) : 0;
                k = W.k_head + ids[0] * W.k_page + in_page * static_cast<int64_t>(k_row);
                v = W.v_head + ids[0] * W.v_page + in_page * static_cast<int64_t>(v_row);
                if (rows <= 0) k = v = A.plan_ptr;
            }
            const u4 kr = tile_rsrc(k, rows > 0 ? (rows - 1) * k_row + row_bytes : 0);
            const u4 vr = tile_rsrc(v, rows > 0 ? (rows - 1) * v_row + row_bytes : 0);
#pragma unroll
            for (int i = 0; i < NI; ++i) fetch_buffer(kr, k_at[i], k_lds + i * 1024);
#pragma unroll
            for (int i = 0; i < NI; ++i) fetch_buffer(vr, v_at[i], v_lds + i * 1024);
        } else {
            const int keys = W.end - W.base, off0 = W.base % static_cast<int>(size);
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int row = row0 + i * kRows, x = off0 + row, in_page = x - page_of(x) * static_cast<int>(size);
                const int id = row < keys ? ids[i] : -1;
                const bool held = id >= 0 && id < W.pages;
                const int kc = piece ^ Tile::k_swizzle(row), vc = piece ^ Tile::v_swizzle(row);
                const int64_t k = W.k_head + id * W.k_page + in_page * static_cast<int64_t>(k_row) + kc * 16;
                const int64_t v = W.v_head + id * W.v_page + in_page * static_cast<int64_t>(v_row) + vc * 16;
                // Rows that no page holds, and pieces behind the head, read the plan's zeros.
                fetch_global(held && kc < pieces ? k : A.plan_ptr, k_lds + i * 1024);
                fetch_global(held && vc < pieces ? v : A.plan_ptr, v_lds + i * 1024);
            }
        }
    }
};

// What the rows of a wave see, as scalars.
struct WaveRange {
    int first_low, first_high, last_low, last_high;

    __device__ __forceinline__ void init(const QueryRow& R) {
        first_low = first_high = R.first;
        last_low = last_high = R.last;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            first_low = min(first_low, __shfl_xor(first_low, o));
            first_high = max(first_high, __shfl_xor(first_high, o));
            last_low = min(last_low, __shfl_xor(last_low, o));
            last_high = max(last_high, __shfl_xor(last_high, o));
        }
        first_low = __builtin_amdgcn_readfirstlane(first_low);
        first_high = __builtin_amdgcn_readfirstlane(first_high);
        last_low = __builtin_amdgcn_readfirstlane(last_low);
        last_high = __builtin_amdgcn_readfirstlane(last_high);
    }
    // Whether a row may see a key of a tile, and whether one may not see all of its KT keys.
    __device__ __forceinline__ bool sees(int base, int count) const { return base + count > first_low && base < last_high; }
    // Whether a row may not see one of the tile's own keys.
    __device__ __forceinline__ bool hides(int base, int count) const { return base < first_high || base + count > last_low; }
    __device__ __forceinline__ bool masked(int base, int count, int kt) const {
        return base < first_high || base + kt > last_low || count < kt;
    }
};

// Bit i of seen[b]: whether the row sees the key of register i of block b.
    template <int KB>
__device__ __forceinline__ void seen_keys(uint32_t (&seen)[KB], int first, int last, uint64_t held, int h) {
        // Bits of keys [first, last) of the tile, then those of this lane's half.
        uint64_t bits = first >= 64 || last <= 0 || last <= first ? 0 : ~uint64_t{0} << max(first, 0);
        if (last < 64) bits &= (uint64_t{1} << max(last, 0)) - 1;
        bits &= held;
#pragma unroll
        for (int b = 0; b < KB; ++b) {
            const uint32_t w = static_cast<uint32_t>(bits >> (32 * b)) >> (4 * h);
            seen[b] = (w & 0xfu) | (w >> 4 & 0xf0u) | (w >> 8 & 0xf00u) | (w >> 12 & 0xf000u);
        }
    }

// Adds what the codes of infinite and NaN values (below) say.
__device__ __forceinline__ void add_marks(f16v& sum, const f16v& code) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int n = static_cast<int>(code[i]);
        if (n & 127) sum[i] += INFINITY;
        if (n >> 7 & 127) sum[i] -= INFINITY;
        if (n >= 16384) sum[i] = __builtin_nanf("");
    }
}

// One wave's state over the tiles and the arithmetic of a tile of KB * 32 keys.  LEAN: with fewer registers.  PAIRS: a tile
// that lanes write two neighbouring pieces of eight channels to (CodeFetch), in two stores.  Eight lanes store 128 bytes at a
// time, so that every other piece of a row would meet each bank twice: a piece's low bit goes where eight lanes' bits do not
// (a chunk's kernel spent 66 cycles of LDS on such meetings for a wave's tile, beside 98 of its own).
template <int DT, int NB, int KB, bool LEAN = false, bool PAIRS = false>
struct RowTile {
    typedef Half<DT> H;
    typedef typename H::type T;
    typedef typename H::vec8 vec8;
    typedef typename H::vec4 vec4;
    static constexpr int ES = 2, RB = NB <= 2 ? 128 : NB <= 4 ? 256 : 512, kPieces = RB / 16, KT = 32 * KB;
    static constexpr bool kApart = PAIRS && RB > 128;
    static __device__ __forceinline__ int k_swizzle(int row) { return row % kPieces; }
    static __device__ __forceinline__ int v_swizzle(int row) {
        if constexpr (kApart) return (row & 1) | (row & 2) << 1;
        if constexpr (PAIRS) return ((row >> 1) & 1) * 4 | (row & 1);
        return kPieces >= 16 ? (row & 3) * 4 : ((row >> 1) & 1) * 4;
    }
    // Where a row's pieces lie, before the exchange of its swizzle (bits change places: sums of bits stay sums).
    static __device__ __forceinline__ constexpr int k_place(int piece) { return kApart ? piece >> 1 | (piece & 1) * (kPieces / 2) : piece; }
    static __device__ __forceinline__ constexpr int v_place(int piece) { return kApart ? (piece & ~9) | (piece & 1) << 3 | (piece >> 3 & 1) : piece; }

    vec8 q[2 * NB];
    f16v o[NB];
    Reference reference;
    float sum;
    // LDS byte offsets within a tile; of wide heads the first, from which the others follow by an exclusive or.
    static constexpr bool kWide = NB > 4 || LEAN;
    uint32_t k_lane[kWide ? 1 : 2 * NB], v_lane[kWide ? 1 : NB];
    __device__ __forceinline__ uint32_t k_at(int s) const { return kWide ? k_lane[0] ^ (k_place(2 * s) * 16) : k_lane[s]; }
    __device__ __forceinline__ uint32_t v_at(int b) const { return kWide ? v_lane[0] ^ (v_place(4 * b) * 16) : v_lane[b]; }

    __device__ __forceinline__ void init(const rch_attend& A, const AttendItem& I, const QueryRow& R, int lane) {
        const int n = lane & 31, h = lane >> 5;
        const int64_t at = A.q_ptr + 2 * ((I.q_row + R.token) * A.q_token_stride + R.head * A.q_head_stride);
#pragma unroll
        for (int s = 0; s < 2 * NB; ++s) {
            const int d = 16 * s + 8 * h;
            q[s] = __builtin_bit_cast(vec8, *gin<u4>(R.valid && d < A.head_dim ? at + 2 * d : A.plan_ptr));  // or zeros
            if (!kWide || s == 0) k_lane[s] = n * RB + ((k_place(2 * s + h) ^ k_swizzle(n)) * 16);
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) {
            if (!kWide || b == 0) v_lane[b] = value_offset(b, lane);
            o[b] = f16v{};
        }
        reference.init();
        sum = 0.0f;
    }

    // One tile.  [first, last): keys of the tile that the lane's row sees; held: keys in pages (bits).  masked
    // (wave-uniform): whether a row of the wave may see fewer than all.  RARE: the values may be infinite or NaN
    // where masked (the callers go on in a loop of its own then: its registers would cost the usual one).
    template <bool RARE>
    __device__ __forceinline__ void step(const lds_char* k_tile, const lds_char* v_tile, float scale, int first, int last,
                                         uint64_t held, bool masked, int lane) {
        const int h = lane >> 5;
        f16v s[KB];
#pragma unroll
        for (int b = 0; b < KB; ++b) s[b] = f16v{};
        // The blocks' chains side by side, the reads kAhead products ahead (2, 4 or 6: the same within 1 %; in the
        // compiler's own order a chunk takes 951 us against 943).
#pragma unroll
        for (int c = 0; c < 2 * NB; ++c)
#pragma unroll
            for (int b = 0; b < KB; ++b) {
                const vec8 k = *reinterpret_cast<const __attribute__((address_space(3))) vec8*>(k_tile + k_at(c) + b * 32 * RB);
                s[b] = H::mfma(k, q[c], s[b]);
            }
        constexpr int kAhead = 6, kProducts = 2 * NB * KB;
        __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
        for (int i = 0; i < kProducts; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
            if (i + kAhead < kProducts) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        if (masked) {
            uint32_t seen[KB];
            seen_keys(seen, first, last, held, h);
#pragma unroll
            for (int b = 0; b < KB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[b][i] = seen[b] >> i & 1u ? s[b][i] : -INFINITY;
        }
        // The first values, on their way while the weights are computed.
        constexpr int kRing = NB > 4 ? 4 : LEAN ? 2 : NB;  // values read ahead
        vec8 v[kRing];
        if constexpr (!RARE) {
#pragma unroll
            for (int b = 0; b < kRing; ++b) v[b] = values(v_tile + v_at(b), 0);
        }
        float top = s[0][0];
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = fmaxf(top, s[b][i]);
        top = row_max(top);
        const float scaled = top * scale - H::kBias;
        if (__any(scaled > reference.limit)) {
            const float fade = reference.move(top, scaled, scale, H::kBias, s);
            sum *= fade;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[b][i] *= fade;
        }
        vec8 p[2 * KB];
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int b = 0; b < KB; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float w = exp2_of(__builtin_fmaf(s[b][i], scale, -reference.value));
                part[i & 3] += w;
                p[2 * b + (i >> 3)][i & 7] = static_cast<T>(w);
            }
        sum += (part[0] + part[1]) + (part[2] + part[3]);
        if constexpr (RARE) {
            if (masked) {
                Rare rare;
#pragma unroll
                for (int b = 0; b < NB; ++b) rare.o[b] = o[b];
#pragma unroll
                for (int c = 0; c < 2 * KB; ++c) rare.p[c] = p[c];
                seen_keys(rare.seen, first, last, held, h);
                add_infinite(&rare, v_tile, lane);
#pragma unroll
                for (int b = 0; b < NB; ++b) o[b] = rare.o[b];
                return;
            }
        }
#pragma unroll
        for (int c = 0; c < 2 * KB; ++c)
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const int at = c * NB + b, next = at + kRing;
                const vec8 now = RARE ? values(v_tile + v_at(b), c) : v[at % kRing];
                if (!RARE && next < 2 * KB * NB) v[at % kRing] = values(v_tile + v_at(next % NB), next / NB);
                o[b] = H::mfma(now, p[c], o[b]);
            }
    }

    // Whether a value of the tile is infinite or NaN: with a weight of 0 (a key that a row does not see) its
    // product would be NaN.
    static __device__ __forceinline__ bool any_infinite(const lds_char* v_tile, int lane) {
        uint32_t found = 0;
#pragma unroll 4
        for (int i = 0; i < KT * RB / 1024; ++i) {
            const u4 raw = *reinterpret_cast<const __attribute__((address_space(3))) u4*>(v_tile + i * 1024 + lane * 16);
#pragma unroll
            for (int w = 0; w < 4; ++w)
                found |= ((raw[w] & H::kExponent) == H::kExponent) | ((raw[w] >> 16 & H::kExponent) == H::kExponent);
        }
        return __any(found != 0);
    }

    // The second product of a tile with infinite or NaN values: the finite ones as always, and beside them a
    // product of ones for the keys that a row sees with a code for the others (1: inf, 128: -inf, 16384: NaN;
    // at most 64 of each), from whose exact sum the channel's result follows.  A call through memory, out of
    // the registers of the tiles' arithmetic.
    struct Rare {
        f16v o[NB];
        vec8 p[2 * KB];
        uint32_t seen[KB];
    };
    static __device__ __attribute__((noinline)) void add_infinite(Rare* rare, const lds_char* v_tile, int lane) {
#pragma unroll 1
        for (int b = 0; b < NB; ++b) {
            const uint32_t at = value_offset(b, lane);
            f16v code = f16v{}, sum = rare->o[b];
#pragma unroll 1
            for (int c = 0; c < 2 * KB; ++c) {
                vec8 v = values(v_tile + at, c), mark, one;
                const uint32_t seen = rare->seen[c >> 1] >> (8 * (c & 1));
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = static_cast<float>(v[e]);
                    mark[e] = static_cast<T>(x != x ? 16384.0f : (x == INFINITY ? 1.0f : (x == -INFINITY ? 128.0f : 0.0f)));
                    v[e] = __builtin_fabsf(x) < INFINITY ? v[e] : static_cast<T>(0.0f);
                    one[e] = static_cast<T>(seen >> e & 1u ? 1.0f : 0.0f);
                }
                sum = H::mfma(v, rare->p[c], sum);
                code = H::mfma(mark, one, code);
            }
            add_marks(sum, code);
            rare->o[b] = sum;
        }
    }

    // A lane's offset, within a tile, of the A operand V^T of channels 32 b .. 32 b + 31, and the operand of
    // keys 16 c .. 16 c + 15 from there.
    static __device__ __forceinline__ uint32_t value_offset(int b, int lane) {
        const int p = lane & 15, key = 4 * (lane >> 5) + (p >> 2), half = (lane >> 4) & 1;
        const int piece = v_place(4 * b + 2 * half + ((p & 3) >> 1)) ^ v_swizzle(key);
        return key * RB + piece * 16 + (p & 1) * 8;
    }
    static __device__ __forceinline__ vec8 values(const lds_char* at, int c) {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef short s8 __attribute__((ext_vector_type(8)));
        typedef __attribute__((address_space(3))) s4 lds_s4;
        const s4 low = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + c * 16 * RB));
        const s4 high = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + c * 16 * RB + 8 * RB));
        return __builtin_bit_cast(vec8, static_cast<s8>(__builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7)));
    }

    // Channel of register i of block b, and a row's channels i .. i + 3 into memory.
    static __device__ __forceinline__ int channel_of(int b, int i, int h) { return 32 * b + 8 * (i >> 2) + 4 * h + (i & 3); }
    static __device__ __forceinline__ void store4(int64_t to, f4 v) {
        vec4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = static_cast<T>(v[e]);
        *gout<u2>(to) = __builtin_bit_cast(u2, r);
    }
};

// The same for fp32, 32 keys to a tile, by v_mfma_f32_32x32x2: its inner index is the lane's half alone, so a
// 16-byte piece of K (and of Q) feeds four products, and register i of S^T is, as it is, the B operand of the
// keys that registers i of both halves hold; V^T is read one value a lane.
template <int NB>
struct RowTile<RCH_DT_F32, NB, 1, false, false> {
    typedef float T;
    static constexpr int ES = 4, RB = NB <= 2 ? 256 : NB <= 4 ? 512 : 1024, kPieces = RB / 16, KT = 32;
    static __device__ __forceinline__ int k_swizzle(int row) { return row % kPieces; }
    // The two halves read keys 4 apart at the same channels: half a 256-byte bank row apart.
    static __device__ __forceinline__ int v_swizzle(int row) { return ((row >> 2) & 1) * 8; }

    f4 q[4 * NB];
    f16v o[NB];
    Reference reference;
    float sum;
    uint32_t k_lane, v_lane, k_turn;

    __device__ __forceinline__ void init(const rch_attend& A, const AttendItem& I, const QueryRow& R, int lane) {
        const int n = lane & 31, h = lane >> 5;
        const int64_t at = A.q_ptr + 4 * ((I.q_row + R.token) * A.q_token_stride + R.head * A.q_head_stride);
#pragma unroll
        for (int s = 0; s < 4 * NB; ++s) {
            const int d = 8 * s + 4 * h;
            q[s] = __builtin_bit_cast(f4, *gin<u4>(R.valid && d < A.head_dim ? at + 4 * d : A.plan_ptr));  // or zeros
        }
        k_lane = n * RB;
        k_turn = (k_swizzle(n) ^ h) * 16;
        v_lane = 4 * h * RB + ((n >> 2) ^ v_swizzle(4 * h)) * 16 + (n & 3) * 4;
#pragma unroll
        for (int b = 0; b < NB; ++b) o[b] = f16v{};
        reference.init();
        sum = 0.0f;
    }

    template <bool RARE>
    __device__ __forceinline__ void step(const lds_char* k_tile, const lds_char* v_tile, float scale, int first, int last,
                                         uint64_t held, bool masked, int lane) {
        const int h = lane >> 5;
        f16v s[1] = {f16v{}};
#pragma unroll
        for (int c = 0; c < 4 * NB; ++c) {
            const f4 k = *reinterpret_cast<const __attribute__((address_space(3))) f4*>(k_tile + k_lane + (k_turn ^ (c * 32)));
#pragma unroll
            for (int j = 0; j < 4; ++j) s[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(k[j], q[c][j], s[0], 0, 0, 0);
        }
        uint32_t seen[1] = {0xffffu};
        if (masked) {
            seen_keys(seen, first, last, held, h);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[0][i] = seen[0] >> i & 1u ? s[0][i] : -INFINITY;
        }
        float top = s[0][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[0][i]);
        top = row_max(top);
        if (__any(top * scale > reference.limit)) {
            const float fade = reference.move(top, top * scale, scale, 0.0f, s);
            sum *= fade;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[b][i] *= fade;
        }
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            s[0][i] = exp2_of(__builtin_fmaf(s[0][i], scale, -reference.value));
            part[i & 3] += s[0][i];
        }
        sum += (part[0] + part[1]) + (part[2] + part[3]);
        if constexpr (RARE) {
            if (masked) {
                Rare rare;
#pragma unroll
                for (int b = 0; b < NB; ++b) rare.o[b] = o[b];
#pragma unroll
                for (int i = 0; i < 16; ++i) rare.p[i] = s[0][i];
                rare.seen = seen[0];
                add_infinite(&rare, v_tile, v_lane);
#pragma unroll
                for (int b = 0; b < NB; ++b) o[b] = rare.o[b];
                return;
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
#pragma unroll
            for (int b = 0; b < NB; ++b) o[b] = __builtin_amdgcn_mfma_f32_32x32x2f32(value(v_tile, v_lane, b, i), s[0][i], o[b], 0, 0, 0);
    }

    // Key 8 (i / 4) + 4 h + i % 4 (its row's swizzle depends on h alone), channel 32 b + lane % 32.
    static __device__ __forceinline__ float value(const lds_char* v_tile, uint32_t v_lane, int b, int i) {
        const uint32_t row = (8 * (i >> 2) + (i & 3)) * RB;
        return *reinterpret_cast<const __attribute__((address_space(3))) float*>(v_tile + row + (v_lane ^ (b * 128)));
    }

    static __device__ __forceinline__ bool any_infinite(const lds_char* v_tile, int lane) {
        uint32_t found = 0;
#pragma unroll 4
        for (int i = 0; i < KT * RB / 1024; ++i) {
            const u4 raw = *reinterpret_cast<const __attribute__((address_space(3))) u4*>(v_tile + i * 1024 + lane * 16);
#pragma unroll
            for (int w = 0; w < 4; ++w) found |= (raw[w] & 0x7f800000u) == 0x7f800000u;
        }
        return __any(found != 0);
    }

    struct Rare {
        f16v o[NB];
        float p[16];
        uint32_t seen;
    };
    static __device__ __attribute__((noinline)) void add_infinite(Rare* rare, const lds_char* v_tile, uint32_t v_lane) {
#pragma unroll 1
        for (int b = 0; b < NB; ++b) {
            f16v code = f16v{}, sum = rare->o[b];
#pragma unroll 1
            for (int i = 0; i < 16; ++i) {
                const float x = value(v_tile, v_lane, b, i);
                const float mark = x != x ? 16384.0f : (x == INFINITY ? 1.0f : (x == -INFINITY ? 128.0f : 0.0f));
                sum = __builtin_amdgcn_mfma_f32_32x32x2f32(__builtin_fabsf(x) < INFINITY ? x : 0.0f, rare->p[i], sum, 0, 0, 0);
                code = __builtin_amdgcn_mfma_f32_32x32x2f32(mark, rare->seen >> i & 1u ? 1.0f : 0.0f, code, 0, 0, 0);
            }
            add_marks(sum, code);
            rare->o[b] = sum;
        }
    }

    static __device__ __forceinline__ int channel_of(int b, int i, int h) { return 32 * b + 8 * (i >> 2) + 4 * h + (i & 3); }
    static __device__ __forceinline__ void store4(int64_t to, f4 v) { *gout<f4>(to) = v; }
};

}  // namespace rch
