// Attention of single tokens over pools in 8-bit codes: a wave (and workgroup) to an item, whose rows (the query heads of a
// key head, at most 32) are one token's.
//
// Bound: memory, one byte of every key and value.  A tile of 32 keys and values travels as codes from memory to LDS
// directly, a tile ahead, in a ring that is the wave's own: no barrier, and several such waves to a CU keep enough bytes
// on their way.  The products are those of attend_tile.h (S^T = K Q^T, O^T += V^T P^T, 32 x 32 x 16); codes become 16-bit
// operands as they are read.  K: the inner index of the products may run over the channels in any order that K and Q share,
// so a lane reads 16 codes of its key at once, channels 32 c + 16 h .., and feeds two products.  V: a transposed read of
// 8-bit values gives a lane eight keys of its channel, in the order that the weights' registers hold them.
// All rows see the same keys: a key that they do not see gets no weight, and its codes and scale are zeroed in LDS, so that
// it may be anything; the tile's loads may repeat a valid row where there is none.
//
// Measured: 4 tokens of 32 query heads over 20000 to 65536 keys of 8 heads of 128 channels in int8, 65 us at 5.2 TB/s (a large
// copy reaches 4.8, reads alone 5.4), and 11 of the join; the row tiles of attend_rows.h took 94 in all, since 128 rows of
// which 4 are there convert every value in full for them.
#pragma once

#include "attend_tile.h"
#include "codes.h"

namespace rch {

// LDS layout of a tile of codes: rows of RB bytes, 16-byte pieces exchanged so that reads meet no bank twice.
template <int NB>
struct CodeTile {
    static constexpr int KT = 32, RB = NB <= 2 ? 64 : NB <= 4 ? 128 : 256, kPieces = RB / 16, kRows = 1024 / RB, NI = KT / kRows;
    static constexpr int kBytes = 2 * KT * RB + 2 * KT * 4;  // keys, values, scales of both
    // Rows of one 256-byte line of the banks share no piece: K is read 16 rows at a piece.
    static __device__ __forceinline__ int k_swizzle(int row) { return row / (256 / RB) % kPieces; }
    // V is read keys {0..3, 8..11} + 4 h of 16 at two neighbouring pieces.
    static __device__ __forceinline__ int v_swizzle(int row) {
        if constexpr (RB == 64) return 2 * ((row >> 3) & 1);
        else if constexpr (RB == 128) return 2 * (((row >> 1) & 1) | ((row >> 2) & 2));
        else return 2 * ((row & 3) | ((row >> 1) & 4));
    }
};

// 16 bytes a lane from a wave-uniform address plus the lane's offset to LDS at `lds` + 16 * lane, and 4 bytes a lane from
// the lane's own address to `lds` + 4 * lane; not waited for (see fetch_buffer).
__device__ __forceinline__ void fetch_rows(int64_t base, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ void fetch_words(int64_t address, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds), "v"(address) : "memory", "m0");
}
__device__ __forceinline__ int64_t uniform64(int64_t x) {
    const uint32_t low = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x)), high = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x >> 32));
    return static_cast<int64_t>(static_cast<uint64_t>(high) << 32 | low);
}

template <int DT, int NB, int MODE, int FMT>
__global__ void __launch_bounds__(64, NB <= 2 ? 3 : NB <= 4 ? 2 : 1) attend_single_kernel(const rch_attend A) {
    typedef Half<DT> H;
    typedef typename H::type T;
    typedef typename H::vec8 vec8;
    typedef CodeTile<NB> Tile;
    typedef RowTile<DT, NB, 1> Layout;  // of the output
    constexpr int KT = Tile::KT, RB = Tile::RB, NI = Tile::NI, kPieces = Tile::kPieces, kRows = Tile::kRows;
    constexpr int kStages = 2, kLoads = 2 * NI + 1;  // of a tile
    __shared__ __attribute__((aligned(1024))) char lds[kStages * Tile::kBytes];
    const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
    const AttendItem I = attend_item(A, blockIdx.x);
    if (I.row_begin >= I.row_end) return;  // a plan's filling
    const QueryRow R = query_row(A, I, I.row_begin + n);
    const int row_first = __builtin_amdgcn_readfirstlane(R.first), row_last = __builtin_amdgcn_readfirstlane(R.last);
    const float scale = __int_as_float(static_cast<int>(A.scale_bits));

    Reference reference;
    reference.init();
    float sum = 0.0f;

    KeyWalk<KT, MODE, true> walk;
    walk.begin(A, I, 1);
    // The lane's place in a load: its row among kRows, and the channel piece that belongs there (behind the head's channels:
    // its first piece, where Q is 0).
    const int pieces = static_cast<int>(A.head_dim) / 16, row0 = lane / kPieces, spot = lane % kPieces;
    const uint32_t k_row = static_cast<uint32_t>(A.k_token_stride), v_row = static_cast<uint32_t>(A.v_token_stride);
    const int size = static_cast<int>(A.page_tokens);
    const bool of_values = h != 0;  // the scale that the lane fetches: of key or value n
    const int64_t scale_head = of_values ? A.v_scale_ptr + 4 * I.kv_head * A.v_scale_head_stride : A.k_scale_ptr + 4 * I.kv_head * A.k_scale_head_stride;
    const int64_t scale_page = 4 * (of_values ? A.v_scale_page_stride : A.k_scale_page_stride);
    uint32_t k_at[MODE == kRow ? 1 : NI], v_at[MODE == kRow ? 1 : NI];  // the lane's byte offsets in a tile of one page
    if constexpr (MODE != kRow) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int row = i * kRows + row0, kc = spot ^ Tile::k_swizzle(row), vc = spot ^ Tile::v_swizzle(row);
            k_at[i] = row * k_row + (kc < pieces ? kc * 16 : 0);
            v_at[i] = row * v_row + (vc < pieces ? vc * 16 : 0);
        }
    }
    const uint32_t ring = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((lds_char*)lds));

    // Tiles on their way, the oldest first: first key, and the keys that the rows see (bits).
    int pending = 0, stage = 0;
    uint32_t seen[kStages - 1];
    auto issue = [&](int to) -> uint32_t {
        const int base = walk.base, count = walk.count();
        const uint32_t at = ring + to * Tile::kBytes;
        uint64_t bits = row_first - base >= 32 || row_last <= base ? 0 : ~uint64_t{0} << max(row_first - base, 0);
        const int last = min(row_last - base, count);
        if (last < 32) bits &= (uint64_t{1} << max(last, 0)) - 1;
        uint32_t shown = static_cast<uint32_t>(bits);
        if constexpr (MODE == kPage || MODE == kList) {
            const int64_t k = uniform64(walk.k), v = uniform64(walk.v);
            if (count == KT) {
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    fetch_rows(k, k_at[i], at + i * 1024);
                    fetch_rows(v, v_at[i], at + KT * RB + i * 1024);
                }
            } else {
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    const int row = i * kRows + row0, back = max(row - (count - 1), 0);  // rows to the last one
                    fetch_rows(k, k_at[i] - back * k_row, at + i * 1024);
                    fetch_rows(v, v_at[i] - back * v_row, at + KT * RB + i * 1024);
                }
            }
            fetch_words(scale_head + walk.id * scale_page + 4 * static_cast<int64_t>(walk.in_page + min(n, count - 1)), at + 2 * KT * RB);
        } else {
            // Rows of several pages.  A row without a key takes the last one, one of a dropped page a row of page 0.
            const int page0 = base / size, off0 = base - page0 * size;
            auto place = [&](int row, int& id, int& in_page) {
                const int x = off0 + min(row, count - 1), page = x / size;
                in_page = x - page * size;
                id = page_entry(walk.table, page0 + page);
                return id >= 0 && id < walk.pages;
            };
            int id, in_page;
            const bool held = place(n, id, in_page);
            shown &= static_cast<uint32_t>(__ballot(held));
            const int64_t scales = scale_head + (held ? id : 0) * scale_page + 4 * static_cast<int64_t>(in_page);
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int row = i * kRows + row0;
                // The lane that looked this row's place up holds it.
                const int rid = __shfl(held ? id : 0, row), rin = __shfl(in_page, row);
                const int kc = spot ^ Tile::k_swizzle(row), vc = spot ^ Tile::v_swizzle(row);
                fetch_global(walk.k_head + rid * walk.k_page + rin * static_cast<int64_t>(k_row) + (kc < pieces ? kc * 16 : 0), at + i * 1024);
                fetch_global(walk.v_head + rid * walk.v_page + rin * static_cast<int64_t>(v_row) + (vc < pieces ? vc * 16 : 0), at + KT * RB + i * 1024);
            }
            fetch_words(scales, at + 2 * KT * RB);
        }
        walk.next();
        return shown;
    };
#pragma unroll
    for (int s = 0; s < kStages - 1; ++s)
        if (!walk.done()) seen[s] = issue(s), ++pending;

    // Q: product 2 c + e takes channels 32 c + 16 h + 8 e ...
    vec8 q[2 * NB];
    f16v o[NB];
    {  // (after the first tiles' loads; waited for before the loop, where a wait for them would be one for every tile's)
        const int64_t at = A.q_ptr + 2 * ((I.q_row + R.token) * A.q_token_stride + R.head * A.q_head_stride);
#pragma unroll
        for (int c = 0; c < 2 * NB; ++c) {
            const int d = 32 * (c >> 1) + 16 * h + 8 * (c & 1);
            q[c] = __builtin_bit_cast(vec8, *gin<u4>(R.valid && d < A.head_dim ? at + 2 * d : A.plan_ptr));  // or zeros
        }
#pragma unroll
        for (int b = 0; b < NB; ++b) o[b] = f16v{};
    }
    wait_vector_memory();

    // A lane's offsets within a tile: of its key's codes at piece h (piece 2 c + h from there by an exclusive or), and of the
    // transposed read of channel block 0 for the first 16 keys.
    const uint32_t k_lane = n * RB, k_turn = static_cast<uint32_t>(Tile::k_swizzle(n) ^ h) * 16;
    const int p = lane & 15, v_key = 4 * h + ((p >> 1) & 3) + 8 * (p >> 3);
    const uint32_t v_lane = v_key * RB + (p & 1) * 8, v_turn = static_cast<uint32_t>(Tile::v_swizzle(v_key) ^ ((lane >> 4) & 1)) * 16;

    while (pending > 0) {
        // The oldest tile has landed, and its ring's next place is read no more.
        if (pending == kStages - 1) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((kStages - 2) * kLoads) : "memory");
        else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        const uint32_t shown = seen[0];
#pragma unroll
        for (int s = 0; s + 2 < kStages; ++s) seen[s] = seen[s + 1];
        const int here = stage, there = stage >= 1 ? stage - 1 : kStages - 1;
        stage = stage + 1 == kStages ? 0 : stage + 1;
        --pending;
        if (!walk.done()) {
            const uint32_t next = issue(there);
#pragma unroll
            for (int s = 0; s < kStages - 1; ++s) seen[s] = s == pending ? next : seen[s];
            ++pending;
        }
        lds_char* const k_tile = (lds_char*)lds + here * Tile::kBytes;
        lds_char* const v_tile = k_tile + KT * RB;
        typedef __attribute__((address_space(3))) float lds_float;
        typedef __attribute__((address_space(3))) f4 lds_f4;
        typedef __attribute__((address_space(3))) u4 lds_u4;
        lds_float* const scales = (lds_float*)(k_tile + 2 * KT * RB);
        if (shown == 0) continue;
        // 8-bit floats in bf16: the values' scales, powers of two, go to the weights, whose rounding stays what it is while the
        // products are far from bf16's subnormals and its end (a weight of 2^-17 and a scale of 2^-115 would keep two bits).
        // Scales below 2^-64 and above 2^64 go there by what they differ from 2^-95 and 2^95, in products of their own whose
        // values take the rest: no product is below 2^-64 of its weight, or more than 2^64 of it.  fp16 does not hold such
        // weights, and integers times other scales are rounded as values.
        constexpr bool kScaled = DT == RCH_DT_BF16 && FMT == RCH_CODES_E4M3;
        float own = 0.0f;
        uint64_t small = 0, large = 0;  // keys of such scales (bits of the lanes that fetched them)
        if constexpr (FMT == RCH_CODES_E4M3) {
            own = code_scale<FMT>(scales[lane]);
            bool apart = false;
            if constexpr (kScaled) {
                const bool counts = of_values && (shown >> n & 1u), low = counts && own < 0x1p-64f, high = counts && own > 0x1p64f;
                small = __ballot(low);
                large = __ballot(high);
                apart = low || high;
            }
            scales[lane] = apart ? 0.0f : own;
        }
        if (shown != ~0u) {
#pragma unroll
            for (int i = 0; i < NI; ++i)
                if (!(shown >> (i * kRows + row0) & 1u)) *(lds_u4*)(v_tile + i * 1024 + lane * 16) = u4{};
            if (of_values && !(shown >> n & 1u)) scales[lane] = 0.0f;
        }
        const float k_scale = scales[n];
        f16v s[1] = {f16v{}};
#pragma unroll
        for (int c = 0; c < NB; ++c) {
            const u4 codes = *(lds_u4*)(k_tile + k_lane + (k_turn ^ (c * 32)));
            s[0] = H::mfma(code_values<DT, FMT>(codes[0], codes[1], k_scale), q[2 * c], s[0]);
            s[0] = H::mfma(code_values<DT, FMT>(codes[2], codes[3], k_scale), q[2 * c + 1], s[0]);
        }
        if (shown != ~0u) {
            const uint32_t w = shown >> (4 * h), bits = (w & 0xfu) | (w >> 4 & 0xf0u) | (w >> 8 & 0xf00u) | (w >> 12 & 0xf000u);
#pragma unroll
            for (int i = 0; i < 16; ++i) s[0][i] = bits >> i & 1u ? s[0][i] : -INFINITY;
        }
        float top = s[0][0];
#pragma unroll
        for (int i = 1; i < 16; ++i) top = fmaxf(top, s[0][i]);
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
        f4 v_scale[4];  // of the keys of registers 4 i ..
#pragma unroll
        for (int i = 0; i < 4; ++i) v_scale[i] = *(lds_f4*)(scales + 32 + 8 * i + 4 * h);
        vec8 w[2];
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float x = exp2_of(__builtin_fmaf(s[0][i], scale, -reference.value));
            part[i & 3] += x;
            w[i >> 3][i & 7] = static_cast<T>(kScaled ? x * v_scale[i >> 2][i & 3] : x);
            if constexpr (kScaled) s[0][i] = x;
        }
        sum += (part[0] + part[1]) + (part[2] + part[3]);
        auto add_values = [&](float unit) {  // unit: what the values' own scale is, where the weights take the rest of it
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    typedef int i2 __attribute__((ext_vector_type(2)));
                    typedef __attribute__((address_space(3))) i2 lds_i2;
                    const i2 codes = __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i2*)(v_tile + v_lane + half * 16 * RB + (v_turn ^ (b * 32))));
                    const uint32_t low = static_cast<uint32_t>(codes[0]), high = static_cast<uint32_t>(codes[1]);
                    if constexpr (kScaled) o[b] = H::mfma(code_values<DT, FMT>(low, high, unit), w[half], o[b]);
                    else o[b] = H::mfma(code_values<DT, FMT>(low, high, v_scale[2 * half], v_scale[2 * half + 1]), w[half], o[b]);
                }
            }
        };
        add_values(1.0f);
        if constexpr (kScaled) {
            while (__builtin_expect((small | large) != 0, 0)) {
                const uint64_t these = small ? small : large;
                const float unit = small ? 0x1p-95f : 0x1p95f, rest = small ? 0x1p95f : 0x1p-95f;
                if (small) small = 0;
                else large = 0;
                scales[lane] = these >> lane & 1u ? own * rest : 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) v_scale[i] = *(lds_f4*)(scales + 32 + 8 * i + 4 * h);
#pragma unroll
                for (int i = 0; i < 16; ++i) w[i >> 3][i & 7] = static_cast<T>(s[0][i] * v_scale[i >> 2][i & 3]);
                add_values(unit);
            }
        }
    }

    if (!R.valid) return;
    const int row = I.row_begin + n;
    sum = row_sum(sum);
    bool blank = false;
    if (sum == 0.0f) {
        const int per = (static_cast<int>(A.block_tokens) + KT - 1) / KT;
        if constexpr (MODE == kList) blank = sees_any_listed(A, I, R.first, R.last, I.key_begin / per, (I.key_end + per - 1) / per);
        else blank = sees_any(A, I, R.first, R.last);
    }
    if (I.part >= 0) {
        const int64_t at = I.part + row - I.row_begin, to = partial_sums(A, at);
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int d = Layout::channel_of(b, i, h);
                if (d < A.head_dim) *gout<f4>(to + 4 * d) = f4{o[b][i], o[b][i + 1], o[b][i + 2], o[b][i + 3]};
            }
        if (h == 0) *gout<f2>(partial_stats(A, at)) = f2{part_reference(reference.whole(scale), sum, blank), sum};
        return;
    }
    const float inverse = row_factor(sum, blank);
    const int64_t to = A.out_ptr + 2 * ((I.q_row + R.token) * A.out_token_stride + R.head * A.out_head_stride);
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int d = Layout::channel_of(b, i, h);
            if (d < A.head_dim) Layout::store4(to + 2 * d, f4{o[b][i] * inverse, o[b][i + 1] * inverse, o[b][i + 2] * inverse, o[b][i + 3] * inverse});
        }
    if (h == 0 && A.lse_ptr) gout<float>(A.lse_ptr)[(I.q_row + R.token) * A.heads + R.head] = row_lse(reference.whole(scale), sum);
}

}  // namespace rch
