// New tokens into the 8-bit pages of a cache, and back.
//
// A token's head of D values x (keys rotated first, in fp32) gets one scale s from m = max |x|, and D codes:
//   int8: s = max(m / 127, 2^-126), c = rint(x (1 / s)): off by at most (1/2 + 2^-15) s (the reciprocal and the product
//         are rounded: 127 (3/2) 2^-23 of a step)
//   e4m3: s = 2^e with m <= 448 s (exact), c = x / s to 4 bits of mantissa: off by 2^-4 of x, or 2^-10 s of small ones
// A code stands for c s, rounded once to the cache's type (e4m3: exact in bf16).  The scale is a row's own, so a token is
// quantised as it is written and never again, and a row that holds an infinity or a NaN harms no other: its scale is NaN.
//
// Bound: memory, 2 bytes read and 1 written of each value (or the reverse), 4 bytes of scale to a row.  A row lies in 8,
// 16 or 32 lanes with eight channels each (a wave's row maxima meet by lane moves, no LDS), and a thread holds that
// piece of four heads, so that the places and cosines are fetched once for them.  Measured: a chunk of 4680 tokens of 12 heads
// of 128 bf16 channels stored (rotated) as int8 in 14 us (43 MB, 3 TB/s: 9 us of bytes, 6 of instructions, and the chain place, angles, store), read
// back in 11.5; a history of 32760 tokens read from e4m3 in 55 us into the same outputs over and over (302 MB, 5.5 TB/s), in 67
// where every call has other pages and new outputs.
#include "codes.h"
#include "turn.h"

namespace rch {

namespace {

// Heads of a thread: 32760 tokens of 12 heads of 128 channels are read in 57.5 / 56.6 / 59.6 / 61.5 us with 1 / 2 / 3 / 4 of
// them (more bytes than the caches hold, so short threads), 4680 tokens stored and read back in 23.5 / 22.9 / 23.1 / 23.4 us
// with 2 / 3 / 4 / 6.
constexpr int kHeads = 4, kHeadsRead = 2;

// One side (K or V) of the arguments.
struct Side {
    int64_t dense, token, head, codes, page, row, codes_head, scales, scale_page, scale_head;
};
__device__ __forceinline__ Side side_of(const rch_codes& A, bool values) {
    if (values)
        return {A.v_ptr, A.v_token_stride, A.v_head_stride, A.v_codes_ptr, A.v_page_stride, A.v_row_stride, A.v_codes_head_stride,
                A.v_scales_ptr, A.v_scale_page_stride, A.v_scale_head_stride};
    return {A.k_ptr, A.k_token_stride, A.k_head_stride, A.k_codes_ptr, A.k_page_stride, A.k_row_stride, A.k_codes_head_stride,
            A.k_scales_ptr, A.k_scale_page_stride, A.k_scale_head_stride};
}

template <int CONTROL>
__device__ __forceinline__ uint32_t moved(uint32_t x) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CONTROL, 0xf, 0xf, true));
}
// The largest of L neighbouring lanes, in each of them.
template <int L>
__device__ __forceinline__ uint32_t largest(uint32_t x) {
    x = max(x, moved<0xb1>(x));   // lanes 1 0 3 2
    x = max(x, moved<0x4e>(x));   // lanes 2 3 0 1
    x = max(x, moved<0x141>(x));  // mirrored in 8
    if constexpr (L >= 16) x = max(x, moved<0x140>(x));  // mirrored in 16
    if constexpr (L >= 32) x = max(x, static_cast<uint32_t>(__shfl_xor(static_cast<int>(x), 16)));
    if constexpr (L >= 64) x = max(x, static_cast<uint32_t>(__shfl_xor(static_cast<int>(x), 32)));
    return x;
}

// A head's scale and its reciprocal, from the bits of its largest magnitude (infinities and NaN are above all others).
struct Scale {
    float scale, inverse, limit;  // limit: the largest code
};
template <int DT, int FMT>
__device__ __forceinline__ Scale scale_of(uint32_t bits) {
    const float most = __uint_as_float(bits);
    if (bits >= 0x7f800000u) return {__builtin_nanf(""), 0.0f, 0.0f};
    if constexpr (FMT == RCH_CODES_INT8) {
        const float scale = fmaxf(__fdiv_rn(most, 127.0f), 1.17549435e-38f);
        return {scale, __fdiv_rn(1.0f, scale), 127.0f};
    } else {
        // most = f 2^x with f in [1, 2): the least e with most <= 1.75 2^8 2^e (0 and subnormals: the least of all).
        const int x = static_cast<int>(bits >> 23) - 127;
        const int e = max(x - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), -126);
        // Where a code of 256 stands for more than the type holds, the largest values are rounded down, not to infinity.
        return {pow2f(e), pow2f(-e), e >= (DT == RCH_DT_F16 ? 8 : 120) ? 240.0f : 448.0f};
    }
}

// Codes of four values.  int8: no product is above 127 (1 + 2^-22), which rounds to 127, and a sum with 1.5 2^23 is rounded
// to an integer whose low byte is the code.
template <int FMT>
__device__ __forceinline__ uint32_t encode(f4 x, const Scale& scale) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __fmul_rn(x[i], scale.inverse);
    if constexpr (FMT == RCH_CODES_INT8) {
        uint32_t y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = __float_as_uint(__fadd_rn(x[i], 12582912.0f));
        const uint32_t low = __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0400u), high = __builtin_amdgcn_perm(y[3], y[2], 0x04000c0cu);
        return low | high;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = __builtin_amdgcn_fmed3f(x[i], -scale.limit, scale.limit);
        const int word = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
        return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], word, true));
    }
}

// V channels of a head in a lane, L lanes to a head.  V = 8 needs rows of whole aligned pieces; V = 4 (L = 64) takes every
// other head size and alignment, element by element.
template <int DT, int FMT, int V, int L>
__global__ void __launch_bounds__(256) codes_store_kernel(const rch_codes A) {
    typedef typename Coded<DT>::type T;
    const bool values = blockIdx.z != 0;
    const Side S = side_of(A, values);
    const int dim = static_cast<int>(A.head_dim), pairs = values ? 0 : static_cast<int>(A.pairs);
    const int64_t token = static_cast<int64_t>(blockIdx.x) * (256 / L) + threadIdx.x / L;
    const int lane = threadIdx.x % L, first = lane * V, head0 = blockIdx.y * kHeads;
    const int heads = min(static_cast<int>(A.heads) - head0, kHeads);
    const bool live = token < A.tokens, mine = live && first < dim;
    int slot = -1;
    if (live) slot = gin<int32_t>(A.slots_ptr)[token];
    const uint32_t page_tokens = static_cast<uint32_t>(A.page_tokens);
    const bool kept = slot >= 0 && static_cast<uint32_t>(slot) < static_cast<uint32_t>(A.pages) * page_tokens;  // a slot outside the pool (padding) drops the token

    float x[kHeads][V];
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
#pragma unroll
        for (int i = 0; i < V; ++i) x[u][i] = 0.0f;
        if (!mine || u >= heads) continue;
        const RCH_GLOBAL T* from = gin<T>(S.dense) + token * S.token + (head0 + u) * S.head + first;
        if constexpr (V == 8) {
            typedef T t8 __attribute__((ext_vector_type(8)));
            const t8 raw = __builtin_bit_cast(t8, *reinterpret_cast<const RCH_GLOBAL u4*>(from));
#pragma unroll
            for (int i = 0; i < V; ++i) x[u][i] = static_cast<float>(raw[i]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (first + i < dim) x[u][i] = static_cast<float>(from[i]);
        }
    }
    if (pairs && mine && first < 2 * pairs) {
        const TurningRows row = turning_rows(A, 0, token);
        f2 angle[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            angle[i] = f2{1.0f, 0.0f};
            if (first / 2 + i < pairs) angle[i] = turning_angle(A, row, first / 2 + i, pairs);
        }
#pragma unroll
        for (int u = 0; u < kHeads; ++u)
#pragma unroll
            for (int i = 0; i < V / 2; ++i)
                if (first / 2 + i < pairs) rotate_pair(x[u][2 * i], x[u][2 * i + 1], angle[i][0], angle[i][1]);
    }
    const uint32_t at = kept ? static_cast<uint32_t>(slot) : 0u, page_at = at / page_tokens;  // (of 32 bits: quotients of 64 take ten times as long)
    const int64_t page = page_at, in_page = at - page_at * page_tokens;
#pragma unroll
    for (int u = 0; u < kHeads; ++u) {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) most = max(most, __float_as_uint(x[u][i]) & 0x7fffffffu);
        most = largest<L>(most);
        if (!kept || u >= heads) continue;
        const Scale scale = scale_of<DT, FMT>(most);
        if (lane == 0)
            gout<float>(S.scales)[page * S.scale_page + (head0 + u) * S.scale_head + in_page] = scale.scale;
        if (!mine) continue;
        const bool finite = most < 0x7f800000u;
        uint32_t word[V / 4];
#pragma unroll
        for (int w = 0; w < V / 4; ++w)
            word[w] = finite ? encode<FMT>(f4{x[u][4 * w], x[u][4 * w + 1], x[u][4 * w + 2], x[u][4 * w + 3]}, scale) : 0;
        const int64_t to = S.codes + page * S.page + in_page * S.row + (head0 + u) * S.codes_head + first;
        if constexpr (V == 8) {
            *gout<u2>(to) = u2{word[0], word[1]};
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (first + i < dim) gout<uint8_t>(to)[i] = static_cast<uint8_t>(word[i / 4] >> (8 * (i % 4)));
        }
    }
}

// V channels to a thread: 16 of aligned rows, or one.
template <int DT, int FMT, int V>
__global__ void __launch_bounds__(256) codes_read_kernel(const rch_codes A) {
    typedef typename Coded<DT>::type T;
    const Side S = side_of(A, blockIdx.z != 0);
    const uint32_t pieces = static_cast<uint32_t>(A.head_dim) / V, unit = blockIdx.x * 256 + threadIdx.x, row = unit / pieces;
    const int64_t token = row;
    const int first = static_cast<int>(unit - row * pieces) * V, head0 = blockIdx.y * kHeadsRead;
    if (token >= A.tokens) return;
    const int heads = min(static_cast<int>(A.heads) - head0, kHeadsRead);
    const int slot = gin<int32_t>(A.slots_ptr)[token];
    const uint32_t page_tokens = static_cast<uint32_t>(A.page_tokens);
    const bool kept = slot >= 0 && static_cast<uint32_t>(slot) < static_cast<uint32_t>(A.pages) * page_tokens;
    const uint32_t at = kept ? static_cast<uint32_t>(slot) : 0u, page_at = at / page_tokens;
    const int64_t page = page_at, in_page = at - page_at * page_tokens;
    const int64_t codes = S.codes + page * S.page + in_page * S.row + head0 * S.codes_head + first;
    const int64_t scales = S.scales + 4 * (page * S.scale_page + head0 * S.scale_head + in_page);
    RCH_GLOBAL T* to = gout<T>(S.dense) + token * S.token + head0 * S.head + first;
    float scale[kHeadsRead];
    u4 raw[kHeadsRead];
#pragma unroll
    for (int u = 0; u < kHeadsRead; ++u) {
        const int h = min(u, heads - 1);
        scale[u] = kept ? gin<float>(scales)[h * S.scale_head] : __builtin_nanf("");
        if constexpr (V == 16) raw[u] = kept ? *gin<u4>(codes + h * S.codes_head) : u4{};
        else raw[u] = u4{kept ? gin<uint8_t>(codes)[h * S.codes_head] : 0u, 0u, 0u, 0u};
    }
#pragma unroll
    for (int u = 0; u < kHeadsRead; ++u) {
        if (u >= heads) break;
        if constexpr (V == 16) {
            RCH_GLOBAL u4* whole = reinterpret_cast<RCH_GLOBAL u4*>(to + u * S.head);
            whole[0] = __builtin_bit_cast(u4, code_values<DT, FMT>(raw[u][0], raw[u][1], scale[u]));
            whole[1] = __builtin_bit_cast(u4, code_values<DT, FMT>(raw[u][2], raw[u][3], scale[u]));
        } else {
            to[u * S.head] = code_value<DT, FMT>(static_cast<uint8_t>(raw[u][0]), scale[u]);
        }
    }
}

int invalid(const rch_codes& A, int dtype, const char* what) {
    if (dtype != RCH_DT_F16 && dtype != RCH_DT_BF16) return fail(RCH_E_UNSUPPORTED, "%s: codes stand for f16 or bf16 values", what);
    if (A.format != RCH_CODES_INT8 && A.format != RCH_CODES_E4M3) return fail(RCH_E_CONFIG, "%s: unknown format of codes", what);
    if (A.tokens < 0 || A.heads < 1 || A.head_dim < 1 || A.pages < 1 || A.page_tokens < 1 || A.tokens > 0x7fffffff
        || A.heads > kHeadsRead * 65535 || A.pages > 0x7fffffff || A.page_tokens > 0x7fffffff || A.pages * A.page_tokens > 0x7fffffff)
        return fail(RCH_E_CONFIG, "%s: invalid sizes", what);
    if (A.head_dim > RCH_CODES_MAX_DIM) return fail(RCH_E_UNSUPPORTED, "%s: heads of at most %d channels", what, RCH_CODES_MAX_DIM);
    if (A.pairs < 0 || 2 * A.pairs > A.head_dim
        || (A.pairs && ((A.axes != 1 && A.axes != 3) || !A.pairs_ptr || (!A.rows_ptr && A.axes == 3 && (A.grid_h < 1 || A.grid_w < 1)))))
        return fail(RCH_E_CONFIG, "%s: invalid positions", what);
    if (A.tokens && (!A.k_ptr || !A.v_ptr || !A.k_codes_ptr || !A.v_codes_ptr || !A.k_scales_ptr || !A.v_scales_ptr || !A.slots_ptr))
        return fail(RCH_E_CONFIG, "%s: null address", what);
    return RCH_OK;
}

// Whether rows of `piece` channels are aligned: 16 bytes of the dense tensors (or as many), a byte to a code.
bool aligned(const rch_codes& A, int64_t piece) {
    const int64_t dense = 2 * (A.k_token_stride | A.k_head_stride | A.v_token_stride | A.v_head_stride) | A.k_ptr | A.v_ptr;
    const int64_t codes = A.k_codes_ptr | A.v_codes_ptr | A.k_page_stride | A.k_row_stride | A.k_codes_head_stride
                          | A.v_page_stride | A.v_row_stride | A.v_codes_head_stride;
    return A.head_dim % piece == 0 && dense % 16 == 0 && codes % piece == 0;
}

// A grid of `units` threads (a launch has fewer than 2^32 along an axis).
bool grid_of(const rch_codes& A, int64_t units, int heads, dim3* grid) {
    *grid = dim3(static_cast<uint32_t>((units + 255) / 256), static_cast<uint32_t>((A.heads + heads - 1) / heads), 2);
    return units <= 0xffffff00ll;
}

template <int DT, int FMT, int V, int L>
int store(const rch_codes& A, hipStream_t stream) {
    dim3 grid;
    if (!grid_of(A, A.tokens * L, kHeads, &grid)) return fail(RCH_E_CONFIG, "rch_codes_store: too many tokens for one launch");
    hipLaunchKernelGGL((codes_store_kernel<DT, FMT, V, L>), grid, dim3(256), 0, stream, A);
    return check_launch("rch_codes_store");
}

template <int DT, int FMT>
int store_rows(const rch_codes& A, hipStream_t stream) {
    if (!aligned(A, 8)) return store<DT, FMT, 4, 64>(A, stream);
    if (A.head_dim <= 64) return store<DT, FMT, 8, 8>(A, stream);
    return A.head_dim <= 128 ? store<DT, FMT, 8, 16>(A, stream) : store<DT, FMT, 8, 32>(A, stream);
}

template <int DT, int FMT>
int read_rows(const rch_codes& A, hipStream_t stream) {
    const bool wide = aligned(A, 16);
    dim3 grid;
    if (!grid_of(A, A.tokens * (wide ? A.head_dim / 16 : A.head_dim), kHeadsRead, &grid)) return fail(RCH_E_CONFIG, "rch_codes_read: too many tokens for one launch");
    if (wide) hipLaunchKernelGGL((codes_read_kernel<DT, FMT, 16>), grid, dim3(256), 0, stream, A);
    else hipLaunchKernelGGL((codes_read_kernel<DT, FMT, 1>), grid, dim3(256), 0, stream, A);
    return check_launch("rch_codes_read");
}

}  // namespace

}  // namespace rch

extern "C" {

int rch_codes_size(void) { return static_cast<int>(sizeof(rch_codes)); }

int rch_codes_store(const rch_codes* args_host, int dtype, void* stream) {
    using namespace rch;
    if (!args_host) return fail(RCH_E_CONFIG, "rch_codes_store: no arguments");
    const rch_codes& A = *args_host;
    const int status = invalid(A, dtype, "rch_codes_store");
    if (status != RCH_OK || A.tokens == 0) return status;
    hipStream_t s = as_stream(stream);
    if (dtype == RCH_DT_F16)
        return A.format == RCH_CODES_INT8 ? store_rows<RCH_DT_F16, RCH_CODES_INT8>(A, s) : store_rows<RCH_DT_F16, RCH_CODES_E4M3>(A, s);
    return A.format == RCH_CODES_INT8 ? store_rows<RCH_DT_BF16, RCH_CODES_INT8>(A, s) : store_rows<RCH_DT_BF16, RCH_CODES_E4M3>(A, s);
}

int rch_codes_read(const rch_codes* args_host, int dtype, void* stream) {
    using namespace rch;
    if (!args_host) return fail(RCH_E_CONFIG, "rch_codes_read: no arguments");
    const rch_codes& A = *args_host;
    const int status = invalid(A, dtype, "rch_codes_read");
    if (status != RCH_OK || A.tokens == 0) return status;
    hipStream_t s = as_stream(stream);
    if (dtype == RCH_DT_F16)
        return A.format == RCH_CODES_INT8 ? read_rows<RCH_DT_F16, RCH_CODES_INT8>(A, s) : read_rows<RCH_DT_F16, RCH_CODES_E4M3>(A, s);
    return A.format == RCH_CODES_INT8 ? read_rows<RCH_DT_BF16, RCH_CODES_INT8>(A, s) : read_rows<RCH_DT_BF16, RCH_CODES_E4M3>(A, s);
}

}  // extern "C"
