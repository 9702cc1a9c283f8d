// Attention over a paged cache: the general form, the merge of partial results and the entry point.
//
// For a row q (a query token and head) over the keys it sees:
//   s_j = scale q.k_j,  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m >= max_j s_j roughly:
// any reference m gives the same quotient, so one pass over the keys keeps a running m, sum and
// weighted sum, all in fp32, and multiplies both sums by exp(m_old - m_new) where m moves.  Exponents
// are base 2 (scale carries log2 e).  Two parts of a row's keys join the same way.
//
// The general form takes every head_dim up to 256, alignment and element type: one wave per row, a
// lane per key for the scores, a lane per channel for the sums.  Bound by the latency of its loads, element
// by element: single tokens of 4 sequences of 4000 tokens, 16 heads of 250 bf16, take 450 us (0.57 TB/s).  Only
// pools, or head sizes, whose rows are no 16-byte pieces come here, and pools whose token rows lie more than 2^22
// elements apart; the form that tiles for the matrix cores (16 heads of 200: 80 us) is in attend_rows.hip.
#include "attend.h"

namespace rch {

namespace {

template <int DT>
__global__ void __launch_bounds__(256) attend_general_kernel(const rch_attend A) {
    typedef typename AttendType<DT>::type T;
    __shared__ float query[4][RCH_ATTEND_MAX_DIM];
    __shared__ float weight[4][64];
    __shared__ int64_t place_of[4][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const AttendItem I = attend_item(A, blockIdx.x);
    const int dim = static_cast<int>(A.head_dim), group = static_cast<int>(A.group);
    const float scale = __int_as_float(static_cast<int>(A.scale_bits));
    const int size = static_cast<int>(A.page_tokens);
    const RCH_GLOBAL int32_t* table = gin<int32_t>(A.plan_ptr) + I.table;
    const int64_t k_head = I.kv_head * A.k_head_stride, v_head = I.kv_head * A.v_head_stride;

    for (int row = I.row_begin + wave; row < I.row_end; row += 4) {
        const int token = row / group, head = I.kv_head * group + row % group;
        int begin, end;
        attend_range(A, I, token, begin, end);
        const int from = begin > I.key_begin ? begin : I.key_begin, to = end < I.key_end ? end : I.key_end;
        const RCH_GLOBAL T* q = gin<T>(A.q_ptr) + (I.q_row + token) * A.q_token_stride + head * A.q_head_stride;
        __builtin_amdgcn_wave_barrier();
        for (int d = lane; d < dim; d += 64) query[wave][d] = static_cast<float>(q[d]);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        float reference = kNoReference, sum = 0.0f, acc[RCH_ATTEND_MAX_DIM / 64];
        bool blank = false;  // a key was seen
#pragma unroll
        for (int c = 0; c < RCH_ATTEND_MAX_DIM / 64; ++c) acc[c] = 0.0f;
        for (int base = from; base < to; base += 64) {
            const int key = base + lane;
            bool seen = key < to;
            int page = -1;
            if (seen) page = table[key / size];
            seen = seen && page >= 0 && page < A.pages;
            const int in_page = key % size;
            float score = -INFINITY;
            if (seen) {
                const RCH_GLOBAL T* k = gin<T>(A.k_ptr) + page * A.k_page_stride + in_page * A.k_token_stride + k_head;
                float dot = 0.0f;
                for (int d = 0; d < dim; ++d) dot = __builtin_fmaf(query[wave][d], static_cast<float>(k[d]), dot);
                score = dot * scale;
            }
            uint64_t left = __ballot(seen);
            if (left == 0) continue;
            blank = true;
            float top = score;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
            const float next = fmaxf(reference, top), fade = exp2_of(reference - next);
            reference = next;
            const float w = seen ? exp2_of(score - next) : 0.0f;
            float total = w;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) total += __shfl_xor(total, o);
            sum = __builtin_fmaf(sum, fade, total);
            __builtin_amdgcn_wave_barrier();
            weight[wave][lane] = w;
            place_of[wave][lane] = page * A.v_page_stride + in_page * A.v_token_stride + v_head;
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int c = 0; c < RCH_ATTEND_MAX_DIM / 64; ++c) acc[c] *= fade;
            while (left) {  // only keys that the row sees: the others' values may be anything
                const int j = __builtin_ctzll(left);
                left &= left - 1;
                const float wj = weight[wave][j];
                const RCH_GLOBAL T* v = gin<T>(A.v_ptr) + place_of[wave][j];
#pragma unroll
                for (int c = 0; c < RCH_ATTEND_MAX_DIM / 64; ++c)
                    if (lane + 64 * c < dim) acc[c] = __builtin_fmaf(wj, static_cast<float>(v[lane + 64 * c]), acc[c]);
            }
        }
        if (I.part >= 0) {
            const int64_t at = I.part + row - I.row_begin;
#pragma unroll
            for (int c = 0; c < RCH_ATTEND_MAX_DIM / 64; ++c)
                if (lane + 64 * c < dim) gout<float>(partial_sums(A, at))[lane + 64 * c] = acc[c];
            if (lane == 0) *gout<f2>(partial_stats(A, at)) = f2{part_reference(reference, sum, blank), sum};
            continue;
        }
        RCH_GLOBAL T* out = gout<T>(A.out_ptr) + (I.q_row + token) * A.out_token_stride + head * A.out_head_stride;
        const float inverse = row_factor(sum, blank);
#pragma unroll
        for (int c = 0; c < RCH_ATTEND_MAX_DIM / 64; ++c)
            if (lane + 64 * c < dim) out[lane + 64 * c] = static_cast<T>(acc[c] * inverse);
        if (lane == 0 && A.lse_ptr) gout<float>(A.lse_ptr)[(I.q_row + token) * A.heads + head] = row_lse(reference, sum);
    }
}

// Joins the parts of rows whose keys were split (the same order whatever the timing).  Bound: the latency of
// the partial results (other XCDs wrote them), so all or many of a row's loads are in flight at once.  Rows of
// more than kFewParts parts (single tokens over long histories), or of a step with few, take a workgroup each, whose
// waves share the parts; the others a thread per eight channels.  Rows of 128 channels: 228 blocks of 128 rows in 3 and 7 parts
// take 10.4 us so and 43 us with a workgroup each (29184 workgroups); 32 blocks of 4 rows in 11 or 16 parts 4.0 us
// with a workgroup each and, with a thread per eight channels over groups of 8 parts, 5.8 and 7.4 us.
// A workgroup has 16 waves where at most kWideRows rows are joined (8 rows in 159 parts: 7.2 us, with 4 waves
// 14.9 us; 32 rows in 32 parts: 4.6, 5.0 us), else 4 (128 rows in 16 parts: 4.0 us, with 16 waves 4.4 us; 2048
// rows in 16 parts: 6.5, 19.5 us).
constexpr int kFewParts = RCH_ATTEND_FEW_PARTS, kWideRows = 64;

struct MergedRow {
    int64_t out, lse;  // element offsets of the row's output and logarithm
};
__device__ __forceinline__ MergedRow merged_row(const rch_attend& A, int q_row, int row, int kv_head) {
    const int group = static_cast<int>(A.group), token = row / group, head = kv_head * group + row - token * group;
    return {(q_row + token) * A.out_token_stride + head * A.out_head_stride, (q_row + token) * A.heads + head};
}

template <int DT, int C, int W>
__global__ void __launch_bounds__(64 * W) attend_merge_many_kernel(const rch_attend A) {
    typedef typename AttendType<DT>::type T;
    constexpr int kAhead = 32 / C;  // parts in flight in a wave
    __shared__ float sums[W][64 * C], stat[W][2];
    const RCH_GLOBAL int32_t* w = gin<int32_t>(A.plan_ptr) + A.merges + static_cast<int64_t>(blockIdx.x) * RCH_ATTEND_MERGE;
    const int rows = w[2], parts = w[5], dim = static_cast<int>(A.head_dim), r = blockIdx.y;
    if (r >= rows) return;
    const int64_t first = static_cast<int64_t>(w[4]) + r;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // A wave takes parts wave, wave + W, ..: its own reference, sum and weighted sums.
    float reference = kNoReference, sum = 0.0f, acc[C];
    bool blank = false;
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = 0.0f;
    for (int base = wave; base < parts; base += 64 * W) {
        const int part = base + W * lane;
        f2 stats = {kNoReference, 0.0f};
        if (part < parts) stats = *gin<f2>(partial_stats(A, first + static_cast<int64_t>(part) * rows));
        blank = blank || part_blank(stats[0], stats[1]);
        float next = stats[1] != 0.0f ? stats[0] : kNoReference;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) next = fmaxf(next, __shfl_xor(next, o));
        next = fmaxf(next, reference);
        const float old = exp2_of(reference - next), mine = stats[1] != 0.0f ? exp2_of(stats[0] - next) : 0.0f;
        reference = next;
        float total = stats[1] * mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) total += __shfl_xor(total, o);
        sum = __builtin_fmaf(sum, old, total);
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] *= old;
        const int count = min(64, (parts - base + W - 1) / W);
        for (int p0 = 0; p0 < count; p0 += kAhead) {
            float x[kAhead][C];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int p = min(p0 + i, count - 1);
                const RCH_GLOBAL float* from = gin<float>(partial_sums(A, first + static_cast<int64_t>(base + W * p) * rows));
#pragma unroll
                for (int c = 0; c < C; ++c) x[i][c] = from[min(lane + 64 * c, dim - 1)];
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (p0 + i >= count) break;
                const float fade = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(mine), p0 + i));
#pragma unroll
                for (int c = 0; c < C; ++c) acc[c] = __builtin_fmaf(x[i][c], fade, acc[c]);
            }
        }
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
        if (lane + 64 * c < dim) sums[wave][lane + 64 * c] = acc[c];
    if (sum == 0.0f) reference = part_reference(reference, sum, __any(blank));
    if (lane == 0) {
        stat[wave][0] = reference;
        stat[wave][1] = sum;
    }
    __syncthreads();
    const int d = threadIdx.x;
    reference = kNoReference;
#pragma unroll
    for (int i = 0; i < W; ++i)
        if (stat[i][1] != 0.0f) reference = fmaxf(reference, stat[i][0]);
    float value = 0.0f;
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const float fade = stat[i][1] != 0.0f ? exp2_of(stat[i][0] - reference) : 0.0f;
        sum = __builtin_fmaf(stat[i][1], fade, sum);
        if (d < dim) value = __builtin_fmaf(sums[i][d], fade, value);
    }
    blank = false;
    if (sum == 0.0f)
        for (int i = 0; i < W; ++i) blank = blank || part_blank(stat[i][0], stat[i][1]);
    const MergedRow M = merged_row(A, w[0], w[1] + r, w[3]);
    if (d < dim) gout<T>(A.out_ptr)[M.out + d] = static_cast<T>(value * row_factor(sum, blank));
    if (d == 0 && A.lse_ptr) gout<float>(A.lse_ptr)[M.lse] = row_lse(reference, sum);
}

// TPR: threads of a row (8 channels each).
template <int DT, int TPR>
__global__ void __launch_bounds__(256) attend_merge_kernel(const rch_attend A) {
    typedef typename AttendType<DT>::type T;
    const RCH_GLOBAL int32_t* w = gin<int32_t>(A.plan_ptr) + A.merges
                                  + (static_cast<int64_t>(blockIdx.x) + A.n_many) * RCH_ATTEND_MERGE;
    const int rows = w[2], parts = w[5], dim = static_cast<int>(A.head_dim);
    const int64_t first = w[4];
    const int r = blockIdx.y * (256 / TPR) + threadIdx.x / TPR, d = threadIdx.x % TPR * 8;
    if (r >= rows || d >= dim) return;
    const MergedRow M = merged_row(A, w[0], w[1] + r, w[3]);
    f2 stats[kFewParts];
    f4 low[kFewParts], high[kFewParts];
    float reference = kNoReference;
#pragma unroll
    for (int p = 0; p < kFewParts; ++p) {
        if (p < parts) {
            const int64_t at = first + static_cast<int64_t>(p) * rows + r;
            stats[p] = *gin<f2>(partial_stats(A, at));
            low[p] = gin<f4>(partial_sums(A, at) + 4 * d)[0];
            high[p] = gin<f4>(partial_sums(A, at) + 4 * d)[1];
        }
    }
#pragma unroll
    for (int p = 0; p < kFewParts; ++p)
        if (p < parts && stats[p][1] != 0.0f) reference = fmaxf(reference, stats[p][0]);
    float sum = 0.0f, acc[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int p = 0; p < kFewParts; ++p) {
        if (p < parts) {
            const float fade = stats[p][1] != 0.0f ? exp2_of(stats[p][0] - reference) : 0.0f;
            sum = __builtin_fmaf(stats[p][1], fade, sum);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                acc[e] = __builtin_fmaf(low[p][e], fade, acc[e]);
                acc[4 + e] = __builtin_fmaf(high[p][e], fade, acc[4 + e]);
            }
        }
    }
    bool blank = false;
    if (sum == 0.0f) {
#pragma unroll
        for (int p = 0; p < kFewParts; ++p) blank = blank || (p < parts && part_blank(stats[p][0], stats[p][1]));
    }
    const float inverse = row_factor(sum, blank);
    typedef T t8 __attribute__((ext_vector_type(8), aligned(16)));
    t8 v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = static_cast<T>(acc[e] * inverse);
    *reinterpret_cast<RCH_GLOBAL t8*>(gout<T>(A.out_ptr) + M.out + d) = v;
    if (d == 0 && A.lse_ptr) gout<float>(A.lse_ptr)[M.lse] = row_lse(reference, sum);
}

template <int DT, int C>
int merge_many(const rch_attend& A, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(A.n_many), static_cast<uint32_t>(A.most_rows_many));
    if (A.n_many * A.most_rows_many <= kWideRows) hipLaunchKernelGGL((attend_merge_many_kernel<DT, C, 16>), grid, dim3(1024), 0, stream, A);
    else hipLaunchKernelGGL((attend_merge_many_kernel<DT, C, 4>), grid, dim3(256), 0, stream, A);
    return check_launch("rch_attend_run (merge)");
}

template <int DT, int TPR>
int merge_few(const rch_attend& A, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(A.n_merges - A.n_many), static_cast<uint32_t>((A.most_rows * TPR + 255) / 256));
    hipLaunchKernelGGL((attend_merge_kernel<DT, TPR>), grid, dim3(256), 0, stream, A);
    return check_launch("rch_attend_run (merge)");
}

template <int DT>
int run(const rch_attend& A, hipStream_t stream) {
    if (A.n_general) hipLaunchKernelGGL(attend_general_kernel<DT>, dim3(static_cast<uint32_t>(A.n_general)), dim3(256), 0, stream, A);
    const int status = A.n_general ? check_launch("rch_attend_run") : launch_attend_rows(A, DT, stream);
    if (status != RCH_OK) return status;
    if (A.n_many) {
        const int status = A.head_dim <= 128 ? merge_many<DT, 2>(A, stream) : merge_many<DT, 4>(A, stream);
        if (status != RCH_OK) return status;
    }
    if (A.n_merges > A.n_many) return A.head_dim <= 128 ? merge_few<DT, 16>(A, stream) : merge_few<DT, 32>(A, stream);
    return RCH_OK;
}

}  // namespace

}  // namespace rch

extern "C" {

int rch_attend_size(void) { return static_cast<int>(sizeof(rch_attend)); }

int rch_attend_run(const rch_attend* args_host, int dtype, void* stream) {
    using namespace rch;
    if (!args_host) return fail(RCH_E_CONFIG, "rch_attend_run: no arguments");
    const rch_attend& A = *args_host;
    if (A.group < 1 || A.heads < 1 || A.head_dim < 1 || A.head_dim > RCH_ATTEND_MAX_DIM || A.page_tokens < 1 || A.pages < 1
        || A.page_tokens > 0x7fffffff || A.pages > 0x7fffffff || A.block < 0 || A.window < 0 || A.block > 0x7fffffff)
        return fail(RCH_E_CONFIG, "rch_attend_run: invalid sizes");
    if (A.n_general < 0 || A.n_rows < 0 || A.n_merges < 0 || (A.n_general && A.n_rows)
        || A.n_general + A.n_rows > 0x7fffffff)
        return fail(RCH_E_CONFIG, "rch_attend_run: invalid item counts");
    if (A.n_merges && (!A.partial_ptr || A.partial_ptr % 16 || A.n_many < 0 || A.n_many > A.n_merges || A.most_rows < 0 || A.most_rows_many < 0
                       || A.most_rows_many > 65535))
        return fail(RCH_E_CONFIG, "rch_attend_run: invalid merges");
    // Rows of few parts are joined in aligned pieces of eight channels.
    if (A.n_merges > A.n_many && (A.head_dim % 8 || A.out_ptr % 16
                                  || (A.out_token_stride | A.out_head_stride) * (dtype == RCH_DT_F32 ? 4 : 2) % 16))
        return fail(RCH_E_CONFIG, "rch_attend_run: merges of few parts need aligned rows of 8n channels");
    if (A.n_general + A.n_rows == 0) return RCH_OK;
    const uint32_t scale = static_cast<uint32_t>(A.scale_bits);
    if (scale < 0x00800000u || scale >= 0x7f800000u) return fail(RCH_E_CONFIG, "rch_attend_run: scale must be a positive normal number");
    if (!A.q_ptr || !A.k_ptr || !A.v_ptr || !A.out_ptr || !A.plan_ptr) return fail(RCH_E_CONFIG, "rch_attend_run: null address");
    if (A.n_rows) {
        // The tiled forms: whole 16-byte pieces, a tile's rows within 2 GiB, tiles that start over at a page of
        // at least a tile or at 64 keys.
        const int64_t size = dtype == RCH_DT_F32 ? 4 : 2;
        const int64_t mix = A.q_token_stride | A.q_head_stride | A.k_page_stride | A.k_token_stride | A.k_head_stride
                            | A.v_page_stride | A.v_token_stride | A.v_head_stride | A.out_token_stride | A.out_head_stride;
        if (A.head_dim * size % 16 || A.head_dim > RCH_ATTEND_FAST_DIM || mix * size % 16
            || (A.q_ptr | A.k_ptr | A.v_ptr | A.out_ptr | A.plan_ptr) % 16)
            return fail(RCH_E_UNSUPPORTED, "rch_attend_run: the tiled form needs aligned rows of whole 16-byte pieces and at most %d channels",
                        RCH_ATTEND_FAST_DIM);
        if (A.k_token_stride < 0 || A.v_token_stride < 0 || A.k_token_stride > (1 << 22) || A.v_token_stride > (1 << 22))
            return fail(RCH_E_UNSUPPORTED, "rch_attend_run: token rows too far apart for the tiled forms");
        if (!(A.tile_unit == 64 || (A.tile_unit == A.page_tokens && A.page_tokens >= 64)))
            return fail(RCH_E_CONFIG, "rch_attend_run: tiles start over at a page of 64 or more tokens, or at 64 keys");
    }
    hipStream_t s = as_stream(stream);
    switch (dtype) {
        case RCH_DT_F32: return run<RCH_DT_F32>(A, s);
        case RCH_DT_F16: return run<RCH_DT_F16>(A, s);
        case RCH_DT_BF16: return run<RCH_DT_BF16>(A, s);
        default: return fail(RCH_E_CONFIG, "rch_attend_run: dtype must be f32, f16 or bf16");
    }
}

}  // extern "C"
