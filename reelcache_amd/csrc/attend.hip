// Attention over a paged cache: the general form, the merge of partial results and the entry point.
//
// For a row q (a query token and head) over the keys it sees:
//   s_j = scale q.k_j,  out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  m >= max_j s_j roughly:
// any reference m gives the same quotient, so one pass over the keys keeps a running m, sum and
// weighted sum, all in fp32, and multiplies both sums by exp(m_old - m_new) where m moves.  Exponents
// are base 2 (scale carries log2 e).  Two parts of a row's keys join the same way.
//
// The general form takes every head_dim up to 256, alignment and element type: one wave per row, a
// lane per key for the scores, a lane per channel for the sums.  The forms that tile for the matrix
// cores are in attend_rows.hip and attend_tokens.hip.
#include "attend.h"

namespace rch {

namespace {

template <int DT>
__global__ void __launch_bounds__(256) attend_general_kernel(const rch_attend A, int first_item) {
    typedef typename AttendType<DT>::type T;
    __shared__ float query[4][RCH_ATTEND_MAX_DIM];
    __shared__ float weight[4][64];
    __shared__ int64_t place_of[4][64];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const AttendItem I = attend_item(A, first_item + blockIdx.x);
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
            if (lane == 0) *gout<f2>(partial_stats(A, at)) = f2{reference, sum};
            continue;
        }
        RCH_GLOBAL T* out = gout<T>(A.out_ptr) + (I.q_row + token) * A.out_token_stride + head * A.out_head_stride;
        const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
        for (int c = 0; c < RCH_ATTEND_MAX_DIM / 64; ++c)
            if (lane + 64 * c < dim) out[lane + 64 * c] = static_cast<T>(acc[c] * inverse);
        if (lane == 0 && A.lse_ptr) gout<float>(A.lse_ptr)[(I.q_row + token) * A.heads + head] = row_lse(reference, sum);
    }
}

// Joins the parts of rows whose keys were split: a thread per row and channel, parts in order.
template <int DT>
__global__ void __launch_bounds__(256) attend_merge_kernel(const rch_attend A) {
    typedef typename AttendType<DT>::type T;
    const RCH_GLOBAL int32_t* w = gin<int32_t>(A.plan_ptr) + A.merges + static_cast<int64_t>(blockIdx.x) * RCH_ATTEND_MERGE;
    const int q_row = w[0], row_begin = w[1], rows = w[2], kv_head = w[3], first = w[4], parts = w[5];
    const int dim = static_cast<int>(A.head_dim), group = static_cast<int>(A.group);
    const int index = blockIdx.y * 256 + threadIdx.x;
    const int r = index / dim, d = index - r * dim;
    if (r >= rows) return;
    const int token = (row_begin + r) / group, head = kv_head * group + (row_begin + r) % group;
    float reference = kNoReference;
    for (int p = 0; p < parts; ++p) {
        const f2 stats = *gin<f2>(partial_stats(A, first + static_cast<int64_t>(p) * rows + r));
        if (stats[1] != 0.0f) reference = fmaxf(reference, stats[0]);
    }
    float sum = 0.0f, acc = 0.0f;
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {
        const int64_t at = first + static_cast<int64_t>(p) * rows + r;
        const f2 stats = *gin<f2>(partial_stats(A, at));
        const float fade = stats[1] != 0.0f ? exp2_of(stats[0] - reference) : 0.0f;
        sum = __builtin_fmaf(stats[1], fade, sum);
        acc = __builtin_fmaf(gin<float>(partial_sums(A, at))[d], fade, acc);
    }
    const float inverse = sum == 0.0f ? 0.0f : 1.0f / sum;
    gout<T>(A.out_ptr)[(q_row + token) * A.out_token_stride + head * A.out_head_stride + d] = static_cast<T>(acc * inverse);
    if (d == 0 && A.lse_ptr) gout<float>(A.lse_ptr)[(q_row + token) * A.heads + head] = row_lse(reference, sum);
}

template <int DT>
int run(const rch_attend& A, hipStream_t stream) {
    int first = 0;
    if (A.n_general) {
        hipLaunchKernelGGL(attend_general_kernel<DT>, dim3(static_cast<uint32_t>(A.n_general)), dim3(256), 0, stream, A, first);
        const int status = check_launch("rch_attend_run");
        if (status != RCH_OK) return status;
        first += static_cast<int>(A.n_general);
    }
    if (A.n_rows) {
        const int status = launch_attend_rows(A, DT, first, stream);
        if (status != RCH_OK) return status;
    }
    if (A.n_merges) {
        const uint32_t blocks = static_cast<uint32_t>((A.most_rows * A.head_dim + 255) / 256);
        hipLaunchKernelGGL(attend_merge_kernel<DT>, dim3(static_cast<uint32_t>(A.n_merges), blocks), dim3(256), 0, stream, A);
        return check_launch("rch_attend_run (merge)");
    }
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
    if (A.n_general < 0 || A.n_rows < 0 || A.n_tokens < 0 || A.n_merges < 0 || A.n_general + A.n_rows + A.n_tokens > 0x7fffffff)
        return fail(RCH_E_CONFIG, "rch_attend_run: invalid item counts");
    if (A.n_merges && (!A.partial_ptr || A.most_rows < 1)) return fail(RCH_E_CONFIG, "rch_attend_run: merges need partials");
    if (A.n_general + A.n_rows + A.n_tokens == 0) return RCH_OK;
    if (!A.q_ptr || !A.k_ptr || !A.v_ptr || !A.out_ptr || !A.plan_ptr) return fail(RCH_E_CONFIG, "rch_attend_run: null address");
    if (A.n_rows + A.n_tokens) {
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
