// Blocks of a cache's keys: their means, and the choice of the blocks that a run of queries attends to.
//
// A block is B consecutive tokens of a page.  Its mean key is summed in FP64 and rounded (by way of FP32); the score of a block for a
// run of queries is (sum of the run's query rows of a key head) . mean, also summed in FP64, so that the order of the sums
// decides no choice between blocks (two scores of FP32 sums over 128 channels differ in their last places, and then a
// block more or less is read).  FP64 costs nothing here: a mean is read once for every D products.
#include "attend.h"
#include "codes.h"

namespace rch {

namespace {

template <int DT, int FMT>
struct Row {
    typedef typename AttendType<DT>::type T;
    static constexpr int kBytes = FMT != RCH_CODES_NONE ? 1 : static_cast<int>(sizeof(T));
    // Eight channels (or fewer: V) of a row of keys as FP64 values.
    template <int V>
    static __device__ __forceinline__ void load(int64_t at, float scale, double (&x)[V]) {
        if constexpr (FMT != RCH_CODES_NONE) {
            uint32_t word[V >= 4 ? V / 4 : 1];
            if constexpr (V == 8) {
                const u2 raw = *gin<u2>(at);
                word[0] = raw[0], word[1] = raw[1];
            } else {
                word[0] = *gin<uint8_t>(at);
            }
#pragma unroll
            for (int i = 0; i < V; ++i) x[i] = static_cast<float>(static_cast<T>(code_numbers<FMT>(word[i / 4])[i % 4] * scale));
        } else if constexpr (V == 8) {
            typedef T t8 __attribute__((ext_vector_type(8), aligned(16)));
            const t8 raw = *gin<t8>(at);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(raw[i]);
        } else {
            x[0] = static_cast<float>(*gin<T>(at));
        }
    }
};

// One workgroup for `share` tokens and a key head: where a token is the last one of its block among its neighbours, the
// block's rows are summed, V channels and every kRows-th row to a thread.
template <int DT, int FMT, int V>
__global__ void __launch_bounds__(256) blocks_update_kernel(const rch_blocks B, int share) {
    typedef typename AttendType<DT>::type T;
    typedef Row<DT, FMT> R;
    __shared__ double sums[256 * V];
    const int dim = static_cast<int>(B.head_dim), size = static_cast<int>(B.block_tokens), head = blockIdx.y;
    const int lanes = dim / V, rows = 256 / lanes;  // threads of a row, rows at once
    const int mine = threadIdx.x / lanes, piece = threadIdx.x - mine * lanes;
    const RCH_GLOBAL int32_t* slots = gin<int32_t>(B.slots_ptr);
    const int64_t first = static_cast<int64_t>(blockIdx.x) * share, behind = first + share < B.tokens ? first + share : B.tokens;
    const int64_t limit = B.pages * B.page_tokens, per = B.page_tokens / size;
    for (int64_t token = first; token < behind; ++token) {
        const int64_t slot = slots[token];
        if (slot < 0 || slot >= limit) continue;
        const int64_t block = slot / size;
        if (token + 1 < B.tokens) {
            const int64_t next = slots[token + 1];
            if (next >= 0 && next < limit && next / size == block) continue;
        }
        const int64_t page = block / per, row0 = (block - page * per) * size;
        const int64_t keys = B.keys_ptr + R::kBytes * (page * B.page_stride + row0 * B.token_stride + head * B.head_stride + piece * V);
        const int64_t scales = FMT == RCH_CODES_NONE ? 0 : B.scales_ptr + 4 * (page * B.scale_page_stride + head * B.scale_head_stride + row0);
        double sum[V];
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] = 0.0;
        if (mine < rows) {
#pragma unroll 4
            for (int row = mine; row < size; row += rows) {
                double x[V];
                float scale = 0.0f;
                if constexpr (FMT != RCH_CODES_NONE) scale = gin<float>(scales)[row];
                R::template load<V>(keys + R::kBytes * row * B.token_stride, scale, x);
#pragma unroll
                for (int i = 0; i < V; ++i) sum[i] += x[i];
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) sums[i * 256 + threadIdx.x] = sum[i];
        __syncthreads();
        const int channel = threadIdx.x;
        if (channel < dim) {
            double total = 0.0;
            for (int r = 0; r < rows; ++r) total += sums[channel % V * 256 + r * lanes + channel / V];
            gout<T>(B.means_ptr)[(block * B.heads + head) * dim + channel] = static_cast<T>(static_cast<float>(total / size));
        }
        __syncthreads();
    }
}

// Order of scores as unsigned numbers: larger scores are larger, NaN is the largest; 0 is kept for blocks that are no
// candidates (below -inf, whose number is 2^52 - 1).
__device__ __forceinline__ uint64_t order_of(double score) {
    if (score != score) return ~uint64_t{0};
    const uint64_t bits = static_cast<uint64_t>(__double_as_longlong(score + 0.0));  // -0 is 0
    return bits >> 63 ? ~bits : bits | uint64_t{1} << 63;
}

struct Run {
    int table, q_row, queries, first, last, scored, scored_end, kept, kept_end;
};
__device__ __forceinline__ Run run_of(const rch_blocks& B, int index) {
    const RCH_GLOBAL int32_t* w = gin<int32_t>(B.plan_ptr) + B.runs + static_cast<int64_t>(index) * RCH_BLOCKS_RUN;
    return {w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7], w[8]};
}
// The pool's page of a block, or -1 where it lies in a hole.
__device__ __forceinline__ int page_of(const rch_blocks& B, const Run& R, int block, int per) {
    const int id = gin<int32_t>(B.plan_ptr)[R.table + block / per];
    return id >= 0 && id < B.pages ? id : -1;
}

constexpr int kScored = 128;  // blocks that a workgroup scores

// Scores kScored blocks for a run and key head.  V channels to a lane.
template <int DT, int V>
__global__ void __launch_bounds__(256) blocks_score_kernel(const rch_blocks B) {
    typedef typename AttendType<DT>::type T;
    typedef Row<DT, RCH_CODES_NONE> K;
    __shared__ double pooled[256], sums[256 * V];
    const Run R = run_of(B, blockIdx.x);
    const int head = blockIdx.z, dim = static_cast<int>(B.head_dim), group = static_cast<int>(B.group);
    const int begin = R.scored + blockIdx.y * kScored, end = min(begin + kScored, R.scored_end);
    if (begin >= end) return;
    const int lanes = dim / V, rows = 256 / lanes, mine = threadIdx.x / lanes, piece = threadIdx.x - mine * lanes;
    {
        double sum[V];
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] = 0.0;
        if (mine < rows) {
#pragma unroll 4
            for (int row = mine; row < R.queries * group; row += rows) {
                const int token = row / group, member = head * group + row - token * group;
                double x[V];
                K::template load<V>(B.q_ptr + static_cast<int64_t>(sizeof(T)) * ((R.q_row + token) * B.q_token_stride + member * B.q_head_stride + piece * V),
                                    0.0f, x);
#pragma unroll
                for (int i = 0; i < V; ++i) sum[i] += x[i];
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) sums[i * 256 + threadIdx.x] = sum[i];
        __syncthreads();
        const int channel = threadIdx.x;
        double total = 0.0;
        if (channel < dim)
            for (int r = 0; r < rows; ++r) total += sums[channel % V * 256 + r * lanes + channel / V];
        pooled[channel] = total;
        __syncthreads();
    }
    // A block's mean lies in W lanes (a power of two).
    const int per = static_cast<int>(B.page_tokens / B.block_tokens), lane = threadIdx.x & 63;
    int width = 1;
    while (width * V < dim && width < 64) width *= 2;
    const int at = lane & (width - 1), step = 256 / width;
    RCH_GLOBAL uint64_t* out = gout<uint64_t>(B.scores_ptr)
                               + (static_cast<int64_t>(blockIdx.x) * B.heads + head) * B.scores - R.scored;
    for (int block = begin + threadIdx.x / width; block - static_cast<int>(threadIdx.x) / width < end; block += step) {
        const int page = block < end ? page_of(B, R, block, per) : -1;
        double score = 0.0;
        if (page >= 0) {
            const int64_t mean = B.means_ptr
                                 + static_cast<int64_t>(sizeof(T)) * ((static_cast<int64_t>(page) * per + block % per) * B.heads + head) * dim;
            for (int d = at * V; d < dim; d += width * V) {
                double x[V];
                K::template load<V>(mean + static_cast<int64_t>(sizeof(T)) * d, 0.0f, x);
#pragma unroll
                for (int i = 0; i < V; ++i) score = __builtin_fma(x[i], pooled[d + i], score);
            }
        }
        for (int o = 1; o < width; o <<= 1) score += __shfl_xor(score, o);
        if (at == 0 && block < end) out[block] = page >= 0 ? order_of(score) : 0;
    }
}

// Writes the blocks of a run and key head: all that are not scored, those kept anyway and the `top` best of the others.
// The top-th best number is found eight bits at a time (a count of each value of the bits among the numbers that agree in
// the bits before), until the blocks above and at it are just as many.
__global__ void __launch_bounds__(256) blocks_take_kernel(const rch_blocks B) {
    __shared__ uint32_t count[256], waves[2][4];
    __shared__ uint32_t found[3];
    const Run R = run_of(B, blockIdx.x);
    const int head = blockIdx.y, per = static_cast<int>(B.page_tokens / B.block_tokens);
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const RCH_GLOBAL uint64_t* scores = gin<uint64_t>(B.scores_ptr)
                                        + (static_cast<int64_t>(blockIdx.x) * B.heads + head) * B.scores - R.scored;
    auto chosen_by_score = [&](int block) { return block >= R.scored && block < R.scored_end && !(block >= R.kept && block < R.kept_end); };

    // Numbers above `bar` are taken, and the first `even` of those equal to it (in the bits of `mask`).
    uint64_t bar = 0, mask = 0;
    uint32_t even = static_cast<uint32_t>(B.top);
    bool all = false;  // no more candidates than are wanted
    for (int shift = 56; even && shift >= 0; shift -= 8) {
        count[t] = 0;
        __syncthreads();
        for (int block = R.scored + t; block < R.scored_end; block += 256) {
            if (!chosen_by_score(block)) continue;
            const uint64_t number = scores[block];
            if (number != 0 && (number & mask) == bar) atomicAdd(&count[number >> shift & 255], 1u);
        }
        __syncthreads();
        if (wave == 0) {
            // From the highest value down: lane i counts values 255 - 4 i .. 252 - 4 i.
            uint32_t c[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = count[255 - 4 * lane - i], sum += c[i];
            uint32_t upto = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t other = __shfl_up(upto, o);
                if (lane >= o) upto += other;
            }
            uint32_t before = upto - sum;
            if (lane == 63) found[0] = upto;
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // the value that the last wanted one has (of one lane, where there are enough)
                if (before < even && before + c[i] >= even) found[1] = 255 - 4 * lane - i, found[2] = even - before;
                before += c[i];
            }
        }
        __syncthreads();
        const uint32_t total = found[0], value = found[1], rest = found[2];
        if (total <= even) {  // every one that agrees so far; at first those are all candidates
            all = mask == 0;
            break;
        }
        bar |= static_cast<uint64_t>(value) << shift;
        mask |= uint64_t{255} << shift;
        even = rest;
    }
    // In ascending order: the place of a block is the number of taken ones before it.
    RCH_GLOBAL int32_t* list = gout<int32_t>(B.lists_ptr) + (static_cast<int64_t>(blockIdx.x) * B.heads + head) * B.width;
    int written = 0;
    uint32_t equal = 0;
    for (int base = R.first; base < R.last; base += 256) {
        const int block = base + t;
        bool taken = false, same = false;
        if (block < R.last && page_of(B, R, block, per) >= 0) {
            if (all || !chosen_by_score(block)) {
                taken = true;
            } else if (mask) {  // (none is wanted otherwise, and there may be no scores)
                const uint64_t number = scores[block] & mask;
                taken = number > bar;
                same = number == bar;
            }
        }
        // Equal ones by their number.
        const uint64_t alike = __ballot(same);
        if (lane == 0) waves[0][wave] = __popcll(alike);
        __syncthreads();
        uint32_t before = equal;
        for (int w = 0; w < 4; ++w) {
            if (w < wave) before += waves[0][w];
            equal += waves[0][w];
        }
        before += __popcll(alike & ((uint64_t{1} << lane) - 1));
        taken = taken || (same && before < even);
        const uint64_t votes = __ballot(taken);
        if (lane == 0) waves[1][wave] = __popcll(votes);
        __syncthreads();
        int place = written;
        for (int w = 0; w < 4; ++w) {
            if (w < wave) place += waves[1][w];
            written += waves[1][w];
        }
        place += __popcll(votes & ((uint64_t{1} << lane) - 1));
        if (taken && place < B.width) list[place] = block;
    }
    for (int at = written + t; at < B.width; at += 256) list[at] = -1;
}

// What both entry points need of the pools' description.
int invalid(const rch_blocks& B, int dtype, const char* what) {
    if (dtype != RCH_DT_F32 && dtype != RCH_DT_F16 && dtype != RCH_DT_BF16) return fail(RCH_E_CONFIG, "%s: dtype must be f32, f16 or bf16", what);
    if (B.heads < 1 || B.heads > 65535 || B.head_dim < 1 || B.head_dim > RCH_ATTEND_MAX_DIM || B.pages < 1 || B.page_tokens < 1 || B.block_tokens < 1
        || B.page_tokens % B.block_tokens || B.pages > 0x7fffffff || B.page_tokens > 0x7fffffff || B.pages * B.page_tokens > 0x7fffffff)
        return fail(RCH_E_CONFIG, "%s: invalid sizes", what);
    return RCH_OK;
}

template <int DT, int FMT>
int update(const rch_blocks& B, hipStream_t stream) {
    // Tokens of a workgroup: one while that makes few of them, so that the touched blocks of single tokens run at once.
    const int64_t wanted = B.tokens * B.heads / 4096;
    const int share = static_cast<int>(wanted < 1 ? 1 : wanted > 64 ? 64 : wanted);
    const dim3 grid(static_cast<uint32_t>((B.tokens + share - 1) / share), static_cast<uint32_t>(B.heads));
    const int64_t bytes = Row<DT, FMT>::kBytes, piece = FMT == RCH_CODES_NONE ? 16 : 8;
    const bool wide = B.head_dim % 8 == 0 && B.keys_ptr % piece == 0 && (B.page_stride | B.token_stride | B.head_stride) * bytes % piece == 0;
    if (wide) hipLaunchKernelGGL((blocks_update_kernel<DT, FMT, 8>), grid, dim3(256), 0, stream, B, share);
    else hipLaunchKernelGGL((blocks_update_kernel<DT, FMT, 1>), grid, dim3(256), 0, stream, B, share);
    return check_launch("rch_blocks_update");
}

template <int DT>
int update_of(const rch_blocks& B, hipStream_t stream) {
    if constexpr (DT != RCH_DT_F32) {
        if (B.codes == RCH_CODES_INT8) return update<DT, RCH_CODES_INT8>(B, stream);
        if (B.codes == RCH_CODES_E4M3) return update<DT, RCH_CODES_E4M3>(B, stream);
    }
    return update<DT, RCH_CODES_NONE>(B, stream);
}

template <int DT>
int select(const rch_blocks& B, hipStream_t stream) {
    const int64_t size = DT == RCH_DT_F32 ? 4 : 2;
    if (B.scores) {
        const dim3 grid(static_cast<uint32_t>(B.n_runs), static_cast<uint32_t>((B.scores + kScored - 1) / kScored), static_cast<uint32_t>(B.heads));
        const bool wide = B.head_dim % 8 == 0 && (B.q_ptr | B.means_ptr) % 16 == 0 && (B.q_token_stride | B.q_head_stride) * size % 16 == 0;
        if (wide) hipLaunchKernelGGL((blocks_score_kernel<DT, 8>), grid, dim3(256), 0, stream, B);
        else hipLaunchKernelGGL((blocks_score_kernel<DT, 1>), grid, dim3(256), 0, stream, B);
        const int status = check_launch("rch_blocks_select (scores)");
        if (status != RCH_OK) return status;
    }
    const dim3 grid(static_cast<uint32_t>(B.n_runs), static_cast<uint32_t>(B.heads));
    hipLaunchKernelGGL(blocks_take_kernel, grid, dim3(256), 0, stream, B);
    return check_launch("rch_blocks_select");
}

}  // namespace

}  // namespace rch

extern "C" {

int rch_blocks_size(void) { return static_cast<int>(sizeof(rch_blocks)); }

int rch_blocks_update(const rch_blocks* args_host, int dtype, void* stream) {
    using namespace rch;
    if (!args_host) return fail(RCH_E_CONFIG, "rch_blocks_update: no arguments");
    const rch_blocks& B = *args_host;
    const int status = invalid(B, dtype, "rch_blocks_update");
    if (status != RCH_OK) return status;
    if (B.codes != RCH_CODES_NONE && B.codes != RCH_CODES_INT8 && B.codes != RCH_CODES_E4M3)
        return fail(RCH_E_CONFIG, "rch_blocks_update: unknown format of codes");
    if (B.codes != RCH_CODES_NONE && dtype == RCH_DT_F32) return fail(RCH_E_UNSUPPORTED, "rch_blocks_update: codes stand for f16 or bf16 values");
    if (B.tokens < 0 || B.tokens > 0x7fffffff) return fail(RCH_E_CONFIG, "rch_blocks_update: invalid token count");
    if (B.tokens == 0) return RCH_OK;
    if (!B.means_ptr || !B.keys_ptr || !B.slots_ptr || (B.codes != RCH_CODES_NONE && !B.scales_ptr)) return fail(RCH_E_CONFIG, "rch_blocks_update: null address");
    hipStream_t s = as_stream(stream);
    if (dtype == RCH_DT_F32) return update_of<RCH_DT_F32>(B, s);
    return dtype == RCH_DT_F16 ? update_of<RCH_DT_F16>(B, s) : update_of<RCH_DT_BF16>(B, s);
}

int rch_blocks_select(const rch_blocks* args_host, int dtype, void* stream) {
    using namespace rch;
    if (!args_host) return fail(RCH_E_CONFIG, "rch_blocks_select: no arguments");
    const rch_blocks& B = *args_host;
    const int status = invalid(B, dtype, "rch_blocks_select");
    if (status != RCH_OK) return status;
    if (B.group < 1 || B.n_runs < 0 || B.n_runs > 0x7fffffff || B.scores < 0 || B.scores > 65535 * kScored || B.width < 0 || B.width > 0x7fffffff || B.top < 0
        || B.top > 0x7fffffff)
        return fail(RCH_E_CONFIG, "rch_blocks_select: invalid runs");
    if (B.n_runs == 0 || B.width == 0) return RCH_OK;
    if (!B.means_ptr || !B.q_ptr || !B.plan_ptr || !B.lists_ptr || (B.scores && !B.scores_ptr) || B.scores_ptr % 8)
        return fail(RCH_E_CONFIG, "rch_blocks_select: null or misaligned address");
    hipStream_t s = as_stream(stream);
    if (dtype == RCH_DT_F32) return select<RCH_DT_F32>(B, s);
    return dtype == RCH_DT_F16 ? select<RCH_DT_F16>(B, s) : select<RCH_DT_BF16>(B, s);
}

}  // extern "C"
