// Blocks of a cache's keys: their means, and the choice of the blocks that a run of queries attends to.
//
// A block is B consecutive tokens of a page.  Its mean key is summed in FP64 and rounded (by way of FP32); the score of a block for a
// run of queries is (sum of the run's query rows of a key head) . mean, also summed in FP64, so that the order of the sums
// decides no choice between blocks (two scores of FP32 sums over 128 channels differ in their last places, and then a
// block more or less is read).  FP64 costs nothing here: a mean is read once for every D products.
//
// Bound: latency.  Means of the 39 blocks of 120 that 4680 tokens of 12 heads of 128 touch take 5.7 us (14 MB), of one block
// of 64 in each of 32 sequences 4.0.  The choice for 39 runs of 120 queries among 273 blocks takes 17-19 us in one launch, of
// which the sums over 7 MB of queries, eight rows in flight to a thread, are a third; for four single tokens of 32 heads
// among up to 1024 blocks 6.6 us to score and 7.9 to take.
#include "attend_tile.h"
#include "codes.h"

namespace rch {

namespace {

// V channels of a row of keys (8, in aligned pieces, or 1): fetched, so that several are in flight, then taken as FP64.
template <int DT, int FMT, int V>
struct Row {
    typedef typename AttendType<DT>::type T;
    static constexpr int kBytes = FMT != RCH_CODES_NONE ? 1 : static_cast<int>(sizeof(T)), kWords = V * kBytes / 4;
    uint32_t word[kWords ? kWords : 1];
    float scale;

    __device__ __forceinline__ void fetch(int64_t at, float s = 0.0f) {
        scale = s;
        if constexpr (kWords == 0 && kBytes == 1) {
            word[0] = *gin<uint8_t>(at);
        } else if constexpr (kWords == 0) {
            word[0] = *gin<uint16_t>(at);
        } else if constexpr (kWords == 1) {
            word[0] = *gin<uint32_t>(at);
        } else if constexpr (kWords == 2) {
            const u2 raw = *gin<u2>(at);
            word[0] = raw[0], word[1] = raw[1];
        } else {
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                const u4 raw = gin<u4>(at)[i];
#pragma unroll
                for (int j = 0; j < 4; ++j) word[4 * i + j] = raw[j];
            }
        }
    }
    __device__ __forceinline__ void clear_unless(bool kept) {
#pragma unroll
        for (uint32_t& w : word) w = kept ? w : 0u;
        if constexpr (FMT != RCH_CODES_NONE) scale = kept ? scale : 0.0f;
    }
    __device__ __forceinline__ double value(int i) const {
        if constexpr (FMT != RCH_CODES_NONE) {
            if constexpr (V == 8) return static_cast<float>(code_values<DT, FMT>(word[0], word[1], scale)[i]);
            else return static_cast<float>(code_value<DT, FMT>(static_cast<uint8_t>(word[0]), scale));
        } else if constexpr (sizeof(T) == 4) {
            return __uint_as_float(word[i]);
        } else if constexpr (DT == RCH_DT_BF16) {
            return __uint_as_float(i % 2 ? word[i / 2] & 0xffff0000u : word[i / 2] << 16);
        } else {
            const h2 pair = __builtin_bit_cast(h2, word[i / 2]);
            return static_cast<float>(pair[i % 2]);
        }
    }
};

// Keeps loads that are to be in flight together from being waited for one by one.
__device__ __forceinline__ void all_issued() { __builtin_amdgcn_sched_barrier(0); }

// One workgroup for up to 64 tokens (`share`) and a key head: where a token is the last one of its block among its
// neighbours, the block's rows are summed, V channels and every kRows-th row to a thread.
template <int DT, int FMT, int V>
__global__ void __launch_bounds__(256) blocks_update_kernel(const rch_blocks B, int share) {
    typedef typename AttendType<DT>::type T;
    typedef Row<DT, FMT, V> R;
    constexpr int kAhead = 8;  // rows in flight
    __shared__ double sums[256 * V];
    const int dim = static_cast<int>(B.head_dim), size = static_cast<int>(B.block_tokens), head = blockIdx.y;
    const int lanes = dim / V, rows = 256 / lanes;  // threads of a row, rows at once
    const int mine = threadIdx.x / lanes, piece = threadIdx.x - mine * lanes, lane = threadIdx.x & 63;
    const RCH_GLOBAL int32_t* slots = gin<int32_t>(B.slots_ptr);
    const int64_t limit = B.pages * B.page_tokens;
    const uint32_t per = static_cast<uint32_t>(B.page_tokens) / static_cast<uint32_t>(size);
    // Every wave finds the workgroup's blocks, a lane to a token.
    const int64_t token = static_cast<int64_t>(blockIdx.x) * share + lane;
    const bool there = lane < share && token < B.tokens;
    const int slot = there ? slots[token] : -1, next = there && token + 1 < B.tokens ? slots[token + 1] : -1;
    const bool held = slot >= 0 && slot < limit;
    const int number = held ? slot / size : -1;
    uint64_t ends = __ballot(held && !(next >= 0 && next < limit && next / size == number));
    while (ends) {
        const uint32_t found = __shfl(number, __builtin_ctzll(ends)), page_found = found / per;
        ends &= ends - 1;
        const int64_t block = found, page = page_found, row0 = static_cast<int64_t>(found - page_found * per) * size;
        const int64_t keys = B.keys_ptr + R::kBytes * (page * B.page_stride + row0 * B.token_stride + head * B.head_stride + piece * V);
        const int64_t scales = FMT == RCH_CODES_NONE ? 0 : B.scales_ptr + 4 * (page * B.scale_page_stride + head * B.scale_head_stride + row0);
        double sum[V];
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] = 0.0;
        if (mine < rows) {
            for (int row = mine; row < size; row += rows * kAhead) {
                R x[kAhead];
#pragma unroll
                for (int a = 0; a < kAhead; ++a) {
                    const int at = min(row + a * rows, size - 1);
                    float scale = 0.0f;
                    if constexpr (FMT != RCH_CODES_NONE) scale = gin<float>(scales)[at];
                    x[a].fetch(keys + R::kBytes * (at * B.token_stride), scale);
                }
                all_issued();
#pragma unroll
                for (int a = 0; a < kAhead; ++a) {
                    x[a].clear_unless(row + a * rows < size);
#pragma unroll
                    for (int i = 0; i < V; ++i) sum[i] += x[a].value(i);
                }
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
    const const_int* w = (const const_int*)(uintptr_t)(B.plan_ptr + 4 * (B.runs + static_cast<int64_t>(index) * RCH_BLOCKS_RUN));
    return {w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7], w[8]};
}
// The entry of a run's table for its `index`-th page, and whether it is no hole.
__device__ __forceinline__ int page_of(const rch_blocks& B, const Run& R, int index) { return gin<int32_t>(B.plan_ptr)[R.table + index]; }
__device__ __forceinline__ bool page_held(const rch_blocks& B, int id) { return id >= 0 && id < static_cast<int>(B.pages); }

constexpr int kScored = 128;     // blocks that a workgroup of the separate scoring takes
constexpr int kTogether = RCH_BLOCKS_TOGETHER;  // most scored blocks of a run whose numbers fit in LDS, scored and taken by one workgroup

// The sum of a run's query rows of a key head, in FP64.  V channels to a thread.
template <int DT, int V, int THREADS>
__device__ __forceinline__ void pool_queries(const rch_blocks& B, const Run& R, int head, double* sums, double* pooled) {
    typedef typename AttendType<DT>::type T;
    constexpr int kAhead = 8;
    const int dim = static_cast<int>(B.head_dim), group = static_cast<int>(B.group), count = R.queries * group;
    const int lanes = dim / V, rows = 256 / lanes, mine = threadIdx.x / lanes, piece = threadIdx.x - mine * lanes;
    Divider by_group;
    by_group.init(group);
    if (threadIdx.x < 256) {
        double sum[V];
#pragma unroll
        for (int i = 0; i < V; ++i) sum[i] = 0.0;
        if (mine < rows) {
            for (int row = mine; row < count; row += rows * kAhead) {
                Row<DT, RCH_CODES_NONE, V> x[kAhead];
#pragma unroll
                for (int a = 0; a < kAhead; ++a) {
                    const int at = min(row + a * rows, count - 1), token = by_group.quotient(at), member = head * group + at - token * group;
                    x[a].fetch(B.q_ptr + static_cast<int64_t>(sizeof(T)) * ((R.q_row + token) * B.q_token_stride + member * B.q_head_stride + piece * V));
                }
                all_issued();
#pragma unroll
                for (int a = 0; a < kAhead; ++a) {
                    x[a].clear_unless(row + a * rows < count);
#pragma unroll
                    for (int i = 0; i < V; ++i) sum[i] += x[a].value(i);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i) sums[i * 256 + threadIdx.x] = sum[i];
    }
    __syncthreads();
    if (threadIdx.x < 256) {
        const int channel = threadIdx.x;
        double total = 0.0;
        if (channel < dim)
            for (int r = 0; r < rows; ++r) total += sums[channel % V * 256 + r * lanes + channel / V];
        pooled[channel] = total;
    }
    __syncthreads();
}

// Lanes with `upper` keep the upper N of 2 N sums, the others the lower ones, each with its neighbour's (lane ^ N) added.
template <int N>
__device__ __forceinline__ void fold(double* x, bool upper) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const double give = upper ? x[i] : x[N + i], keep = upper ? x[N + i] : x[i];
        x[i] = keep + __shfl_xor(give, N);
    }
}

// Numbers of blocks [begin, end) of a run and key head, to out(block, number).  A block's mean lies in `width` lanes (a power
// of two), V channels to a lane; a thread has kAhead blocks in flight (pages first, then means).
template <int DT, int V, int THREADS, typename Out>
__device__ __forceinline__ void score_blocks(const rch_blocks& B, const Run& R, int head, int begin, int end, const double* pooled, Out out) {
    typedef typename AttendType<DT>::type T;
    constexpr int kAhead = V == 1 ? 1 : 8;
    const int lane = threadIdx.x & 63, dim = static_cast<int>(B.head_dim);
    Divider by_page;
    by_page.init(static_cast<uint32_t>(B.page_tokens) / static_cast<uint32_t>(B.block_tokens));
    const int per = static_cast<int>(by_page.by);
    int width = 1;
    while (width * V < dim && width < 64) width *= 2;
    const int at = lane & (width - 1), step = THREADS / width;
    const int64_t base = B.means_ptr + static_cast<int64_t>(sizeof(T)) * head * dim, block_bytes = static_cast<int64_t>(sizeof(T)) * B.heads * dim;
    double q[V];  // V == 8: all that the lane needs of the queries
#pragma unroll
    for (int i = 0; i < V; ++i) q[i] = at * V + i < dim ? pooled[at * V + i] : 0.0;
    for (int first = begin; first < end; first += step * kAhead) {
        int page[kAhead], in_page[kAhead];
#pragma unroll
        for (int a = 0; a < kAhead; ++a) {
            const int block = min(first + a * step + static_cast<int>(threadIdx.x) / width, end - 1), index = by_page.quotient(block);
            in_page[a] = block - index * per;
            page[a] = page_of(B, R, index);
        }
        all_issued();
#pragma unroll
        for (int a = 0; a < kAhead; ++a) page[a] = page_held(B, page[a]) ? page[a] : -1;
        double score[kAhead];
        if constexpr (V == 8) {
            Row<DT, RCH_CODES_NONE, V> x[kAhead];
            const bool in = at * V < dim;
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {  // (of a hole, page 0's; behind the head's channels, the first ones)
                const int64_t block = static_cast<int64_t>(max(page[a], 0)) * per + in_page[a];
                x[a].fetch(base + block * block_bytes + (in ? static_cast<int64_t>(sizeof(T)) * at * V : 0));
            }
            all_issued();
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                score[a] = 0.0;
                if (first + a * step >= end) continue;
                x[a].clear_unless(in);
#pragma unroll
                for (int i = 0; i < V; ++i) score[a] = __builtin_fma(x[a].value(i), q[i], score[a]);
            }
        } else {
            score[0] = 0.0;
            const int64_t mean = base + (static_cast<int64_t>(max(page[0], 0)) * per + in_page[0]) * block_bytes;
            for (int d = at; d < dim; d += width) {
                Row<DT, RCH_CODES_NONE, 1> x;
                x.fetch(mean + static_cast<int64_t>(sizeof(T)) * d);
                score[0] = __builtin_fma(x.value(0), pooled[d], score[0]);
            }
        }
        const int block = first + static_cast<int>(threadIdx.x) / width;
        if (kAhead == 8 && width >= 8) {
            // The sums over a block's lanes: each step joins two of the blocks into one, half of the lanes for each, so that
            // lane `at` ends with block at % 8.
            int held = page[0];
#pragma unroll
            for (int a = 1; a < kAhead; ++a) held = (at & 7) == a ? page[a] : held;
            fold<4>(score, at & 4);
            fold<2>(score, at & 2);
            fold<1>(score, at & 1);
            double own = score[0];
            for (int o = 8; o < width; o <<= 1) own += __shfl_xor(own, o);
            if (at < 8 && block + at * step < end) out(block + at * step, held >= 0 ? order_of(own) : 0);
        } else {
            for (int o = 1; o < width; o <<= 1)
#pragma unroll
                for (int a = 0; a < kAhead; ++a) score[a] += __shfl_xor(score[a], o);
            if (at == 0)
#pragma unroll
                for (int a = 0; a < kAhead; ++a)
                    if (block + a * step < end) out(block + a * step, page[a] >= 0 ? order_of(score[a]) : 0);
        }
    }
}

// Writes the blocks of a run and key head: all that are not scored, those kept anyway and the `top` best of the others.
// The top-th best number is found eight bits at a time, from the highest bit in which any two differ on (a count of each
// value of the bits among the numbers that agree in the bits before), until the numbers that agree are no more than are
// wanted.  number(block): of a scored one.
struct Taking {
    uint32_t count[256], found[3], waves[2][16];
};
template <int CONTROL>
__device__ __forceinline__ uint32_t moved(uint32_t x) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CONTROL, 0xf, 0xf, true));
}
template <typename Join>
__device__ __forceinline__ uint32_t joined(uint32_t x, Join join) {
    x = join(x, moved<0xb1>(x));   // lanes 1 0 3 2
    x = join(x, moved<0x4e>(x));   // lanes 2 3 0 1
    x = join(x, moved<0x141>(x));  // mirrored in 8
    x = join(x, moved<0x140>(x));  // mirrored in 16
    x = join(x, static_cast<uint32_t>(__shfl_xor(static_cast<int>(x), 16)));
    return join(x, static_cast<uint32_t>(__shfl_xor(static_cast<int>(x), 32)));
}
template <int THREADS, typename Number>
__device__ __forceinline__ void take_blocks(const rch_blocks& B, const Run& R, int head, Taking& L, Number number) {
    Divider by_page;
    by_page.init(static_cast<uint32_t>(B.page_tokens) / static_cast<uint32_t>(B.block_tokens));
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    auto chosen_by_score = [&](int block) { return block >= R.scored && block < R.scored_end && !(block >= R.kept && block < R.kept_end); };

    // Numbers above `bar` are taken, and the first `even` of those equal to it (in the bits of `mask`).
    uint64_t bar = 0, mask = 0;
    uint32_t even = static_cast<uint32_t>(B.top);
    bool all = false;  // no more candidates than are wanted
    int shift = 0;
    if (even) {
        // The bits that all numbers share (of their upper halves).
        uint32_t every = ~0u, any = 0;
        for (int block = R.scored + t; block < R.scored_end; block += THREADS) {
            if (!chosen_by_score(block)) continue;
            const uint64_t n = number(block);
            if (n != 0) every &= static_cast<uint32_t>(n >> 32), any |= static_cast<uint32_t>(n >> 32);
        }
        every = joined(every, [](uint32_t a, uint32_t b) { return a & b; });
        any = joined(any, [](uint32_t a, uint32_t b) { return a | b; });
        if (lane == 0) L.waves[0][wave] = every, L.waves[1][wave] = any;
        __syncthreads();
        for (int w = 0; w < THREADS / 64; ++w) every &= L.waves[0][w], any |= L.waves[1][w];
        const uint32_t differ = every ^ any;
        const int top = differ ? 63 - __builtin_clz(differ) : 31;  // the first bit to look at
        shift = top - 7;
        mask = top == 63 ? 0 : ~uint64_t{0} << (top + 1);
        bar = (static_cast<uint64_t>(every) << 32) & mask;
    }
    for (bool first = true; even; first = false) {
        if (t < 256) L.count[t] = 0;
        __syncthreads();
        for (int block = R.scored + t; block < R.scored_end; block += THREADS) {
            if (!chosen_by_score(block)) continue;
            const uint64_t n = number(block);
            if (n != 0 && (n & mask) == bar) atomicAdd(&L.count[n >> shift & 255], 1u);
        }
        __syncthreads();
        if (wave == 0) {
            // From the highest value down: lane i counts values 255 - 4 i .. 252 - 4 i.
            uint32_t c[4], sum = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) c[i] = L.count[255 - 4 * lane - i], sum += c[i];
            uint32_t upto = sum;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const uint32_t other = __shfl_up(upto, o);
                if (lane >= o) upto += other;
            }
            uint32_t before = upto - sum;
            if (lane == 63) L.found[0] = upto;
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // the value that the last wanted one has (of one lane, where there are enough)
                if (before < even && before + c[i] >= even) {
                    L.found[1] = 255 - 4 * lane - i;
                    L.found[2] = even - before | (before + c[i] == even ? 1u << 31 : 0);  // and whether all that have it are wanted
                }
                before += c[i];
            }
        }
        __syncthreads();
        const uint32_t total = L.found[0], value = L.found[1], rest = L.found[2];
        if (total <= even) {  // every one that agrees so far; at first those are all candidates
            all = first;
            break;
        }
        bar |= static_cast<uint64_t>(value) << shift;
        mask |= uint64_t{255} << shift;
        even = rest & 0x7fffffffu;
        if (rest >> 31 || shift == 0) break;
        shift = max(shift - 8, 0);
    }
    // In ascending order: the place of a block is the number of taken ones before it.
    RCH_GLOBAL int32_t* list = gout<int32_t>(B.lists_ptr) + (static_cast<int64_t>(blockIdx.x) * B.heads + head) * B.width;
    int written = 0;
    uint32_t equal = 0;
    for (int base = R.first; base < R.last; base += THREADS) {
        const int block = base + t;
        bool taken = false, same = false;
        if (block < R.last && page_held(B, page_of(B, R, by_page.quotient(block)))) {
            if (all || !chosen_by_score(block)) {
                taken = true;
            } else if (mask) {  // (none is wanted otherwise, and there may be no scores)
                const uint64_t n = number(block) & mask;
                taken = n > bar;
                same = n == bar;
            }
        }
        // Equal ones by their number.
        const uint64_t alike = __ballot(same);
        if (lane == 0) L.waves[0][wave] = __popcll(alike);
        __syncthreads();
        uint32_t before = equal;
        for (int w = 0; w < THREADS / 64; ++w) {
            if (w < wave) before += L.waves[0][w];
            equal += L.waves[0][w];
        }
        before += __popcll(alike & ((uint64_t{1} << lane) - 1));
        taken = taken || (same && before < even);
        const uint64_t votes = __ballot(taken);
        if (lane == 0) L.waves[1][wave] = __popcll(votes);
        __syncthreads();
        int place = written;
        for (int w = 0; w < THREADS / 64; ++w) {
            if (w < wave) place += L.waves[1][w];
            written += L.waves[1][w];
        }
        place += __popcll(votes & ((uint64_t{1} << lane) - 1));
        if (taken && place < B.width) list[place] = block;
    }
    for (int at = written + t; at < B.width; at += THREADS) list[at] = -1;
}

// Without scratch, runs of at most kTogether scored blocks: one workgroup to a run and key head.
template <int DT, int V, int THREADS>
__global__ void __launch_bounds__(THREADS) blocks_select_kernel(const rch_blocks B) {
    __shared__ double pooled[256];
    __shared__ union {
        double sums[256 * V];
        uint64_t numbers[kTogether];
    } S;
    __shared__ Taking L;
    const Run R = run_of(B, blockIdx.x);
    const int head = blockIdx.y;
    if (B.top && R.scored < R.scored_end) {
        pool_queries<DT, V, THREADS>(B, R, head, S.sums, pooled);
        score_blocks<DT, V, THREADS>(B, R, head, R.scored, R.scored_end, pooled, [&](int block, uint64_t number) { S.numbers[block - R.scored] = number; });
        __syncthreads();
    }
    take_blocks<THREADS>(B, R, head, L, [&](int block) { return S.numbers[block - R.scored]; });
}

// With scratch: workgroups of their own score kScored blocks each, and another launch takes them.
template <int DT, int V>
__global__ void __launch_bounds__(256) blocks_score_kernel(const rch_blocks B) {
    __shared__ double pooled[256], sums[256 * V];
    const Run R = run_of(B, blockIdx.x);
    const int head = blockIdx.z, begin = R.scored + blockIdx.y * kScored, end = min(begin + kScored, R.scored_end);
    if (begin >= end) return;
    pool_queries<DT, V, 256>(B, R, head, sums, pooled);
    RCH_GLOBAL uint64_t* out = gout<uint64_t>(B.scores_ptr) + (static_cast<int64_t>(blockIdx.x) * B.heads + head) * B.scores - R.scored;
    score_blocks<DT, V, 256>(B, R, head, begin, end, pooled, [&](int block, uint64_t number) { out[block] = number; });
}

// (1024 threads to a choice among up to 1024 blocks for 4 single tokens: 30.0 us with its score and attention, 512 30.1, 256 32.3)
__global__ void __launch_bounds__(1024) blocks_take_kernel(const rch_blocks B) {
    __shared__ uint64_t kept[kTogether];
    __shared__ Taking L;
    const Run R = run_of(B, blockIdx.x);
    const int head = blockIdx.y, count = R.scored_end - R.scored;
    const RCH_GLOBAL uint64_t* numbers = gin<uint64_t>(B.scores_ptr) + (static_cast<int64_t>(blockIdx.x) * B.heads + head) * B.scores;
    if (count <= kTogether) {
        if (B.top)
            for (int i = threadIdx.x; i < count; i += 1024) kept[i] = numbers[i];
        __syncthreads();
        take_blocks<1024>(B, R, head, L, [&](int block) { return kept[block - R.scored]; });
    } else {
        take_blocks<1024>(B, R, head, L, [&](int block) { return numbers[block - R.scored]; });
    }
}

// What both entry points need of the pools' description.
int invalid(const rch_blocks& B, int dtype, const char* what) {
    if (dtype != RCH_DT_F32 && dtype != RCH_DT_F16 && dtype != RCH_DT_BF16) return fail(RCH_E_CONFIG, "%s: dtype must be f32, f16 or bf16", what);
    if (B.heads < 1 || B.heads > 65535 || B.head_dim < 1 || B.head_dim > RCH_ATTEND_MAX_DIM || B.pages < 1 || B.page_tokens < 1 || B.block_tokens < 1
        || B.block_tokens > RCH_BLOCKS_TOKENS || B.page_tokens % B.block_tokens || B.pages > 0x7fffffff || B.page_tokens > 0x7fffffff || B.pages * B.page_tokens > 0x7fffffff)
        return fail(RCH_E_CONFIG, "%s: invalid sizes", what);
    return RCH_OK;
}

template <int DT, int FMT>
int update(const rch_blocks& B, hipStream_t stream) {
    // Tokens of a workgroup: one while that makes few of them, so that the touched blocks of single tokens run at once, and so
    // many that no workgroup only looks for blocks (1 / 8 / 64 to a workgroup: a chunk of 4680 tokens in blocks of 120 takes
    // 46 / 9.3 / 6.2 us, 32 single tokens 3.9 / 12.3 / 40.8; by this rule 5.7 and 4.0).
    const int64_t wanted = B.tokens * B.heads / 1024;
    const int share = static_cast<int>(wanted < 1 ? 1 : wanted > 64 ? 64 : wanted);
    const dim3 grid(static_cast<uint32_t>((B.tokens + share - 1) / share), static_cast<uint32_t>(B.heads));
    const int64_t bytes = Row<DT, FMT, 8>::kBytes, piece = FMT == RCH_CODES_NONE ? 16 : 8;
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

template <int DT, int V>
int select_rows(const rch_blocks& B, hipStream_t stream) {
    const dim3 grid(static_cast<uint32_t>(B.n_runs), static_cast<uint32_t>(B.heads));
    if (!B.scores_ptr) {
        hipLaunchKernelGGL((blocks_select_kernel<DT, V, 256>), grid, dim3(256), 0, stream, B);
        return check_launch("rch_blocks_select");
    }
    const dim3 scored(static_cast<uint32_t>(B.n_runs), static_cast<uint32_t>((B.scores + kScored - 1) / kScored), static_cast<uint32_t>(B.heads));
    hipLaunchKernelGGL((blocks_score_kernel<DT, V>), scored, dim3(256), 0, stream, B);
    const int status = check_launch("rch_blocks_select (scores)");
    if (status != RCH_OK) return status;
    hipLaunchKernelGGL(blocks_take_kernel, grid, dim3(1024), 0, stream, B);
    return check_launch("rch_blocks_select");
}

template <int DT>
int select(const rch_blocks& B, hipStream_t stream) {
    const int64_t size = DT == RCH_DT_F32 ? 4 : 2;
    const bool wide = B.head_dim % 8 == 0 && (B.q_ptr | B.means_ptr) % 16 == 0 && (B.q_token_stride | B.q_head_stride) * size % 16 == 0;
    return wide ? select_rows<DT, 8>(B, stream) : select_rows<DT, 1>(B, stream);
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
    if (!B.means_ptr || !B.q_ptr || !B.plan_ptr || !B.lists_ptr || (B.scores > kTogether && !B.scores_ptr) || (B.scores_ptr && !B.scores) || B.scores_ptr % 8)
        return fail(RCH_E_CONFIG, "rch_blocks_select: null or misaligned address");
    hipStream_t s = as_stream(stream);
    if (dtype == RCH_DT_F32) return select<RCH_DT_F32>(B, s);
    return dtype == RCH_DT_F16 ? select<RCH_DT_F16>(B, s) : select<RCH_DT_BF16>(B, s);
}

}  // extern "C"
