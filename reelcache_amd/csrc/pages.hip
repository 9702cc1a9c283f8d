// Copies of cache pages: dst page = src page for a list of moves, in every pool (the K and the V of
// every layer) in one launch.
//
// Bound: memory, one read and one write of each moved byte.  The moves travel in the kernel's
// arguments (no upload, and a captured call carries them); a pool's page is `segments` runs of
// `rows` token rows, which are one piece of memory where the rows lie next to each other.  A
// workgroup copies 16 KiB of one page of one pool; a thread has four 16-byte loads in flight.  Twelve pages
// of 256 tokens x 12 heads x 128 bf16 in 60 pools (1.13 GB read and written) take 218 us, 5.2 TB/s; eight
// forks of 96 rows (159 MB) 36 us, 4.4 TB/s.
#include "common.h"

namespace rch {

namespace {

constexpr int kThreads = 256, kUnroll = 4;

struct Moves {
    int32_t src[RCH_PAGE_MOVES], dst[RCH_PAGE_MOVES], rows[RCH_PAGE_MOVES];
};

// U: the unit of a copy (16, 4, 2 or 1 bytes), whatever divides every address and row.
template <typename U>
__global__ void __launch_bounds__(kThreads) pages_copy_kernel(rch_pages P, const Moves moves, int chunks) {
    const int move = blockIdx.y;
    const int64_t pool = gin<int64_t>(P.pools_ptr)[blockIdx.z];
    const int64_t rows = moves.rows[move];
    const int64_t src = pool + moves.src[move] * P.page_stride, dst = pool + moves.dst[move] * P.page_stride;
    const bool joined = P.row_stride == P.row_bytes;
    const int64_t run = rows * (P.row_bytes / static_cast<int64_t>(sizeof(U)));  // units of a segment
    const int64_t units = run * P.segments, row_units = P.row_bytes / static_cast<int64_t>(sizeof(U));
    for (int64_t base = static_cast<int64_t>(blockIdx.x) * kThreads * kUnroll; base < units;
         base += static_cast<int64_t>(chunks) * kThreads * kUnroll) {
        U value[kUnroll];
        int64_t at[kUnroll];
#pragma unroll
        for (int i = 0; i < kUnroll; ++i) {
            const int64_t unit = base + i * kThreads + threadIdx.x;
            at[i] = -1;
            if (unit >= units) continue;
            if (joined && P.segments == 1) {
                at[i] = unit * static_cast<int64_t>(sizeof(U));
            } else {
                const uint32_t u = static_cast<uint32_t>(unit), segment = u / static_cast<uint32_t>(run);
                const uint32_t rest = u - segment * static_cast<uint32_t>(run);
                const uint32_t row = rest / static_cast<uint32_t>(row_units);
                at[i] = segment * P.segment_stride + row * P.row_stride
                        + (rest - row * static_cast<uint32_t>(row_units)) * static_cast<int64_t>(sizeof(U));
            }
            value[i] = *gin<U>(src + at[i]);
        }
#pragma unroll
        for (int i = 0; i < kUnroll; ++i)
            if (at[i] >= 0) *gout<U>(dst + at[i]) = value[i];
    }
}

// Words that travel in the launch's arguments: a table of a few hundred entries reaches the device without
// pinned memory and without a copy engine (1.2-5 us on the device, the launch's latency).
struct Words {
    int32_t word[RCH_ARGUMENT_WORDS];
};
__global__ void __launch_bounds__(256) words_store_kernel(int64_t to, const Words words, int count) {
    for (int i = threadIdx.x; i < count; i += 256) gout<int32_t>(to)[i] = words.word[i];
}

// Runs of ascending words: run i writes first, first + 1, .. to `count` words from `at`.  The slots of a step's new
// tokens are one run for each sequence and page, so thousands of them travel in one launch's arguments.
struct Runs {
    int32_t first[RCH_ARGUMENT_RUNS], count[RCH_ARGUMENT_RUNS], at[RCH_ARGUMENT_RUNS];
};
__global__ void __launch_bounds__(256) runs_store_kernel(int64_t to, const Runs runs) {
    const int run = blockIdx.y;
    const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;  // past 2^31 behind the longest runs
    if (i < runs.count[run]) gout<int32_t>(to)[runs.at[run] + i] = static_cast<int32_t>(runs.first[run] + i);
}

}  // namespace

}  // namespace rch

extern "C" {

int rch_words_store(void* words_dev, const int32_t* words_host, int count, void* stream) {
    using namespace rch;
    if (count < 0 || (count > 0 && (!words_dev || !words_host))) return fail(RCH_E_CONFIG, "rch_words_store: invalid arguments");
    for (int first = 0; first < count; first += RCH_ARGUMENT_WORDS) {
        const int n = count - first < RCH_ARGUMENT_WORDS ? count - first : RCH_ARGUMENT_WORDS;
        Words words;
        for (int i = 0; i < n; ++i) words.word[i] = words_host[first + i];
        const int64_t to = reinterpret_cast<int64_t>(words_dev) + 4 * static_cast<int64_t>(first);
        hipLaunchKernelGGL(words_store_kernel, dim3(1), dim3(256), 0, as_stream(stream), to, words, n);
        const int status = check_launch("rch_words_store");
        if (status != RCH_OK) return status;
    }
    return RCH_OK;
}

int rch_runs_store(void* words_dev, const int32_t* runs_host, int n_runs, int64_t words, void* stream) {
    using namespace rch;
    if (n_runs < 0 || words < 0 || words > 0x7fffffff || (n_runs > 0 && (!words_dev || !runs_host)))
        return fail(RCH_E_CONFIG, "rch_runs_store: invalid arguments");
    int64_t at = 0;
    for (int i = 0; i < n_runs; ++i) {
        if (runs_host[2 * i + 1] < 0) return fail(RCH_E_CONFIG, "rch_runs_store: run %d has a negative count", i);
        at += runs_host[2 * i + 1];
    }
    if (at != words) return fail(RCH_E_CONFIG, "rch_runs_store: the runs have %lld words, not %lld", static_cast<long long>(at), static_cast<long long>(words));
    at = 0;
    for (int first = 0; first < n_runs; first += RCH_ARGUMENT_RUNS) {
        const int n = n_runs - first < RCH_ARGUMENT_RUNS ? n_runs - first : RCH_ARGUMENT_RUNS;
        Runs runs;
        int32_t longest = 0;
        for (int i = 0; i < n; ++i) {
            runs.first[i] = runs_host[2 * (first + i)];
            runs.count[i] = runs_host[2 * (first + i) + 1];
            runs.at[i] = static_cast<int32_t>(at);
            at += runs.count[i];
            longest = runs.count[i] > longest ? runs.count[i] : longest;
        }
        if (longest == 0) continue;
        const dim3 grid(static_cast<uint32_t>((static_cast<int64_t>(longest) + 255) / 256), static_cast<uint32_t>(n));
        hipLaunchKernelGGL(runs_store_kernel, grid, dim3(256), 0, as_stream(stream), reinterpret_cast<int64_t>(words_dev), runs);
        const int status = check_launch("rch_runs_store");
        if (status != RCH_OK) return status;
    }
    return RCH_OK;
}

int rch_pages_copy(const rch_pages* pages_host, const int32_t* moves_host, int n_moves, void* stream) {
    using namespace rch;
    if (!pages_host || n_moves < 0 || (n_moves > 0 && !moves_host))
        return fail(RCH_E_CONFIG, "rch_pages_copy: invalid arguments");
    const rch_pages& P = *pages_host;
    if (!P.pools_ptr || P.pools < 1 || P.pools > 65535 || P.pages < 1 || P.page_rows < 1 || P.segments < 1
        || P.row_bytes < 1 || P.row_stride < P.row_bytes || P.page_stride < 0)
        return fail(RCH_E_CONFIG, "rch_pages_copy: invalid pool description");
    if (P.segments * P.page_rows * P.row_bytes >= (int64_t{1} << 31))
        return fail(RCH_E_UNSUPPORTED, "rch_pages_copy: a page of 2 GiB or more");
    for (int i = 0; i < n_moves; ++i) {
        const int32_t* m = moves_host + 3 * i;
        if (m[0] < 0 || m[0] >= P.pages || m[1] < 0 || m[1] >= P.pages || m[0] == m[1] || m[2] < 0 || m[2] > P.page_rows)
            return fail(RCH_E_CONFIG, "rch_pages_copy: move %d (%d -> %d, %d rows) is outside the pool", i, m[0], m[1], m[2]);
    }
    const int64_t mix = P.alignment | P.page_stride | P.segment_stride | P.row_stride | P.row_bytes;
    const int unit = mix % 16 == 0 ? 16 : (mix % 4 == 0 ? 4 : (mix % 2 == 0 ? 2 : 1));
    for (int first = 0; first < n_moves; first += RCH_PAGE_MOVES) {
        const int count = n_moves - first < RCH_PAGE_MOVES ? n_moves - first : RCH_PAGE_MOVES;
        Moves moves;
        int64_t most = 0;
        for (int i = 0; i < count; ++i) {
            const int32_t* m = moves_host + 3 * (first + i);
            moves.src[i] = m[0];
            moves.dst[i] = m[1];
            moves.rows[i] = m[2];
            most = m[2] > most ? m[2] : most;
        }
        if (most == 0) continue;
        const int64_t units = P.segments * most * P.row_bytes / unit;
        const int64_t chunks = (units + kThreads * kUnroll - 1) / (kThreads * kUnroll);
        const dim3 grid(static_cast<uint32_t>(chunks), static_cast<uint32_t>(count), static_cast<uint32_t>(P.pools));
        hipStream_t s = as_stream(stream);
        const int c = static_cast<int>(chunks);
        switch (unit) {
            case 16: hipLaunchKernelGGL(pages_copy_kernel<u4>, grid, dim3(kThreads), 0, s, P, moves, c); break;
            case 4: hipLaunchKernelGGL(pages_copy_kernel<uint32_t>, grid, dim3(kThreads), 0, s, P, moves, c); break;
            case 2: hipLaunchKernelGGL(pages_copy_kernel<uint16_t>, grid, dim3(kThreads), 0, s, P, moves, c); break;
            default: hipLaunchKernelGGL(pages_copy_kernel<uint8_t>, grid, dim3(kThreads), 0, s, P, moves, c); break;
        }
        const int status = check_launch("rch_pages_copy");
        if (status != RCH_OK) return status;
    }
    return RCH_OK;
}

}  // extern "C"
