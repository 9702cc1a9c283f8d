// Rotation of queries and keys by positions of several axes, and the store of new tokens into the
// slots of a paged cache (the same rotation with a scattered destination, or a plain copy).
//
// A pair (a, b) of a head of token t, at pair column j, turns by the table's angle at the token's
// place on j's axis: a' = a cos - b sin, b' = a sin + b cos.  The two products of each are rounded
// apart (no FMA) and the result is rounded once to the tensor's type: the arithmetic of the restore
// kernels, so a key stored here has the bits that a restored one has.
//
// Bound: memory, one read and one write of each value.  A thread holds one 8-channel piece (two for
// the "half" pairing) of a token and walks over heads of it, so the places, table rows and cosines
// are fetched once for all of those heads; neighbouring threads hold neighbouring pieces, so a wave
// reads and writes whole rows of a head.  Four heads to a thread, their loads in flight together: q and k
// of 16 / 1024 / 4680 / 18720 tokens x 12 heads x 128 bf16 take 4.6 / 5.7 / 12.4 / 36.3 us (the last
// 6.3 TB/s, mostly from the caches), with one head 4.5 / 6.6 / 18.0 / 57.3, two 4.5 / 5.8 / 13.8 / 38.6,
// eight 4.4 / 5.9 / 12.2 / 36.5.
#include "common.h"

namespace rch {

namespace {

constexpr int kMaxRotary = 4, kHeads = 4;

struct RotaryJobs {
    rch_rotary_job job[kMaxRotary];
};

template <int DT>
struct Element;
template <>
struct Element<RCH_DT_F32> {
    typedef float type;
};
template <>
struct Element<RCH_DT_F16> {
    typedef _Float16 type;
};
template <>
struct Element<RCH_DT_BF16> {
    typedef __bf16 type;
};

// N values from / to consecutive elements, in 16- or 8-byte pieces where the width promises their alignment (two
// fp32 values do not: their rows may start at any element).
template <typename T, int N>
struct Piece {
    T v[N];
};
template <typename T, int N>
__device__ __forceinline__ Piece<T, N> load_piece(const RCH_GLOBAL T* p) {
    Piece<T, N> out;
    if constexpr (N * sizeof(T) % 16 == 0) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(N * sizeof(T) / 16); ++i) {
            const u4 raw = reinterpret_cast<const RCH_GLOBAL u4*>(p)[i];
            __builtin_memcpy(reinterpret_cast<char*>(out.v) + 16 * i, &raw, 16);
        }
    } else if constexpr (N == 4 && sizeof(T) == 2) {
        const u2 raw = *reinterpret_cast<const RCH_GLOBAL u2*>(p);
        __builtin_memcpy(out.v, &raw, 8);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) out.v[i] = p[i];
    }
    return out;
}
template <typename T, int N>
__device__ __forceinline__ void store_piece(RCH_GLOBAL T* p, const Piece<T, N>& in) {
    if constexpr (N * sizeof(T) % 16 == 0) {
#pragma unroll
        for (int i = 0; i < static_cast<int>(N * sizeof(T) / 16); ++i) {
            u4 raw;
            __builtin_memcpy(&raw, reinterpret_cast<const char*>(in.v) + 16 * i, 16);
            reinterpret_cast<RCH_GLOBAL u4*>(p)[i] = raw;
        }
    } else if constexpr (N == 4 && sizeof(T) == 2) {
        u2 raw;
        __builtin_memcpy(&raw, in.v, 8);
        *reinterpret_cast<RCH_GLOBAL u2*>(p) = raw;
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = in.v[i];
    }
}

__device__ __forceinline__ void rotate_pair(float& e, float& o, float c, float s) {
    const float re = __fsub_rn(__fmul_rn(e, c), __fmul_rn(o, s));
    const float ro = __fadd_rn(__fmul_rn(e, s), __fmul_rn(o, c));
    e = re;
    o = ro;
}

// One piece is V channels: V / 2 interleaved pairs, or V pairs of the half pairing (channels j and
// pairs + j: two pieces).  V = 8 and V = 4 need rows aligned to a piece (16 bytes at most) and widths of
// whole pieces; V = 2 (interleaved) and 1 (half, or no rotation) take everything else.
// A thread takes U heads.
template <int DT, bool HALF, int V>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryJobs jobs) {
    typedef typename Element<DT>::type T;
    constexpr int U = kHeads;
    const rch_rotary_job& J = jobs.job[blockIdx.z];
    const int pairs = static_cast<int>(J.pairs), dim = static_cast<int>(J.head_dim);
    // Work items of a token's head: pieces that turn, then pieces that are copied.
    const int turning = HALF ? pairs / V : 2 * pairs / V;
    const int pieces = turning + (dim - 2 * pairs) / V;
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
    const int64_t at = unit / pieces;  // batch * tokens + token
    const int piece = static_cast<int>(unit - at * pieces);
    const int head0 = blockIdx.y * U;
    if (at >= J.batch * J.tokens || head0 >= J.heads) return;
    const int64_t batch = at / J.tokens, token = at - batch * J.tokens;

    int64_t to;
    if (J.slots_ptr) {
        // A slot outside the pool (padding) drops the token.
        const int64_t slot = gin<int32_t>(J.slots_ptr)[token];
        if (slot < 0 || slot >= J.slots) return;
        const int64_t page = slot / J.page_tokens;
        to = page * J.dst_batch_stride + (slot - page * J.page_tokens) * J.dst_token_stride;
    } else {
        to = batch * J.dst_batch_stride + token * J.dst_token_stride;
    }
    const RCH_GLOBAL T* src = gin<T>(J.src_ptr) + batch * J.src_batch_stride + token * J.src_token_stride;
    RCH_GLOBAL T* dst = gout<T>(J.dst_ptr) + to;
    const int64_t src_head = J.src_head_stride, dst_head = J.dst_head_stride;
    const int heads = min(static_cast<int>(J.heads) - head0, U);
    src += head0 * src_head;
    dst += head0 * dst_head;

    if (piece >= turning) {  // channels behind the rotated ones
        const int channel = 2 * pairs + (piece - turning) * V;
        for (int h = 0; h < heads; ++h)
            store_piece<T, V>(dst + h * dst_head + channel, load_piece<T, V>(src + h * src_head + channel));
        return;
    }

    // The token's place on each axis; a row outside its axis turns to NaN (nothing is read there).
    int row[3];
    if (J.rows_ptr) {
        const RCH_GLOBAL int32_t* r = gin<int32_t>(J.rows_ptr) + batch * J.rows_batch_stride + token * J.rows_token_stride;
#pragma unroll
        for (int a = 0; a < 3; ++a) row[a] = a < J.axes ? r[a * J.rows_axis_stride] : 0;
    } else if (J.axes == 3) {
        const int t = static_cast<int>(token), plane = static_cast<int>(J.grid_h * J.grid_w), w = static_cast<int>(J.grid_w);
        const int f = t / plane, y = (t - f * plane) / w;
        row[0] = static_cast<int>(J.row_t) + f;
        row[1] = static_cast<int>(J.row_h) + y;
        row[2] = static_cast<int>(J.row_w) + t - f * plane - y * w;
    } else {
        row[0] = static_cast<int>(J.row_t + token);
        row[1] = row[2] = 0;
    }
    const int bound1 = static_cast<int>(J.sec_t), bound2 = bound1 + static_cast<int>(J.sec_h);
    constexpr int P = HALF ? V : V / 2;
    const int j0 = piece * P;
    float c[P], s[P];
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const int j = j0 + i, axis = J.axes == 1 ? 0 : (j < bound1 ? 0 : (j < bound2 ? 1 : 2));
        const int r = axis == 0 ? row[0] : (axis == 1 ? row[1] : row[2]);
        const int64_t limit = axis == 0 ? J.limit_t : (axis == 1 ? J.limit_h : J.limit_w);
        f2 pair = {__builtin_nanf(""), __builtin_nanf("")};
        if (r >= 0 && r < limit) pair = gin<f2>(J.pairs_ptr)[static_cast<int64_t>(r) * pairs + j];
        c[i] = pair[0];
        s[i] = J.inverse ? -pair[1] : pair[1];
    }
    const int64_t first = HALF ? j0 : 2 * j0;
    Piece<T, V> a[U], b[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int g = min(u, heads - 1);
        a[u] = load_piece<T, V>(src + g * src_head + first);
        if constexpr (HALF) b[u] = load_piece<T, V>(src + g * src_head + first + pairs);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            T& x = HALF ? a[u].v[i] : a[u].v[2 * i];
            T& y = HALF ? b[u].v[i] : a[u].v[2 * i + 1];
            float e = static_cast<float>(x), o = static_cast<float>(y);
            rotate_pair(e, o, c[i], s[i]);
            x = static_cast<T>(e);
            y = static_cast<T>(o);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        if (u >= heads) break;
        store_piece<T, V>(dst + u * dst_head + first, a[u]);
        if constexpr (HALF) store_piece<T, V>(dst + u * dst_head + first + pairs, b[u]);
    }
}

template <int DT>
void launch(const RotaryJobs& jobs, bool half, int width, dim3 grid, hipStream_t stream) {
    if (half) {
        if (width == 8) hipLaunchKernelGGL((rotary_kernel<DT, true, 8>), grid, dim3(256), 0, stream, jobs);
        else if (width == 4) hipLaunchKernelGGL((rotary_kernel<DT, true, 4>), grid, dim3(256), 0, stream, jobs);
        else hipLaunchKernelGGL((rotary_kernel<DT, true, 1>), grid, dim3(256), 0, stream, jobs);
    } else {
        if (width == 8) hipLaunchKernelGGL((rotary_kernel<DT, false, 8>), grid, dim3(256), 0, stream, jobs);
        else if (width == 4) hipLaunchKernelGGL((rotary_kernel<DT, false, 4>), grid, dim3(256), 0, stream, jobs);
        else hipLaunchKernelGGL((rotary_kernel<DT, false, 2>), grid, dim3(256), 0, stream, jobs);
    }
}

}  // namespace

}  // namespace rch

extern "C" {

int rch_rotary_size(void) { return static_cast<int>(sizeof(rch_rotary_job)); }

int rch_rotary(const rch_rotary_job* jobs_host, int n_jobs, int dtype, int pairing, void* stream) {
    using namespace rch;
    if (!jobs_host || n_jobs < 1 || n_jobs > kMaxRotary)
        return fail(RCH_E_CONFIG, "rch_rotary: 1 to %d tensors", kMaxRotary);
    if (dtype != RCH_DT_F32 && dtype != RCH_DT_F16 && dtype != RCH_DT_BF16)
        return fail(RCH_E_CONFIG, "rch_rotary: dtype must be f32, f16 or bf16");
    if (pairing != RCH_PAIRS_INTERLEAVED && pairing != RCH_PAIRS_HALF)
        return fail(RCH_E_CONFIG, "rch_rotary: unknown pairing %d", pairing);
    bool half = pairing == RCH_PAIRS_HALF, turns = false;
    for (int i = 0; i < n_jobs; ++i) turns = turns || jobs_host[i].pairs > 0;
    half = half || !turns;  // a plain copy has no pairs to keep together
    const int64_t size = dtype == RCH_DT_F32 ? 4 : 2;
    RotaryJobs jobs;
    int64_t mix = 0, channels = 0;
    for (int i = 0; i < n_jobs; ++i) {
        const rch_rotary_job& J = jobs.job[i] = jobs_host[i];
        if (J.batch < 0 || J.tokens < 0 || J.heads < 1 || J.head_dim < 1 || J.pairs < 0 || 2 * J.pairs > J.head_dim
            || J.head_dim > (1 << 20) || J.heads > (1 << 20) || J.tokens > 0x7fffffff || J.batch > 0x7fffffff)
            return fail(RCH_E_CONFIG, "rch_rotary: invalid sizes of tensor %d", i);
        if (J.pairs > 0 && ((J.axes != 1 && J.axes != 3) || !J.pairs_ptr
                            || (!J.rows_ptr && J.axes == 3 && (J.grid_h < 1 || J.grid_w < 1))))
            return fail(RCH_E_CONFIG, "rch_rotary: invalid positions of tensor %d", i);
        if (J.slots_ptr && (J.batch != 1 || J.page_tokens < 1))
            return fail(RCH_E_CONFIG, "rch_rotary: slots take one batch and a page size (tensor %d)", i);
        const int64_t strides = J.src_batch_stride | J.src_token_stride | J.src_head_stride | J.dst_batch_stride
                                | J.dst_token_stride | J.dst_head_stride;
        mix |= J.src_ptr | J.dst_ptr | strides * size;
        channels |= J.head_dim | (half ? J.pairs : 2 * J.pairs);  // every width a piece divides
    }
    // The widest piece that divides every width and whose rows are aligned.
    const int width = channels % 8 == 0 && mix % 16 == 0 ? 8
                      : channels % 4 == 0 && mix % (4 * size) == 0 ? 4 : half ? 1 : 2;
    if (width == 2 && channels % 2) return fail(RCH_E_UNSUPPORTED, "rch_rotary: interleaved pairs need an even head_dim");
    int64_t units = 0, heads = 0;
    for (int i = 0; i < n_jobs; ++i) {
        const rch_rotary_job& J = jobs.job[i];
        const int v = width;
        const int64_t pieces = (half ? J.pairs / v : 2 * J.pairs / v) + (J.head_dim - 2 * J.pairs) / v;
        const int64_t n = J.batch * J.tokens * pieces;
        units = n > units ? n : units;
        heads = J.heads > heads ? J.heads : heads;
    }
    if (units == 0) return RCH_OK;
    const int64_t blocks = (units + 255) / 256, groups = (heads + kHeads - 1) / kHeads;
    if (blocks > 0x7fffffff || groups > 65535) return fail(RCH_E_CONFIG, "rch_rotary: grid too large");
    const dim3 grid(static_cast<uint32_t>(blocks), static_cast<uint32_t>(groups), static_cast<uint32_t>(n_jobs));
    hipStream_t s = as_stream(stream);
    switch (dtype) {
        case RCH_DT_F32: launch<RCH_DT_F32>(jobs, half, width, grid, s); break;
        case RCH_DT_F16: launch<RCH_DT_F16>(jobs, half, width, grid, s); break;
        default: launch<RCH_DT_BF16>(jobs, half, width, grid, s); break;
    }
    return check_launch("rch_rotary");
}

}  // extern "C"
