// The global norm of a model's gradients, and their clipping.
//
//   n = sqrt(sum over all tensors of g^2),   c = min(1, max_norm / (n + 1e-6)),   g' = c g.
//
// Squares and their sums are FP64: those of FP32 overflow from 2e19 on and
// vanish below 1e-23, and a sum of a billion of them is exact to the last bits
// of the norm.  Every sum is made in a fixed order.
//
// The tensors' addresses are arguments of the launch, so that nothing is copied
// to the device before it and a captured graph keeps them.  Workgroups take the
// tensors' chunks in turn, one FP64 sum each; those that scale add up the few
// thousand sums for themselves, which costs less than a launch between.
//
// Bound by HBM: 1.1 billion BF16 gradients 379 us (5.85 TB/s); 432 million clipped in place 496 us (5.2 TB/s), to FP32 150
// for the norm and 531 for the scaling, which reads 0.86 and writes 1.73 GB.  Small models wait for two trips of latency
// (227 tensors, 2.6 million gradients: 14 us from a graph) and for the host.
#include <algorithm>
#include <type_traits>
#include <vector>

#include "bdm_common.h"
#include "selection_ops.h"

namespace bdm {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kChunk = 16384;       // elements of one tensor that a workgroup takes at a time
constexpr int64_t kMostParts = 2048;  // sums of a call: eight workgroups a CU
constexpr uint32_t kSizeMask = (1u << 30) - 1;

// Tensors of one launch: chunk k belongs to the first tensor whose `end` is above it.  The size's upper bits hold the
// types: bit 31 the data's, bit 30 the output's, set for BF16.
template <bool OUTPUTS>
struct Table {
    static constexpr int kTensors = OUTPUTS ? 160 : 240;
    const void *data[kTensors];
    void *out[OUTPUTS ? kTensors : 1];
    uint32_t size[kTensors], end[kTensors];
    int32_t count;
};
static_assert(sizeof(Table<true>) <= 4000 && sizeof(Table<false>) <= 4000, "the arguments of a launch are at most 4 KiB");

template <typename Table>
__device__ __forceinline__ int tensor_of(const Table &b, uint32_t chunk) {
    int low = 0, high = b.count - 1;
    while (low < high) {
        const int middle = (low + high) / 2;
        if (chunk < b.end[middle])
            high = middle;
        else
            low = middle + 1;
    }
    return low;
}

__device__ __forceinline__ double block_sum(double x, double *shared) {
#pragma unroll
    for (int step = kWave / 2; step; step >>= 1) x += __shfl_xor(x, step, kWave);
    if (threadIdx.x % kWave == 0) shared[threadIdx.x / kWave] = x;
    __syncthreads();
    x = shared[0];
    for (int i = 1; i < kWaves; ++i) x += shared[i];
    return x;
}

// The sum of squares of n <= kChunk elements, this thread's share.
template <typename T>
__device__ __forceinline__ double squares(const T *g, int n) {
    constexpr int VE = Vec<T>::kSize, U = 8;
    double sums[2] = {0, 0};
    const int vectors = n / VE;
    const auto add = [&](u32x4 raw) {
        float v[VE];
        Vec<T>::widen(raw, v);
#pragma unroll
        for (int j = 0; j < VE; ++j) sums[j % 2] = fma(double(v[j]), double(v[j]), sums[j % 2]);
    };
    int at = threadIdx.x;
    for (; at + (U - 1) * kThreads < vectors; at += U * kThreads) {
        u32x4 raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = reinterpret_cast<const AnyVector<T> *>(g + (at + u * kThreads) * VE)->bits;
#pragma unroll
        for (int u = 0; u < U; ++u) add(raw[u]);
    }
    for (; at < vectors; at += kThreads) add(reinterpret_cast<const AnyVector<T> *>(g + at * VE)->bits);
    const int odd = vectors * VE + int(threadIdx.x);
    if (odd < n) {
        const double x = double(to_f32(g[odd]));
        sums[0] = fma(x, x, sums[0]);
    }
    return sums[0] + sums[1];
}

__global__ __launch_bounds__(kThreads) void squares_kernel(Table<false> b, uint32_t chunks, double *parts) {
    __shared__ double shared[kWaves];
    double sum = 0;
    for (uint32_t chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
        const int i = tensor_of(b, chunk);
        const int64_t begin = int64_t(chunk - (i ? b.end[i - 1] : 0)) * kChunk;
        const int n = int(min(int64_t(b.size[i] & kSizeMask) - begin, int64_t(kChunk)));
        sum += b.size[i] >> 31 ? squares(static_cast<const bf16_t *>(b.data[i]) + begin, n)
                               : squares(static_cast<const float *>(b.data[i]) + begin, n);
    }
    sum = block_sum(sum, shared);
    if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

// The norm and the factor from the parts, in every thread of a workgroup.
__device__ __forceinline__ float factor_of(const double *parts, int count, double max_norm, double &norm) {
    __shared__ double shared[kWaves];
    double sum = 0;
#pragma unroll 8
    for (int i = threadIdx.x; i < count; i += kThreads) sum += parts[i];
    norm = sqrt(block_sum(sum, shared));
    const double c = max_norm / (norm + 1e-6);
    return c > 1 ? 1.f : float(c);
}

__global__ __launch_bounds__(kThreads) void norm_kernel(const double *parts, int count, double max_norm, float *norm,
                                                        float *scale) {
    double n;
    const float c = factor_of(parts, count, max_norm, n);
    if (threadIdx.x == 0) {
        *norm = float(n);
        if (scale) *scale = c;
    }
}

// N elements that lie together, 8 or 16 bytes.
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

template <int N>
__device__ __forceinline__ void load_some(const bf16_t *g, float (&v)[N]) {
    using Bits = std::conditional_t<N == 8, u32x4_any, u32x2_any>;
    const Bits raw = *reinterpret_cast<const Bits *>(g);
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
        v[2 * j] = __uint_as_float(raw[j] << 16);
        v[2 * j + 1] = __uint_as_float(raw[j] & 0xffff0000u);
    }
}
template <int N>
__device__ __forceinline__ void load_some(const float *g, float (&v)[N]) {
    static_assert(N == 4);
    const u32x4_any raw = *reinterpret_cast<const u32x4_any *>(g);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = __uint_as_float(raw[j]);
}
template <int N>
__device__ __forceinline__ void store_some(bf16_t *out, const float (&v)[N]) {
    using Bits = std::conditional_t<N == 8, u32x4_any, u32x2_any>;
    Bits bits;
#pragma unroll
    for (int j = 0; j < N / 2; ++j) bits[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
    __builtin_nontemporal_store(bits, reinterpret_cast<Bits *>(out));
}
template <int N>
__device__ __forceinline__ void store_some(float *out, const float (&v)[N]) {
    static_assert(N == 4);
    u32x4_any bits;
#pragma unroll
    for (int j = 0; j < 4; ++j) bits[j] = __float_as_uint(v[j]);
    __builtin_nontemporal_store(bits, reinterpret_cast<u32x4_any *>(out));
}

// A wave's accesses of each side lie next to each other: 16 bytes a lane of the wider type, and as many elements of the
// other.  Stores pass by the caches, which keep the data that is still to be read (4 layers, 432 million BF16 gradients
// to FP32: 721 us with 8 elements a lane, whose FP32 halves are stored apart, 698 so, 669 past the caches).
template <typename T, typename O>
__device__ __forceinline__ void scale_part(const T *g, O *out, int n, float scale) {
    constexpr int N = sizeof(T) == 2 && sizeof(O) == 2 ? 8 : 4, U = 32 / N;
    const int vectors = n / N;
    const auto put = [&](int at, float (&v)[N]) {
#pragma unroll
        for (int j = 0; j < N; ++j) v[j] *= scale;
        store_some(out + at * N, v);
    };
    int at = threadIdx.x;
    for (; at + (U - 1) * kThreads < vectors; at += U * kThreads) {
        float v[U][N];
#pragma unroll
        for (int u = 0; u < U; ++u) load_some(g + (at + u * kThreads) * N, v[u]);
#pragma unroll
        for (int u = 0; u < U; ++u) put(at + u * kThreads, v[u]);
    }
    for (; at < vectors; at += kThreads) {
        float v[N];
        load_some(g + at * N, v);
        put(at, v);
    }
    const int odd = vectors * N + int(threadIdx.x);
    if (odd < n) out[odd] = from_f32<O>(to_f32(g[odd]) * scale);
}

// The chunks are taken from the last to the first: the last ones that the norm has read are still in the cache.
__global__ __launch_bounds__(kThreads) void scale_kernel(Table<true> b, uint32_t chunks, const double *parts, int count,
                                                         double max_norm, float *norm) {
    double n;
    const float c = factor_of(parts, count, max_norm, n);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = float(n);
    for (uint32_t turn = blockIdx.x; turn < chunks; turn += gridDim.x) {
        const uint32_t chunk = chunks - 1 - turn;
        const int i = tensor_of(b, chunk);
        const uint32_t size = b.size[i];
        const int64_t begin = int64_t(chunk - (i ? b.end[i - 1] : 0)) * kChunk;
        const int left = int(min(int64_t(size & kSizeMask) - begin, int64_t(kChunk)));
        const void *data = b.data[i];
        void *out = b.out[i];
        if (c == 1.f && out == data) continue;  // as they are
        const bf16_t *half = static_cast<const bf16_t *>(data) + begin;
        const float *single = static_cast<const float *>(data) + begin;
        bf16_t *half_out = static_cast<bf16_t *>(out) + begin;
        float *single_out = static_cast<float *>(out) + begin;
        if (size >> 31)
            size >> 30 & 1 ? scale_part(half, half_out, left, c) : scale_part(half, single_out, left, c);
        else
            size >> 30 & 1 ? scale_part(single, half_out, left, c) : scale_part(single, single_out, left, c);
    }
}

// ------------------------------------------------------------------ host
struct Tensors {
    const void *const *data;
    void *const *out;  // null: none
    const int64_t *size;
    const int32_t *dtype, *out_dtype;
    int32_t count;
};

int check_tensors(const char *what, const Tensors &t, bool outputs) {
    if (t.count < 0 || (t.count && (!t.data || !t.size || !t.dtype || (outputs && (!t.out || !t.out_dtype)))))
        return fail(BDM_ERR_INVALID, "%s: bad tensors", what);
    for (int i = 0; i < t.count; ++i) {
        if (t.size[i] < 0 || (t.dtype[i] != BDM_BF16 && t.dtype[i] != BDM_F32) ||
            (outputs && t.out_dtype[i] != BDM_BF16 && t.out_dtype[i] != BDM_F32))
            return fail(BDM_ERR_INVALID, "%s: tensor %d has a bad size or dtype", what, i);
        if (t.size[i] && (!t.data[i] || (outputs && !t.out[i]))) return fail(BDM_ERR_INVALID, "%s: null pointer", what);
        if (t.size[i] > (int64_t(1) << 40)) return fail(BDM_ERR_UNSUPPORTED, "%s: tensor %d is too large", what, i);
    }
    return BDM_OK;
}

// Tables of the tensors, each to launch(table, its chunks); empty tensors are left out, very large ones take several
// entries.
template <bool OUTPUTS, typename F>
int for_tables(const Tensors &t, F launch) {
    constexpr int64_t kMostEntry = int64_t(1) << 29;  // elements, a multiple of kChunk
    static_assert(kMostEntry % kChunk == 0 && kMostEntry <= kSizeMask);
    constexpr int64_t kMostChunks = int64_t(1) << 31;
    Table<OUTPUTS> b;
    b.count = 0;
    int64_t chunks = 0;
    const auto flush = [&]() -> int {
        const int rc = b.count ? launch(b, uint32_t(chunks)) : BDM_OK;
        chunks = b.count = 0;
        return rc;
    };
    for (int i = 0; i < t.count; ++i) {
        for (int64_t from = 0; from < t.size[i]; from += kMostEntry) {
            const int64_t size = std::min(t.size[i] - from, kMostEntry), more = (size + kChunk - 1) / kChunk;
            if (b.count == Table<OUTPUTS>::kTensors || chunks + more > kMostChunks)
                if (int rc = flush()) return rc;
            chunks += more;
            const bool half = t.dtype[i] == BDM_BF16;
            b.data[b.count] = static_cast<const char *>(t.data[i]) + from * (half ? 2 : 4);
            b.size[b.count] = uint32_t(size) | uint32_t(half) << 31;
            if constexpr (OUTPUTS) {
                const bool half_out = t.out_dtype[i] == BDM_BF16;
                b.out[b.count] = static_cast<char *>(t.out[i]) + from * (half_out ? 2 : 4);
                b.size[b.count] |= uint32_t(half_out) << 30;
            }
            b.end[b.count++] = uint32_t(chunks);
        }
    }
    return flush();
}

// Workgroups of a table's launch: one a chunk, up to a bound that the tables of a call share.
int64_t blocks_of(int64_t chunks, int64_t tables) {
    return std::min(chunks, std::max<int64_t>(kMostParts / tables, 64));
}

int64_t tables_of(const Tensors &t) {
    int64_t tables = 0;
    for_tables<false>(t, [&](const Table<false> &, uint32_t) { return ++tables, BDM_OK; });
    return std::max<int64_t>(tables, 1);
}

// Whether two outputs share memory, or an output shares it with another tensor's gradient or, without being the
// same in place, with its own.
bool share_memory(const Tensors &t) {
    struct Span {
        uintptr_t begin, end;
        bool output;
    };
    std::vector<Span> spans;
    spans.reserve(size_t(t.count) * 2);
    for (int i = 0; i < t.count; ++i) {
        if (!t.size[i]) continue;
        const auto span = [&](const void *p, int32_t dtype, bool output) {
            const uintptr_t begin = reinterpret_cast<uintptr_t>(p);
            spans.push_back({begin, begin + size_t(t.size[i]) * (dtype == BDM_BF16 ? 2 : 4), output});
        };
        span(t.out[i], t.out_dtype[i], true);
        if (t.data[i] != t.out[i] || t.dtype[i] != t.out_dtype[i]) span(t.data[i], t.dtype[i], false);
    }
    std::sort(spans.begin(), spans.end(), [](const Span &a, const Span &b) { return a.begin < b.begin; });
    uintptr_t outputs_end = 0, all_end = 0;
    for (const Span &s : spans) {
        if (s.begin < (s.output ? all_end : outputs_end)) return true;
        all_end = std::max(all_end, s.end);
        if (s.output) outputs_end = std::max(outputs_end, s.end);
    }
    return false;
}

// The parts of the sum of squares, `count` of them.
int launch_squares(const Tensors &t, double *parts, int64_t &count, hipStream_t s) {
    const int64_t tables = tables_of(t);
    count = 0;
    return for_tables<false>(t, [&](const Table<false> &b, uint32_t chunks) {
        const int64_t blocks = blocks_of(chunks, tables);
        squares_kernel<<<unsigned(blocks), kThreads, 0, s>>>(b, chunks, parts + count);
        count += blocks;
        return check_launch("squares_kernel");
    });
}

size_t workspace_of(const Tensors &t) {
    const int64_t tables = tables_of(t);
    int64_t parts = 0;
    for_tables<false>(t, [&](const Table<false> &, uint32_t chunks) { return parts += blocks_of(chunks, tables), BDM_OK; });
    return size_t(std::max<int64_t>(parts, 1)) * sizeof(double);
}

}  // namespace
}  // namespace bdm

using namespace bdm;

extern "C" size_t bdm_gradient_norm_workspace_size(const int64_t *sizes, int32_t count) {
    if (count <= 0 || !sizes) return sizeof(double);
    try {
        // the sizes alone count
        const std::vector<const void *> data(size_t(count), nullptr);
        const std::vector<int32_t> dtypes(size_t(count), BDM_F32);
        return workspace_of({data.data(), nullptr, sizes, dtypes.data(), nullptr, count});
    } catch (...) {
        return 0;
    }
}

extern "C" int bdm_gradient_norm(const void *const *data, const int64_t *sizes, const int32_t *dtypes, int32_t count,
                                 double max_norm, float *norm, float *scale, void *workspace, size_t workspace_bytes,
                                 void *stream) {
    const Tensors t{data, nullptr, sizes, dtypes, nullptr, count};
    if (int rc = check_tensors("gradient_norm", t, false)) return rc;
    if (!norm || !workspace) return fail(BDM_ERR_INVALID, "gradient_norm: null pointer");
    if (scale && !(max_norm >= 0)) return fail(BDM_ERR_INVALID, "gradient_norm: max_norm is negative or NaN");
    if (workspace_bytes < workspace_of(t) || !aligned(workspace, sizeof(double)))
        return fail(BDM_ERR_INVALID, "gradient_norm: workspace too small or not aligned to 8 bytes");
    double *parts = static_cast<double *>(workspace);
    int64_t used = 0;
    if (int rc = launch_squares(t, parts, used, as_stream(stream))) return rc;
    norm_kernel<<<1, kThreads, 0, as_stream(stream)>>>(parts, int(used), max_norm, norm, scale);
    return check_launch("norm_kernel");
}

extern "C" int bdm_clip_gradients(const void *const *data, void *const *out, const int64_t *sizes, const int32_t *dtypes,
                                  const int32_t *out_dtypes, int32_t count, double max_norm, float *norm, void *workspace,
                                  size_t workspace_bytes, void *stream) {
    const Tensors t{data, out, sizes, dtypes, out_dtypes, count};
    if (int rc = check_tensors("clip_gradients", t, true)) return rc;
    if (!norm || !workspace) return fail(BDM_ERR_INVALID, "clip_gradients: null pointer");
    if (!(max_norm >= 0)) return fail(BDM_ERR_INVALID, "clip_gradients: max_norm is negative or NaN");
    if (workspace_bytes < workspace_of(t) || !aligned(workspace, sizeof(double)))
        return fail(BDM_ERR_INVALID, "clip_gradients: workspace too small or not aligned to 8 bytes");
    try {
        if (share_memory(t)) return fail(BDM_ERR_INVALID, "clip_gradients: tensors share memory");
    } catch (...) {
        return fail(BDM_ERR_INVALID, "clip_gradients: out of host memory");
    }
    hipStream_t s = as_stream(stream);
    double *parts = static_cast<double *>(workspace);
    int64_t used = 0;
    if (int rc = launch_squares(t, parts, used, s)) return rc;
    bool first = true;
    if (int rc = for_tables<true>(t, [&](const Table<true> &b, uint32_t chunks) {
            scale_kernel<<<unsigned(std::min<int64_t>(chunks, kMostParts)), kThreads, 0, s>>>(
                b, chunks, parts, int(used), max_norm, first ? norm : nullptr);
            first = false;
            return check_launch("scale_kernel");
        }))
        return rc;
    if (!first) return BDM_OK;
    norm_kernel<<<1, kThreads, 0, s>>>(parts, 0, max_norm, norm, nullptr);  // no elements
    return check_launch("norm_kernel");
}
