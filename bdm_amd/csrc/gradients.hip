// The global norm of a model's gradients, and their clipping.
//
//   n = sqrt(sum over all tensors of g^2),   c = min(1, max_norm / (n + 1e-6)),   g' = c g.
//
// Squares and their sums are FP64: those of FP32 overflow from 2e19 on and
// vanish below 1e-23, and a sum of a billion of them is exact to the last bits
// of the norm.  Every sum is made in a fixed order.
#include <algorithm>
#include <vector>

#include "bdm_common.h"

namespace bdm {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kChunk = 16384;  // elements of one tensor that a workgroup takes
constexpr int kBatch = 100;    // tensors of one launch, in its arguments

struct Batch {
    bdm_gradient tensors[kBatch];
    uint32_t end[kBatch];  // chunks of the batch up to and with this tensor's
    int32_t count;
};
static_assert(sizeof(Batch) <= 4000, "the arguments of a launch are at most 4 KiB");

__device__ __forceinline__ int tensor_of(const Batch &b, uint32_t chunk) {
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

template <typename T>
__device__ __forceinline__ double squares(const T *g, int64_t begin, int64_t end) {
    double sum = 0;
    for (int64_t i = begin + threadIdx.x; i < end; i += kThreads) {
        const double x = double(to_f32(g[i]));
        sum = fma(x, x, sum);
    }
    return sum;
}

__global__ __launch_bounds__(kThreads) void squares_kernel(Batch b, double *parts) {
    __shared__ double shared[kWaves];
    const int i = tensor_of(b, blockIdx.x);
    const bdm_gradient &t = b.tensors[i];
    const int64_t begin = int64_t(blockIdx.x - (i ? b.end[i - 1] : 0)) * kChunk, end = min(t.numel, begin + kChunk);
    const double sum = block_sum(t.dtype == BDM_BF16 ? squares(static_cast<const bf16_t *>(t.data), begin, end)
                                                     : squares(static_cast<const float *>(t.data), begin, end), shared);
    if (threadIdx.x == 0) parts[blockIdx.x] = sum;
}

__global__ __launch_bounds__(kThreads) void norm_kernel(const double *parts, int64_t count, double max_norm, float *norm,
                                                        float *scale) {
    __shared__ double shared[kWaves];
    double sum = 0;
    for (int64_t i = threadIdx.x; i < count; i += kThreads) sum += parts[i];
    sum = block_sum(sum, shared);
    if (threadIdx.x == 0) {
        const double n = sqrt(sum), c = max_norm / (n + 1e-6);
        *norm = float(n);
        if (scale) *scale = c > 1 ? 1.f : float(c);
    }
}

template <typename T, typename O>
__device__ __forceinline__ void scale_part(const bdm_gradient &t, int64_t begin, int64_t end, float scale) {
    const T *g = static_cast<const T *>(t.data);
    O *out = static_cast<O *>(t.out);
    for (int64_t i = begin + threadIdx.x; i < end; i += kThreads) out[i] = from_f32<O>(to_f32(g[i]) * scale);
}

__global__ __launch_bounds__(kThreads) void scale_kernel(Batch b, const float *scale) {
    const int i = tensor_of(b, blockIdx.x);
    const bdm_gradient &t = b.tensors[i];
    const int64_t begin = int64_t(blockIdx.x - (i ? b.end[i - 1] : 0)) * kChunk, end = min(t.numel, begin + kChunk);
    const float c = *scale;
    if (c == 1.f && t.out == t.data) return;  // as they are
    if (t.dtype == BDM_BF16) {
        if (t.out_dtype == BDM_BF16)
            scale_part<bf16_t, bf16_t>(t, begin, end, c);
        else
            scale_part<bf16_t, float>(t, begin, end, c);
    } else {
        if (t.out_dtype == BDM_BF16)
            scale_part<float, bf16_t>(t, begin, end, c);
        else
            scale_part<float, float>(t, begin, end, c);
    }
}

int64_t chunks_of(int64_t numel) { return (numel + kChunk - 1) / kChunk; }

int check_tensors(const char *what, const bdm_gradient *tensors, int32_t count, bool outputs) {
    if (count < 0 || (count && !tensors)) return fail(BDM_ERR_INVALID, "%s: bad tensors", what);
    for (int i = 0; i < count; ++i) {
        const bdm_gradient &t = tensors[i];
        if (t.numel < 0 || (t.dtype != BDM_BF16 && t.dtype != BDM_F32) ||
            (outputs && t.out_dtype != BDM_BF16 && t.out_dtype != BDM_F32))
            return fail(BDM_ERR_INVALID, "%s: tensor %d has a bad size or dtype", what, i);
        if (t.numel && (!t.data || (outputs && !t.out))) return fail(BDM_ERR_INVALID, "%s: null pointer", what);
        if (t.numel > (int64_t(1) << 40)) return fail(BDM_ERR_UNSUPPORTED, "%s: tensor %d is too large", what, i);
    }
    return BDM_OK;
}

// Batches of tensors, each to launch(batch, its chunks, chunks before it); empty tensors are left out.
template <typename F>
int for_batches(const bdm_gradient *tensors, int32_t count, F launch) {
    Batch b{};
    int64_t chunks = 0, before = 0;
    const auto flush = [&]() -> int {
        if (!b.count) return BDM_OK;
        const int rc = launch(b, chunks, before);
        before += chunks;
        chunks = b.count = 0;
        return rc;
    };
    for (int i = 0; i < count; ++i) {
        if (!tensors[i].numel) continue;
        const int64_t more = chunks_of(tensors[i].numel);
        if (b.count == kBatch || !grid_fits(chunks + more, kThreads))
            if (int rc = flush()) return rc;
        if (!grid_fits(more, kThreads)) return fail(BDM_ERR_UNSUPPORTED, "gradients: tensor %d is too large", i);
        chunks += more;
        b.tensors[b.count] = tensors[i];
        b.end[b.count++] = uint32_t(chunks);
    }
    return flush();
}

int64_t total_chunks(const bdm_gradient *tensors, int32_t count) {
    int64_t total = 0;
    for (int i = 0; i < count; ++i) total += tensors[i].numel > 0 ? chunks_of(tensors[i].numel) : 0;
    return total;
}

size_t dtype_bytes(int32_t dtype) { return dtype == BDM_BF16 ? 2 : 4; }

// Whether two outputs share memory, or an output shares it with another tensor's gradient or, without being the
// same in place, with its own.
bool share_memory(const bdm_gradient *tensors, int32_t count) {
    struct Span {
        uintptr_t begin, end;
        int32_t tensor;
        bool output;
    };
    std::vector<Span> spans;
    spans.reserve(size_t(count) * 2);
    for (int i = 0; i < count; ++i) {
        const bdm_gradient &t = tensors[i];
        if (!t.numel) continue;
        const uintptr_t data = reinterpret_cast<uintptr_t>(t.data), out = reinterpret_cast<uintptr_t>(t.out);
        spans.push_back({out, out + size_t(t.numel) * dtype_bytes(t.out_dtype), i, true});
        if (data != out || t.dtype != t.out_dtype) spans.push_back({data, data + size_t(t.numel) * dtype_bytes(t.dtype), i, false});
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

int norm_of(const bdm_gradient *tensors, int32_t count, double max_norm, float *norm, float *scale, double *parts,
            hipStream_t s) {
    if (int rc = for_batches(tensors, count, [&](const Batch &b, int64_t chunks, int64_t before) {
            squares_kernel<<<unsigned(chunks), kThreads, 0, s>>>(b, parts + before);
            return check_launch("squares_kernel");
        }))
        return rc;
    norm_kernel<<<1, kThreads, 0, s>>>(parts, total_chunks(tensors, count), max_norm, norm, scale);
    return check_launch("norm_kernel");
}

}  // namespace
}  // namespace bdm

using namespace bdm;

extern "C" size_t bdm_gradient_norm_workspace_size(const bdm_gradient *tensors, int32_t count) {
    if (count <= 0 || !tensors) return 16;
    return 16 + size_t(total_chunks(tensors, count)) * sizeof(double);
}

extern "C" int bdm_gradient_norm(const bdm_gradient *tensors, int32_t count, double max_norm, float *norm, float *scale,
                                 void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_tensors("gradient_norm", tensors, count, false)) return rc;
    if (!norm || !workspace) return fail(BDM_ERR_INVALID, "gradient_norm: null pointer");
    if (scale && !(max_norm >= 0)) return fail(BDM_ERR_INVALID, "gradient_norm: max_norm is negative or NaN");
    if (workspace_bytes < bdm_gradient_norm_workspace_size(tensors, count) || !aligned(workspace, 16))
        return fail(BDM_ERR_INVALID, "gradient_norm: workspace too small or not aligned to 16 bytes");
    return norm_of(tensors, count, max_norm, norm, scale, static_cast<double *>(workspace) + 2, as_stream(stream));
}

extern "C" int bdm_clip_gradients(const bdm_gradient *tensors, int32_t count, double max_norm, float *norm,
                                  void *workspace, size_t workspace_bytes, void *stream) {
    if (int rc = check_tensors("clip_gradients", tensors, count, true)) return rc;
    if (!norm || !workspace) return fail(BDM_ERR_INVALID, "clip_gradients: null pointer");
    if (!(max_norm >= 0)) return fail(BDM_ERR_INVALID, "clip_gradients: max_norm is negative or NaN");
    if (workspace_bytes < bdm_gradient_norm_workspace_size(tensors, count) || !aligned(workspace, 16))
        return fail(BDM_ERR_INVALID, "clip_gradients: workspace too small or not aligned to 16 bytes");
    try {
        if (share_memory(tensors, count)) return fail(BDM_ERR_INVALID, "clip_gradients: tensors share memory");
    } catch (...) {
        return fail(BDM_ERR_INVALID, "clip_gradients: out of host memory");
    }
    hipStream_t s = as_stream(stream);
    float *scale = static_cast<float *>(workspace);
    if (int rc = norm_of(tensors, count, max_norm, norm, scale, static_cast<double *>(workspace) + 2, s)) return rc;
    return for_batches(tensors, count, [&](const Batch &b, int64_t chunks, int64_t) {
        scale_kernel<<<unsigned(chunks), kThreads, 0, s>>>(b, scale);
        return check_launch("scale_kernel");
    });
}
