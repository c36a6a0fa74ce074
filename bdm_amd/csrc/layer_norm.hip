// Layer normalization, forward and backward, also behind a residual add.
//
//   mu = mean x,  v = mean (x - mu)^2,  r = 1 / sqrt(v + eps),  xh = (x - mu) r,  y = xh w + b,
//   dx = r (dy w - mean(dy w) - xh mean(dy w xh)) + dsum,   dw = sum over rows dy xh,   db = sum over rows dy.
// With a residual, x is the rounded sum, written beside y.  The statistics and
// sums are FP32, the variance from the centred values.
#include "bdm_common.h"
#include "epilogue_ops.h"

namespace bdm {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr int kMaxWidth = 16384;
constexpr int kRowsPerPart = 32;

__device__ __forceinline__ float block_sum(float x, float *shared) {
    x = wave_total<kWave>(x);
    __syncthreads();
    if (threadIdx.x % kWave == 0) shared[threadIdx.x / kWave] = x;
    __syncthreads();
    x = shared[0];
    for (int i = 1; i < kWaves; ++i) x += shared[i];
    return x;
}

template <typename T>
struct Rows {
    const T *x, *residual, *grad_out, *grad_sum;
    const void *weight, *bias;
    T *sum_out, *out;
    float *partials;
    int64_t rows;
    int width, param_dtype;
    float eps;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void layer_norm_kernel(Rows<T> p) {
    __shared__ float shared[kWaves];
    const int64_t base = int64_t(blockIdx.x) * p.width;
    const auto value = [&](int c) {
        const float x = to_f32(p.x[base + c]);
        return p.residual ? round_to<T>(x + to_f32(p.residual[base + c])) : x;
    };
    float sum = 0.f, square = 0.f;
    for (int c = threadIdx.x; c < p.width; c += kThreads) sum += value(c);
    const float mean = block_sum(sum, shared) / float(p.width);
    for (int c = threadIdx.x; c < p.width; c += kThreads) {
        const float d = value(c) - mean;
        square = fmaf(d, d, square);
    }
    const float scale = rsqrtf(block_sum(square, shared) / float(p.width) + p.eps);
    for (int c = threadIdx.x; c < p.width; c += kThreads) {
        const float x = value(c);
        float y = (x - mean) * scale;
        if (p.weight) y *= param_at(p.weight, p.param_dtype, c);
        if (p.bias) y += param_at(p.bias, p.param_dtype, c);
        if (p.residual) p.sum_out[base + c] = from_f32<T>(x);
        p.out[base + c] = from_f32<T>(y);
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void layer_norm_backward_kernel(Rows<T> p) {
    __shared__ float shared[kWaves];
    float *dw = p.partials + int64_t(blockIdx.x) * 2 * p.width, *db = dw + p.width;
    for (int c = threadIdx.x; c < p.width; c += kThreads) dw[c] = db[c] = 0.f;
    const int64_t first = int64_t(blockIdx.x) * kRowsPerPart, last = min(p.rows, first + kRowsPerPart);
    for (int64_t row = first; row < last; ++row) {
        const int64_t base = row * p.width;
        float sum = 0.f, square = 0.f, dot = 0.f, plain = 0.f;
        for (int c = threadIdx.x; c < p.width; c += kThreads) sum += to_f32(p.x[base + c]);
        const float mean = block_sum(sum, shared) / float(p.width);
        for (int c = threadIdx.x; c < p.width; c += kThreads) {
            const float d = to_f32(p.x[base + c]) - mean;
            square = fmaf(d, d, square);
        }
        const float scale = rsqrtf(block_sum(square, shared) / float(p.width) + p.eps);
        for (int c = threadIdx.x; c < p.width; c += kThreads) {
            const float dy = to_f32(p.grad_out[base + c]), xh = (to_f32(p.x[base + c]) - mean) * scale;
            const float g = p.weight ? dy * param_at(p.weight, p.param_dtype, c) : dy;
            plain += g;
            dot = fmaf(g, xh, dot);
            dw[c] = fmaf(dy, xh, dw[c]);
            db[c] += dy;
        }
        plain = block_sum(plain, shared) / float(p.width);
        dot = block_sum(dot, shared) / float(p.width);
        for (int c = threadIdx.x; c < p.width; c += kThreads) {
            const float dy = to_f32(p.grad_out[base + c]), xh = (to_f32(p.x[base + c]) - mean) * scale;
            const float g = p.weight ? dy * param_at(p.weight, p.param_dtype, c) : dy;
            float dx = (g - plain - xh * dot) * scale;
            if (p.grad_sum) dx += to_f32(p.grad_sum[base + c]);
            p.out[base + c] = from_f32<T>(dx);
        }
    }
}

__global__ __launch_bounds__(kThreads) void layer_norm_param_kernel(const float *partials, int64_t parts, int width,
                                                                    void *dw, void *db, int dtype) {
    const int c = int(blockIdx.x) * kThreads + threadIdx.x;
    if (c >= 2 * width) return;
    float total = 0.f;
    for (int64_t i = 0; i < parts; ++i) total += partials[i * 2 * width + c];
    void *out = c < width ? dw : db;
    if (!out) return;
    const int at = c < width ? c : c - width;
    if (dtype == BDM_BF16)
        static_cast<bf16_t *>(out)[at] = from_f32<bf16_t>(total);
    else
        static_cast<float *>(out)[at] = total;
}

int check_rows(const char *what, int64_t rows, int32_t width, int32_t dtype, int32_t param_dtype) {
    if (rows < 0 || width <= 0) return fail(BDM_ERR_INVALID, "%s: bad geometry", what);
    if (width > kMaxWidth) return fail(BDM_ERR_UNSUPPORTED, "%s: width %d > %d", what, width, kMaxWidth);
    if ((dtype != BDM_BF16 && dtype != BDM_F32) || (param_dtype != BDM_BF16 && param_dtype != BDM_F32))
        return fail(BDM_ERR_INVALID, "%s: dtype", what);
    if (!grid_fits(rows, kThreads)) return fail(BDM_ERR_UNSUPPORTED, "%s: too many rows", what);
    return BDM_OK;
}

}  // namespace
}  // namespace bdm

using namespace bdm;

extern "C" int bdm_layer_norm(const void *x, const void *residual, const void *weight, const void *bias, void *sum_out,
                              void *out, int64_t rows, int32_t width, int32_t dtype, int32_t param_dtype, float eps,
                              void *stream) {
    if (int rc = check_rows("layer_norm", rows, width, dtype, param_dtype)) return rc;
    if (rows == 0) return BDM_OK;
    if (!x || !out || (residual && !sum_out)) return fail(BDM_ERR_INVALID, "layer_norm: null pointer");
    const auto run = [&](auto element) {
        using T = decltype(element);
        Rows<T> p{static_cast<const T *>(x), static_cast<const T *>(residual), nullptr, nullptr, weight, bias,
                  static_cast<T *>(sum_out), static_cast<T *>(out), nullptr, rows, width, param_dtype, eps};
        layer_norm_kernel<T><<<unsigned(rows), kThreads, 0, as_stream(stream)>>>(p);
    };
    if (dtype == BDM_BF16)
        run(bf16_t{});
    else
        run(float{});
    return check_launch("layer_norm_kernel");
}

extern "C" size_t bdm_layer_norm_backward_workspace_size(int64_t rows, int32_t width) {
    if (rows <= 0 || width <= 0) return 0;
    return size_t((rows + kRowsPerPart - 1) / kRowsPerPart) * 2 * size_t(width) * sizeof(float);
}

extern "C" int bdm_layer_norm_backward(const void *x, const void *grad_out, const void *grad_sum, const void *weight,
                                       void *grad_x, void *grad_weight, void *grad_bias, int64_t rows, int32_t width,
                                       int32_t dtype, int32_t param_dtype, float eps, void *workspace,
                                       size_t workspace_bytes, void *stream) {
    if (int rc = check_rows("layer_norm_backward", rows, width, dtype, param_dtype)) return rc;
    if (rows && (!x || !grad_out || !grad_x || !workspace))
        return fail(BDM_ERR_INVALID, "layer_norm_backward: null pointer");
    if (workspace_bytes < bdm_layer_norm_backward_workspace_size(rows, width) || !aligned(workspace, 16))
        return fail(BDM_ERR_INVALID, "layer_norm_backward: workspace too small or not aligned to 16 bytes");
    hipStream_t s = as_stream(stream);
    const int64_t parts = (rows + kRowsPerPart - 1) / kRowsPerPart;
    const auto run = [&](auto element) {
        using T = decltype(element);
        Rows<T> p{static_cast<const T *>(x), nullptr, static_cast<const T *>(grad_out), static_cast<const T *>(grad_sum),
                  weight, nullptr, nullptr, static_cast<T *>(grad_x), static_cast<float *>(workspace), rows, width,
                  param_dtype, eps};
        if (parts) layer_norm_backward_kernel<T><<<unsigned(parts), kThreads, 0, s>>>(p);
    };
    if (dtype == BDM_BF16)
        run(bf16_t{});
    else
        run(float{});
    if (int rc = check_launch("layer_norm_backward_kernel")) return rc;
    if (!grad_weight && !grad_bias) return BDM_OK;
    layer_norm_param_kernel<<<unsigned((2 * width + kThreads - 1) / kThreads), kThreads, 0, s>>>(
        static_cast<const float *>(workspace), parts, width, grad_weight, grad_bias, param_dtype);
    return check_launch("layer_norm_param_kernel");
}
