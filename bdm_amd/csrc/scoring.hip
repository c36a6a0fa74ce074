// Log-probabilities of given tokens, the entropy of their distributions and
// the best alternatives, and the gradient of the logits; the mean loss.
//
// For a row x of logits with m = max x, s = sum exp(x - m):
//   log p_i = (x_i - m) - log s,   H = log s - sum exp(x - m) (x - m) / s,
// and with gradients a of log p_t, h of H and b_k of log p at the alternatives
//   dx_i = a [i = t] + sum_k b_k [i = top_k] - p_i (a + sum_k b_k + h (log p_i + H)).
// Everything is FP32.
#include <cfloat>

#include "bdm_common.h"

namespace bdm {
namespace {

constexpr int kAlternativesMax = 32;
constexpr int kThreads = 256, kWaves = kThreads / kWave;

// Unsigned integers in the order of the floating values; -0 counts as +0, a NaN is above all.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t u = __float_as_uint(x + 0.f);
    return x != x ? UINT32_MAX - 1 : u ^ (uint32_t(int32_t(u) >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t u) {
    return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u);
}

template <typename V, typename F>
__device__ __forceinline__ V block_join(V x, F op, V *shared) {
#pragma unroll
    for (int step = kWave / 2; step; step >>= 1) x = op(x, __shfl_xor(x, step, kWave));
    __syncthreads();
    if (threadIdx.x % kWave == 0) shared[threadIdx.x / kWave] = x;
    __syncthreads();
    x = shared[0];
    for (int i = 1; i < kWaves; ++i) x = op(x, shared[i]);
    return x;
}

__device__ __forceinline__ float log_probability(float x, float high, float log_sum) {
    return log_sum == -INFINITY ? -INFINITY : (x - high) - log_sum;
}

// One row per workgroup.
template <typename T>
__global__ __launch_bounds__(kThreads) void token_log_probs_kernel(bdm_token_args a) {
    __shared__ float floats[kWaves];
    __shared__ unsigned long long keys[kWaves];
    const int64_t row = blockIdx.x;
    const T *x = static_cast<const T *>(a.logits) + row * a.row_stride;
    float high = -INFINITY;
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) high = fmaxf(high, to_f32(x[i]));
    high = block_join(high, [](float p, float q) { return fmaxf(p, q); }, floats);
    const float from = high == -INFINITY ? 0.f : high;  // an empty row
    float sum = 0.f, moment = 0.f;
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
        const float d = to_f32(x[i]) - from, e = expf(d);
        sum += e;
        moment += e == 0.f ? 0.f : e * d;
    }
    const auto add = [](float p, float q) { return p + q; };
    sum = block_join(sum, add, floats);
    moment = block_join(moment, add, floats);
    const float log_sum = logf(sum);
    if (threadIdx.x == 0) {
        const int64_t token = a.tokens[row];
        float lp = 0.f;
        if (token != a.ignore_index)
            lp = token >= 0 && token < a.vocab ? log_probability(to_f32(x[token]), from, log_sum) : NAN;
        a.log_probs[row] = lp;
        if (a.entropy) a.entropy[row] = sum == 0.f ? 0.f : log_sum - moment / sum;
        if (a.stats) {
            a.stats[2 * row] = from;
            a.stats[2 * row + 1] = log_sum;
        }
    }
    unsigned long long last = UINT64_MAX;
    for (int k = 0; k < a.alternatives; ++k) {
        unsigned long long best = 0;
        for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
            const unsigned long long key = (unsigned long long)(ordered(to_f32(x[i]))) << 32 | uint32_t(~i);
            if (key < last && key > best) best = key;
        }
        best = block_join(best, [](unsigned long long p, unsigned long long q) { return p > q ? p : q; }, keys);
        if (threadIdx.x == 0) {
            const int token = int(~uint32_t(best));
            a.top_tokens[row * a.alternatives + k] = token;
            a.top_log_probs[row * a.alternatives + k] = log_probability(to_f32(x[token]), from, log_sum);
        }
        last = best;
    }
}

// The gradients that reach a row: of its token's log-probability, its entropy and its alternatives.
struct RowGradient {
    float given, total, entropy;
};

template <typename T>
__global__ __launch_bounds__(kThreads) void token_gradient_kernel(bdm_token_grad_args a) {
    const int64_t row = blockIdx.x;
    const T *x = static_cast<const T *>(a.logits) + row * a.row_stride;
    T *out = static_cast<T *>(a.grad_logits) + row * a.vocab;
    const int64_t token = a.tokens[row];
    const float high = a.stats[2 * row], log_sum = a.stats[2 * row + 1];
    const float h = a.grad_entropy ? a.grad_entropy[row] : 0.f, entropy = a.entropy ? a.entropy[row] : 0.f;
    float given = 0.f;
    if (token != a.ignore_index && (a.grad_loss || a.grad_log_probs)) {
        given = a.grad_loss ? -(a.grad_loss[0] * a.inverse_count[0]) : a.grad_log_probs[row];
        if (token < 0 || token >= a.vocab) given = NAN;
    }
    float total = given;
    const int tops = a.grad_top_log_probs ? a.alternatives : 0;
    for (int k = 0; k < tops; ++k) total += a.grad_top_log_probs[row * tops + k];
    for (int i = threadIdx.x; i < a.vocab; i += kThreads) {
        const float lp = (to_f32(x[i]) - high) - log_sum, p = expf(lp);
        float d = p == 0.f ? 0.f : -p * (total + h * (lp + entropy));
        if (i == token) d += given;
        for (int k = 0; k < tops; ++k)
            if (a.top_tokens[row * tops + k] == i) d += a.grad_top_log_probs[row * tops + k];
        out[i] = from_f32<T>(log_sum == -INFINITY ? 0.f : d);
    }
}

// loss = -sum of the log-probabilities / their number, in FP64 and always in the same order.
__global__ __launch_bounds__(kThreads) void token_loss_kernel(const float *log_probs, const int64_t *tokens, int64_t rows,
                                                              int64_t ignore_index, float *loss, float *inverse_count) {
    __shared__ double values[kWaves];
    double sum = 0, count = 0;
    for (int64_t i = threadIdx.x; i < rows; i += kThreads) {
        if (tokens[i] == ignore_index) continue;
        sum += double(log_probs[i]);
        count += 1;
    }
    const auto add = [](double p, double q) { return p + q; };
    sum = block_join(sum, add, values);
    count = block_join(count, add, values);
    if (threadIdx.x == 0) {
        *loss = float(-sum / count);
        *inverse_count = float(1 / count);
    }
}

int check_rows(const char *what, int64_t rows, int64_t row_stride, int32_t vocab, int32_t dtype, int32_t alternatives) {
    if (rows < 0 || vocab <= 0 || row_stride < 0 || alternatives < 0 || alternatives > vocab)
        return fail(BDM_ERR_INVALID, "%s: bad geometry", what);
    if (dtype != BDM_BF16 && dtype != BDM_F32) return fail(BDM_ERR_INVALID, "%s: dtype", what);
    if (alternatives > kAlternativesMax)
        return fail(BDM_ERR_UNSUPPORTED, "%s: more than %d alternatives", what, kAlternativesMax);
    if (vocab > (1 << 30)) return fail(BDM_ERR_UNSUPPORTED, "%s: vocabulary beyond 2^30", what);
    if (!grid_fits(rows, kThreads)) return fail(BDM_ERR_UNSUPPORTED, "%s: too many rows", what);
    return BDM_OK;
}

}  // namespace
}  // namespace bdm

using namespace bdm;

extern "C" size_t bdm_token_log_probs_workspace_size(const bdm_token_args *) { return 0; }

extern "C" int bdm_token_log_probs(const bdm_token_args *a, void *, size_t, void *stream) {
    if (!a) return fail(BDM_ERR_INVALID, "token_log_probs: null args");
    if (int rc = check_rows("token_log_probs", a->rows, a->row_stride, a->vocab, a->dtype, a->alternatives)) return rc;
    if (a->rows == 0) return BDM_OK;
    if (!a->logits || !a->tokens || !a->log_probs ||
        (a->alternatives && (!a->top_log_probs || !a->top_tokens)))
        return fail(BDM_ERR_INVALID, "token_log_probs: null pointer");
    hipStream_t s = as_stream(stream);
    if (a->dtype == BDM_BF16)
        token_log_probs_kernel<bf16_t><<<unsigned(a->rows), kThreads, 0, s>>>(*a);
    else
        token_log_probs_kernel<float><<<unsigned(a->rows), kThreads, 0, s>>>(*a);
    return check_launch("token_log_probs_kernel");
}

extern "C" int bdm_token_log_probs_backward(const bdm_token_grad_args *a, void *stream) {
    if (!a) return fail(BDM_ERR_INVALID, "token_log_probs_backward: null args");
    if (int rc = check_rows("token_log_probs_backward", a->rows, a->row_stride, a->vocab, a->dtype, a->alternatives))
        return rc;
    if (a->rows == 0) return BDM_OK;
    if (!a->logits || !a->tokens || !a->stats || !a->grad_logits || (a->grad_entropy && !a->entropy) ||
        (a->grad_top_log_probs && !a->top_tokens) || (a->grad_loss && !a->inverse_count))
        return fail(BDM_ERR_INVALID, "token_log_probs_backward: null pointer");
    hipStream_t s = as_stream(stream);
    if (a->dtype == BDM_BF16)
        token_gradient_kernel<bf16_t><<<unsigned(a->rows), kThreads, 0, s>>>(*a);
    else
        token_gradient_kernel<float><<<unsigned(a->rows), kThreads, 0, s>>>(*a);
    return check_launch("token_gradient_kernel");
}

extern "C" int bdm_token_loss(const float *log_probs, const int64_t *tokens, int64_t rows, int64_t ignore_index,
                              float *loss, float *inverse_count, void *stream) {
    if (rows < 0) return fail(BDM_ERR_INVALID, "token_loss: bad geometry");
    if ((rows && (!log_probs || !tokens)) || !loss || !inverse_count)
        return fail(BDM_ERR_INVALID, "token_loss: null pointer");
    token_loss_kernel<<<1, kThreads, 0, as_stream(stream)>>>(log_probs, tokens, rows, ignore_index, loss, inverse_count);
    return check_launch("token_loss_kernel");
}
