// Log-probabilities of given tokens, the entropy of their distributions and
// the best alternatives, and the gradient of the logits; the mean loss.
//
// For a row x of logits with m = max x, s = sum exp(x - m):
//   log p_i = (x_i - m) - log s,   H = log s - sum exp(x - m) (x - m) / s,
// and with gradients a of log p_t, h of H and b_k of log p at the alternatives
//   dx_i = a [i = t] + sum_k b_k [i = top_k] - p_i (a + sum_k b_k + h (log p_i + H)).
// Arithmetic and sums are FP32, those of the loss' mean FP64 and of long rows' parts too; a BF16 gradient is rounded once.
// Times, here and below: of a call in a graph over two to eight tensors of logits in turn; "alone" those of a kernel under
// the profiler.
//
// Forward.  A call without alternatives over many or long rows streams them (stream_kernel): bound by the read of the
// logits (8,192 rows of 50,257 BF16, 823 MB: 149 us, 5.5 TB/s; alone 144).  Others hold a row, or a part of a long one, in
// registers (score_kernel): every value is read once, and the alternatives are found without a second read, by a bound
// that as many lanes' own maxima reach and a ranking of the few values above it.  The parts of a row are joined by a
// second launch (join_kernel).  Bound by latency for few rows (64 of 50,257 with 8 alternatives: 12.1 us; alone 8.7 and
// 4.0), by the instructions of the selection for many (4,096: 113 us, 3.6 TB/s).
// Backward (token_gradient_kernel).  The logits are read again and the gradient is written: HBM (8,192 rows of 50,257
// BF16: 290 us, 5.7 TB/s; alone, behind the forward of the same logits, 267).
#include <algorithm>
#include <cfloat>

#include "bdm_common.h"
#include "selection_ops.h"

namespace bdm {
namespace {

constexpr int kAlternativesMax = 32;
constexpr int kVocabMax = 1 << 24;
constexpr int kThreads = 256, kWaves = kThreads / kWave;
constexpr float kLog2E = 1.4426950408889634f;
constexpr uint32_t kNanKey = UINT32_MAX - 1, kEmptyKey = 0x007fffffu;  // a NaN's, and that of -inf

// ordered() with a NaN above all others.
__device__ __forceinline__ uint32_t ordered_all(float x) { return x != x ? kNanKey : ordered(x); }

__device__ __forceinline__ float log_probability(float x, float high, float log_sum) {
    return log_sum == -INFINITY ? -INFINITY : (x - high) - log_sum;
}

// The results of one row from its statistics: by one thread.
__device__ __forceinline__ void put_row(const bdm_token_args &a, int64_t row, int64_t token, float given, float from,
                                        float log_sum, float entropy) {
    const bool inside = token >= 0 && token < a.vocab;
    a.log_probs[row] = token == a.ignore_index ? 0.f : inside ? log_probability(given, from, log_sum) : NAN;
    if (a.entropy) a.entropy[row] = log_sum == -INFINITY ? 0.f : entropy;
    if (a.stats) {
        a.stats[2 * row] = from;
        a.stats[2 * row + 1] = log_sum;
    }
}

// ------------------------------------------------------------------ a team's part of a row
template <int WAVES, int NV>
struct Team {
    static constexpr int kRoom = WAVES == 1 ? 128 : 256;
    uint64_t list[kRoom];  // ordered value, then ~index: descending order is value, then lowest index
    float high[WAVES], sum[WAVES], moment[WAVES];
    uint32_t bound[WAVES], share[WAVES];
    int found[WAVES];
    int ties[WAVES][NV];
    int count;
};

struct Rows {
    bdm_token_args a;
    float4 *parts;    // [rows, splits] maximum, sum of exponentials, their first moment
    uint64_t *lists;  // [rows, splits, alternatives], 0 behind the last
    int splits;
};

// A lane's vectors of a part.  Vector i has the row's values from `start(i)` on.  The last vector of a row starts early
// enough to end with it; what the one before holds already, and what lies behind the row, is -inf in it.
template <typename T, int WAVES>
struct Place {
    static constexpr int VE = Vec<T>::kSize, kSpan = WAVES * kWave * VE;
    const T *x;                // the part's first value
    int first, length, vocab;  // of the lane's first vector in the part; the part's values; the row's

    __device__ __forceinline__ int begin(int i) const { return first + i * kSpan; }
    __device__ __forceinline__ int start(int i) const { return vocab < VE ? begin(i) : min(begin(i), length - VE); }
    __device__ __forceinline__ bool valid(int i, int j) const {
        const int at = start(i) + j;
        return at >= begin(i) && at < length;
    }
    __device__ __forceinline__ u32x4 load(int i) const { return reinterpret_cast<const AnyVector<T> *>(x + start(i))->bits; }
    // of a row shorter than a vector
    __device__ __forceinline__ u32x4 gather() const {
        u32x4 raw{};
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            const uint32_t bits = __float_as_uint(to_f32(x[min(j, vocab - 1)]));
            if constexpr (VE == 8)
                raw[j / 2] |= j % 2 ? bits : bits >> 16;
            else
                raw[j] = bits;
        }
        return raw;
    }
    __device__ __forceinline__ void mask(int i, u32x4 &raw) const {
        if (begin(i) + VE <= length) return;
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            if (valid(i, j)) continue;
            if constexpr (VE == 8)
                raw[j / 2] = j % 2 ? (raw[j / 2] & 0xffffu) | 0xff800000u : (raw[j / 2] & 0xffff0000u) | 0xff80u;
            else
                raw[j] = 0xff800000u;
        }
    }
};

// The exact `width` best of the team's values to sh.list where the bound does not serve: those above the width-th, then
// of those equal to it the ones of lowest index, which lie in the order of vectors, lanes, places in the vector.  `guess`
// is the width-th's key if no `width` values are above it (equal logits, or a mask over most of the row): three passes
// over the part (4,096 level rows of 50,257 BF16 with 8: 409 us, 113 of others); else that is bisected, a pass a bit.  So
// it is where fewer lanes than `width` hold a value, which gives no bound: vocabularies, or a row's last part, of fewer
// than `width` vectors (8,192 rows of 192 BF16, 24 vectors: 30 us with 24 alternatives, 55 with 25 to 32; of 64 with 16
// 54, 8.4 with 8).  Vector by vector from memory: it takes no registers from the ordinary case.
template <typename T, int WAVES, int NV>
__device__ __forceinline__ int team_exact(Team<WAVES, NV> &sh, const T *x, int length, int vocab, uint32_t guess, int width,
                                       uint32_t offset, int wave, int lane) {
    constexpr int VE = Vec<T>::kSize;
    const Place<T, WAVES> place{x, (wave * kWave + lane) * VE, length, vocab};
    width = min(width, length);
    // f(i, keys of vector i, 0 where it has none)
    const auto each = [&](auto f) {
#pragma unroll 1
        for (int i = 0; i < NV; ++i) {
            const u32x4 raw = vocab < VE ? place.gather() : place.load(i);
            float v[VE];
            uint32_t keys[VE];
            Vec<T>::widen(raw, v);
#pragma unroll
            for (int j = 0; j < VE; ++j) keys[j] = place.valid(i, j) ? ordered_all(v[j]) : 0;
            f(i, keys);
        }
    };
    const auto reach = [&](uint32_t least) {
        int mine = 0;
        each([&](int, const uint32_t *keys) {
#pragma unroll
            for (int j = 0; j < VE; ++j) mine += popcount(__ballot(keys[j] >= least));
        });
        if constexpr (WAVES > 1) {
            if (lane == 0) sh.found[wave] = mine;
            __syncthreads();
            mine = 0;
#pragma unroll
            for (int i = 0; i < WAVES; ++i) mine += sh.found[i];
            __syncthreads();
        }
        return mine;
    };
    team_sync<WAVES>();
    uint32_t value = guess;
    int above = reach(value + 1);
    if (above >= width) {
        value = 0;
#pragma unroll 1
        for (int bit = 31; bit >= 0; --bit) {
            const uint32_t next = value | (1u << bit);
            if (reach(next) >= width) value = next;
        }
        above = reach(value + 1);
    }
    each([&](int i, const uint32_t *keys) {
        int ties = 0;
#pragma unroll
        for (int j = 0; j < VE; ++j) ties += popcount(__ballot(keys[j] == value));
        if (lane == 0) sh.ties[wave][i] = ties;
    });
    if (wave == 0 && lane == 0) sh.count = 0;
    team_sync<WAVES>();
    int before = above;  // candidates ahead of the vector's, in this wave's order
    each([&](int i, const uint32_t *keys) {
        const auto take = [&](int j) {
            // `width` of them, unless another stream changes the logits between two passes
            const int to = atomicAdd(&sh.count, 1);
            if (to < Team<WAVES, NV>::kRoom)
                sh.list[to] = uint64_t(keys[j]) << 32 | uint32_t(~(offset + uint32_t(place.start(i) + j)));
        };
        int at = before;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            at += w < wave ? sh.ties[w][i] : 0;
            before += sh.ties[w][i];
        }
#pragma unroll
        for (int j = 0; j < VE; ++j) at += popcount(__ballot(keys[j] == value) & ((1ull << lane) - 1));
#pragma unroll
        for (int j = 0; j < VE; ++j)
            if (keys[j] > value || (keys[j] == value && at++ < width)) take(j);
    });
    team_sync<WAVES>();
    return min(sh.count, Team<WAVES, NV>::kRoom);
}

// One part of one row, held in registers by a team of WAVES waves.
template <typename T, int WAVES, int NV, bool TOP>
__device__ __forceinline__ void score_part(const Rows &p, Team<WAVES, NV> &sh, int64_t row, int split, int wave, int lane) {
    constexpr int VE = Vec<T>::kSize;
    const bdm_token_args &a = p.a;
    constexpr int kPart = NV * Place<T, WAVES>::kSpan;
    const int offset = split * kPart, thread = wave * kWave + lane;
    const T *x = static_cast<const T *>(a.logits) + row * a.row_stride;
    const Place<T, WAVES> place{x + offset, thread * VE, min(a.vocab - offset, kPart), a.vocab};
    const int64_t token = a.tokens[row];
    const float given = to_f32(x[token >= 0 && token < a.vocab ? token : 0]);
    u32x4 raw[NV];
    if (a.vocab >= VE) {
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = place.load(i);
    } else {
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = place.gather();
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) place.mask(i, raw[i]);
    // f(i, values of vector i)
    const auto each = [&](auto f) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float v[VE];
            Vec<T>::widen(raw[i], v);
            f(i, v);
        }
    };
    float top = -INFINITY;
    each([&](int, const float *v) {
#pragma unroll
        for (int j = 0; j < VE; ++j) top = fmaxf(top, v[j]);
    });
    float high = wave_max(top);
    uint32_t bound = 0;
    if constexpr (WAVES > 1) {
        if constexpr (TOP) {
            // `alternatives` lanes of one wave, or as many of all of them together, reach the bound
            const uint32_t width = uint32_t(a.alternatives);
            const Bounds<2> bounds = nth_of_lanes<2>(top > -INFINITY ? ordered(top) : 0u, {{width, (width + WAVES - 1) / WAVES}});
            if (lane == 0) {
                sh.bound[wave] = bounds.at[0];
                sh.share[wave] = bounds.at[1];
            }
            if (thread == 0) sh.count = 0;
        }
        if (lane == 0) sh.high[wave] = high;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WAVES; ++i) high = fmaxf(high, sh.high[i]);
        if constexpr (TOP) {
            bound = sh.share[0];
#pragma unroll
            for (int i = 1; i < WAVES; ++i) bound = min(bound, sh.share[i]);
#pragma unroll
            for (int i = 0; i < WAVES; ++i) bound = max(bound, sh.bound[i]);
        }
    } else if constexpr (TOP) {
        bound = nth_of_lanes<1>(top > -INFINITY ? ordered(top) : 0u, {{uint32_t(a.alternatives)}}).at[0];
        if (lane == 0) sh.count = 0;
        team_sync<WAVES>();
    }
    const float from = high > -INFINITY ? high : 0.f;  // a part without a finite value has the sum 0
    float sum = 0.f, moment = 0.f;
    each([&](int, const float *v) {
#pragma unroll
        for (int j = 0; j < VE; ++j) {
            const float d = v[j] - from, e = __builtin_amdgcn_exp2f(d * kLog2E);
            sum += e;
            moment = fmaf(e, fmaxf(d, -1e30f), moment);  // e = 0 there: no 0 * inf
        }
    });
    sum = wave_sum(sum);
    moment = wave_sum(moment);
    if constexpr (TOP) {
        const float least = unordered(bound);
        if (bound && top >= least) {
            each([&](int i, const float *v) {
#pragma unroll
                for (int j = 0; j < VE; ++j) {
                    if (v[j] >= least) {
                        const int at = atomicAdd(&sh.count, 1);
                        if (at < Team<WAVES, NV>::kRoom)
                            sh.list[at] = uint64_t(ordered(v[j])) << 32 | uint32_t(~uint32_t(offset + place.start(i) + j));
                    }
                }
            });
        }
    }
    if constexpr (WAVES > 1) {
        if (lane == 0) {
            sh.sum[wave] = sum;
            sh.moment[wave] = moment;
        }
        __syncthreads();
        sum = moment = 0.f;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            sum += sh.sum[i];
            moment += sh.moment[i];
        }
    } else {
        team_sync<WAVES>();
    }
    int count = 0;
    if constexpr (TOP) {
        count = sh.count;
        if (!bound || count > Team<WAVES, NV>::kRoom || sum != sum)
            count = team_exact<T, WAVES, NV>(sh, place.x, place.length, a.vocab, bound ? bound : kEmptyKey, a.alternatives,
                                                  uint32_t(offset), wave, lane);
    }
    const float log_sum = logf(sum);
    if (thread == 0) {
        if (p.splits > 1) {
            p.parts[row * p.splits + split] = make_float4(high, sum, moment, 0.f);
        } else {
            put_row(a, row, token, given, from, log_sum, log_sum - moment / sum);
        }
    }
    if constexpr (TOP) {
        const int64_t out = (row * p.splits + split) * a.alternatives;
        for (int i = thread; i < count; i += WAVES * kWave) {
            const uint64_t mine = sh.list[i];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < count; ++j) rank += sh.list[j] > mine;
            if (rank >= a.alternatives) continue;
            if (p.splits > 1) {
                p.lists[out + rank] = mine;
            } else {
                a.top_tokens[out + rank] = int64_t(~uint32_t(mine));
                a.top_log_probs[out + rank] = log_probability(unordered(uint32_t(mine >> 32)), from, log_sum);
            }
        }
        if (p.splits > 1)
            for (int i = count + thread; i < a.alternatives; i += WAVES * kWave) p.lists[out + i] = 0;
    }
}

template <typename T, int WAVES, int NV, bool TOP>
__global__ __launch_bounds__(kThreads) void score_kernel(Rows p) {
    const int wave = int(threadIdx.x) / kWave, lane = int(threadIdx.x) % kWave;
    if constexpr (WAVES == 1) {
        __shared__ Team<1, NV> teams[4];
        const int64_t row = int64_t(blockIdx.x) * 4 + wave;
        if (row < p.a.rows) score_part<T, 1, NV, TOP>(p, teams[wave], row, 0, 0, lane);
    } else {
        __shared__ Team<WAVES, NV> team;
        const int64_t row = blockIdx.x / uint32_t(p.splits);
        score_part<T, WAVES, NV, TOP>(p, team, row, int(blockIdx.x % uint32_t(p.splits)), wave, lane);
    }
}

// Statistics without alternatives, for calls of many rows: a workgroup streams one row through a running maximum, sum
// and moment in every lane, rescaled once for U vectors.  Vectors start at 16-byte boundaries; the few values in front
// of the first and behind the last one go to a lane each.
// A lane meets vocab / 256 values.  U vectors' are summed by themselves, kGroups such sums one after the other, and what
// that gives goes to a sum in FP64, so that no chain of FP32 additions grows with the vocabulary (one of all values, a best
// token and level others 5 below it, 262,144: log s off by 1.5e-5).  The FP64 sums keep their reference until the maximum
// is kFar above it: what is added is scaled to it, and a row that creeps up does not round all that came before each time.
constexpr float kFar = 4.f;

template <typename T, int U>
__global__ __launch_bounds__(kThreads) void stream_kernel(Rows p) {
    constexpr int VE = Vec<T>::kSize, kGroups = 64 / VE;  // chains of at most 32 additions, then of 8 or 16
    __shared__ float highs[kWaves], sums[kWaves], moments[kWaves];
    const bdm_token_args &a = p.a;
    const int64_t row = blockIdx.x;
    const T *x = static_cast<const T *>(a.logits) + row * a.row_stride;
    const int64_t token = a.tokens[row];
    const float given = to_f32(x[token >= 0 && token < a.vocab ? token : 0]);
    const int lead = int((16 - reinterpret_cast<uintptr_t>(x) % 16) % 16 / sizeof(T));
    const int vectors = (a.vocab - lead) / VE, tail = lead + vectors * VE, thread = int(threadIdx.x);
    const u32x4 *from = reinterpret_cast<const u32x4 *>(x + lead);
    // lanes 0 to 7 take the values in front, lanes 8 to 15 those behind
    const int odd = thread < VE ? (thread < lead ? thread : -1) : (thread < 2 * VE && tail + thread - VE < a.vocab ? tail + thread - VE : -1);
    float high = odd >= 0 ? to_f32(x[odd]) : -INFINITY, sum = 0.f, moment = 0.f;
    const auto add = [&](float v, float &s, float &m) {
        const float d = v - high, e = __builtin_amdgcn_exp2f(d * kLog2E);
        s += e;
        m = fmaf(e, fmaxf(d, -1e30f), m);  // e = 0 there: no 0 * inf
    };
    {
        const float v = high;
        high = fmaxf(high, -FLT_MAX);
        add(v, sum, moment);
    }
    const auto rescale = [&](float to) {
        const float d = fmaxf(high - to, -1e30f), e = __builtin_amdgcn_exp2f(d * kLog2E);
        moment = e * fmaf(sum, d, moment);
        sum *= e;
        high = to;
    };
    // N vectors
    const auto take = [&](const u32x4 *raw, auto count) {
        constexpr int N = decltype(count)::value;
        float v[N][VE], top = high, s = 0.f, m = 0.f;
#pragma unroll
        for (int u = 0; u < N; ++u) {
            Vec<T>::widen(raw[u], v[u]);
#pragma unroll
            for (int j = 0; j < VE; ++j) top = fmaxf(top, v[u][j]);
        }
        rescale(top);
#pragma unroll
        for (int u = 0; u < N; ++u)
#pragma unroll
            for (int j = 0; j < VE; ++j) add(v[u][j], s, m);
        sum += s;
        moment += m;
    };
    double far_sum = 0, far_moment = 0;
    float base = -FLT_MAX;
    int at = thread;
    for (int stop = min(vectors, kGroups * U * kThreads);; stop = min(vectors, stop + kGroups * U * kThreads)) {
        for (; at + (U - 1) * kThreads < stop; at += U * kThreads) {
            u32x4 raw[U];
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = from[at + u * kThreads];
            take(raw, std::integral_constant<int, U>{});
        }
        if (stop == vectors) break;
        if (high > base + kFar) {
            const float d = fmaxf(base - high, -1e30f);
            const double e = double(__builtin_amdgcn_exp2f(d * kLog2E));
            far_moment = e * fma(far_sum, double(d), far_moment);
            far_sum *= e;
            base = high;
        }
        const float d = fmaxf(high - base, 0.f);  // both infinite: the sum is NaN
        const double e = double(__builtin_amdgcn_exp2f(d * kLog2E));
        far_moment = fma(e, fma(double(sum), double(d), double(moment)), far_moment);
        far_sum = fma(e, double(sum), far_sum);
        sum = moment = 0.f;
    }
    for (; at < vectors; at += kThreads) {
        const u32x4 raw = from[at];
        take(&raw, std::integral_constant<int, 1>{});
    }
    if (vectors > kGroups * U * kThreads) {
        const float d = fmaxf(base - high, -1e30f);
        const double e = double(__builtin_amdgcn_exp2f(d * kLog2E));
        moment = float(fma(e, fma(far_sum, double(d), far_moment), double(moment)));
        sum = float(fma(e, far_sum, double(sum)));
    }
    const int wave = thread / kWave;
    rescale(wave_max(high));
    sum = wave_sum(sum);
    moment = wave_sum(moment);
    if (thread % kWave == 0) {
        highs[wave] = high;
        sums[wave] = sum;
        moments[wave] = moment;
    }
    __syncthreads();
    if (thread) return;
    float top = highs[0];
    for (int i = 1; i < kWaves; ++i) top = fmaxf(top, highs[i]);
    float total = 0.f, first = 0.f;
    for (int i = 0; i < kWaves; ++i) {
        high = highs[i], sum = sums[i], moment = moments[i];
        rescale(top);
        total += sum;
        first += moment;
    }
    const float log_sum = logf(total);
    put_row(a, row, token, given, top, log_sum, log_sum - first / total);
}

__device__ __forceinline__ uint64_t largest_key(uint64_t x) {
    const uint32_t high = wave_max(uint32_t(x >> 32));
    return uint64_t(high) << 32 | wave_max(uint32_t(x >> 32) == high ? uint32_t(x) : 0u);
}

// The parts of a row joined: two exchanges between the waves, and the candidates ranked by counting (parts and join of 64
// rows of 50,257 BF16 logits with 8 alternatives: 12.1 us, 3 rows of 262,144 FP32 with 20 12.9; joined by one wave, which
// meets no barrier but ranks alone, 12.0 and 19).
template <typename T>
__global__ __launch_bounds__(kThreads) void join_kernel(Rows p) {
    constexpr int kRoom = 512;
    __shared__ uint64_t list[kRoom], lasts[kWaves], leasts[kWaves];
    __shared__ float highs[kWaves];
    __shared__ float2 sums[kWaves];
    __shared__ int shared_count;
    const bdm_token_args &a = p.a;
    const int64_t row = blockIdx.x;
    const int thread = int(threadIdx.x), wave = thread / kWave, lane = thread % kWave;
    const int k = a.alternatives, total = p.splits * k;
    const float4 *parts = p.parts + row * p.splits;
    const uint64_t *lists = p.lists + row * total;
    const int64_t token = a.tokens[row];
    const T *x = static_cast<const T *>(a.logits) + row * a.row_stride;
    const float given = to_f32(x[token >= 0 && token < a.vocab ? token : 0]);
    // every part's list is in descending order: as many entries as are wanted reach the largest last one of them, and
    // the least of all parts' n-th ones, n the share of a part
    uint64_t last = 0, least = UINT64_MAX;
    float high = -INFINITY;
    const int share = k ? (k + p.splits - 1) / p.splits - 1 : 0;
    for (int i = thread; i < p.splits; i += kThreads) {
        high = fmaxf(high, parts[i].x);
        if (!k) continue;
        last = max(last, lists[i * k + k - 1]);
        least = min(least, lists[i * k + share]);
    }
    high = wave_max(high);
    last = largest_key(last);
    least = ~largest_key(~least);
    if (lane == 0) {
        highs[wave] = high;
        lasts[wave] = last;
        leasts[wave] = least;
    }
    if (thread == 0) shared_count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        high = fmaxf(high, highs[i]);
        last = max(last, lasts[i]);
        least = min(least, leasts[i]);
    }
    const uint64_t bound = max(max(last, least), uint64_t(1));
    const float from = high > -INFINITY ? high : 0.f;
    float sum = 0.f, moment = 0.f;
    for (int i = thread; i < p.splits; i += kThreads) {
        const float4 part = parts[i];
        if (part.y == 0.f) continue;
        const float d = (part.x > -INFINITY ? part.x : 0.f) - from, e = __builtin_amdgcn_exp2f(d * kLog2E);
        sum += part.y * e;
        moment += e == 0.f ? 0.f : e * (part.z + part.y * d);  // d may be near the lowest value
    }
    sum = wave_sum(sum);
    moment = wave_sum(moment);
    for (int first = wave * kWave; first < total; first += kThreads) {
        const uint64_t key = first + lane < total ? lists[first + lane] : 0;
        const uint64_t lanes = __ballot(key >= bound);
        int at = 0;
        if (lane == 0) at = atomicAdd(&shared_count, popcount(lanes));
        at = __builtin_amdgcn_readfirstlane(at) + popcount(lanes & ((1ull << lane) - 1));
        if (key >= bound && at < kRoom) list[at] = key;
    }
    if (lane == 0) sums[wave] = make_float2(sum, moment);
    __syncthreads();
    const int count = shared_count;
    sum = moment = 0.f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        sum += sums[i].x;
        moment += sums[i].y;
    }
    const float log_sum = logf(sum);
    if (thread == 0) put_row(a, row, token, given, from, log_sum, log_sum - moment / sum);
    const auto put = [&](int rank, uint64_t key) {
        a.top_tokens[row * k + rank] = int64_t(~uint32_t(key));
        a.top_log_probs[row * k + rank] = log_probability(unordered(uint32_t(key >> 32)), from, log_sum);
    };
    if (count <= kRoom) {
        for (int i = thread; i < count; i += kThreads) {
            const uint64_t mine = list[i];
            int rank = 0;
#pragma unroll 8
            for (int j = 0; j < count; ++j) rank += list[j] > mine;
            if (rank < k) put(rank, mine);
        }
        return;
    }
    // level lists: one entry after the other
    uint64_t above = UINT64_MAX;
    for (int rank = 0; rank < k; ++rank) {
        uint64_t best = 0;
        for (int i = thread; i < total; i += kThreads) {
            const uint64_t key = lists[i];
            if (key < above && key > best) best = key;
        }
        best = largest_key(best);
        __syncthreads();
        if (lane == 0) lasts[wave] = best;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kWaves; ++i) best = max(best, lasts[i]);
        if (thread == 0) put(rank, best);
        above = best;
    }
}

// The gradient of a row's logits, one pass over them: a team of LANES lanes takes U vectors a lane of one row, which
// start at the gradient's 16-byte boundaries (the logits' too, where both are as torch allocates them); the few values
// in front of the first and behind the last go to a lane each of the row's first team.  Loads and stores pass by the
// caches: kept there, what was written made the next forward slower (its loss and gradient, 8,192 rows of 50,257 BF16
// logits: 477 us, 430 so).  `TOPS`: gradients of the
// alternatives arrive too.
template <typename T, int LANES, int U, bool TOPS>
__global__ __launch_bounds__(kThreads) void token_gradient_kernel(bdm_token_grad_args a, int parts) {
    constexpr int VE = Vec<T>::kSize;
    typedef u32x4 AnyBits __attribute__((aligned(2)));
    __shared__ int spots[kThreads / LANES][kAlternativesMax];
    __shared__ float weights[kThreads / LANES][kAlternativesMax];
    const int team = int(threadIdx.x) / LANES, lane = int(threadIdx.x) % LANES;
    const int64_t item = int64_t(blockIdx.x) * (kThreads / LANES) + team, row = item / parts;
    if (row >= a.rows) return;
    const int part = int(item % parts);
    const T *x = static_cast<const T *>(a.logits) + row * a.row_stride;
    T *out = static_cast<T *>(a.grad_logits) + row * a.vocab;
    const int lead = min(int((16 - reinterpret_cast<uintptr_t>(out) % 16) % 16 / sizeof(T)), a.vocab);
    const int vectors = (a.vocab - lead) / VE, tail = lead + vectors * VE, first = part * LANES * U + lane;
    u32x4 raw[U];
    if (vectors > 0) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            raw[u] = __builtin_nontemporal_load(
                reinterpret_cast<const AnyBits *>(x + lead + min(first + u * LANES, vectors - 1) * VE));
    }
    const int64_t token = a.tokens[row];
    const float high = a.stats[2 * row], log_sum = a.stats[2 * row + 1];
    const float h = a.grad_entropy ? a.grad_entropy[row] : 0.f, entropy = a.grad_entropy ? a.entropy[row] : 0.f;
    float given = 0.f;
    if (token != a.ignore_index && (a.grad_loss || a.grad_log_probs)) {
        given = a.grad_loss ? -(a.grad_loss[0] * a.inverse_count[0]) : a.grad_log_probs[row];
        if (token < 0 || token >= a.vocab) given = NAN;
    }
    float total = given;
    if constexpr (TOPS) {
        if (lane < a.alternatives) {
            spots[team][lane] = int(a.top_tokens[row * a.alternatives + lane]);
            weights[team][lane] = a.grad_top_log_probs[row * a.alternatives + lane];
        }
        team_sync<LANES / kWave>();
        for (int k = 0; k < a.alternatives; ++k) total += weights[team][k];
    }
    const int at = token >= 0 && token < a.vocab ? int(token) : -VE;
    // no distribution, or no gradient: an ignored token's row may hold a NaN, and 0 * NaN is not 0
    const bool none = log_sum == -INFINITY || (!TOPS && !a.grad_entropy && token == a.ignore_index);
    // N values from index `start` on
    const auto gradient = [&](int start, float *v, auto count) {
        constexpr int N = decltype(count)::value;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const float lp = (v[j] - high) - log_sum, p = __builtin_amdgcn_exp2f(lp * kLog2E);
            v[j] = none ? 0.f : -p * (total + h * (fmaxf(lp, -1e30f) + entropy));  // p = 0 there: no 0 * inf
        }
        if (none) return;
        const auto add = [&](int place, float weight) {
            if (unsigned(place) >= unsigned(N)) return;
#pragma unroll
            for (int j = 0; j < N; ++j) v[j] += j == place ? weight : 0.f;
        };
        if constexpr (TOPS)
            for (int k = 0; k < a.alternatives; ++k) add(spots[team][k] - start, weights[team][k]);
        add(at - start, given);
    };
    const int odd = part ? -1 : lane < VE ? (lane < lead ? lane : -1)
                              : (lane < 2 * VE && tail + lane - VE < a.vocab ? tail + lane - VE : -1);
    if (odd >= 0) {
        float v = to_f32(x[odd]);
        gradient(odd, &v, std::integral_constant<int, 1>{});
        out[odd] = from_f32<T>(v);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int vector = first + u * LANES;
        if (vector >= vectors) break;
        float v[VE];
        Vec<T>::widen(raw[u], v);
        gradient(lead + vector * VE, v, std::integral_constant<int, VE>{});
        u32x4 bits;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (VE == 8)
                bits[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
            else
                bits[j] = __float_as_uint(v[j]);
        }
        __builtin_nontemporal_store(bits, reinterpret_cast<u32x4 *>(out + lead + vector * VE));
    }
}

// loss = -sum of the log-probabilities / their number, in FP64 and always in the same order.  One workgroup: its time is
// that of the loads' trips, eight rows a lane at a time.
constexpr int kLossThreads = 1024;

__global__ __launch_bounds__(kLossThreads) void token_loss_kernel(const float *log_probs, const int64_t *tokens, int64_t rows,
                                                                  int64_t ignore_index, float *loss, float *inverse_count) {
    constexpr int U = 8;
    __shared__ double sums[kLossThreads / kWave];
    __shared__ int64_t counts[kLossThreads / kWave];
    double sum = 0;
    int64_t count = 0;
    for (int64_t at = threadIdx.x; at < rows; at += U * kLossThreads) {
        float value[U];
        int64_t token[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t i = min(at + u * kLossThreads, rows - 1);
            value[u] = log_probs[i];
            token[u] = tokens[i];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (at + u * kLossThreads >= rows || token[u] == ignore_index) continue;
            sum += double(value[u]);
            ++count;
        }
    }
#pragma unroll
    for (int step = kWave / 2; step; step >>= 1) {
        sum += __shfl_xor(sum, step, kWave);
        count += __shfl_xor(count, step, kWave);
    }
    if (threadIdx.x % kWave == 0) {
        sums[threadIdx.x / kWave] = sum;
        counts[threadIdx.x / kWave] = count;
    }
    __syncthreads();
    if (threadIdx.x) return;
    for (int i = 1; i < kLossThreads / kWave; ++i) {
        sum += sums[i];
        count += counts[i];
    }
    *loss = float(-sum / double(count));
    *inverse_count = float(1 / double(count));
}

int check_rows(const char *what, int64_t rows, int64_t row_stride, int32_t vocab, int32_t dtype, int32_t alternatives) {
    if (rows < 0 || vocab <= 0 || row_stride < 0 || alternatives < 0 || alternatives > vocab)
        return fail(BDM_ERR_INVALID, "%s: bad geometry", what);
    if (dtype != BDM_BF16 && dtype != BDM_F32) return fail(BDM_ERR_INVALID, "%s: dtype", what);
    if (alternatives > kAlternativesMax)
        return fail(BDM_ERR_UNSUPPORTED, "%s: more than %d alternatives", what, kAlternativesMax);
    if (vocab > kVocabMax) return fail(BDM_ERR_UNSUPPORTED, "%s: vocabulary beyond 2^24", what);
    if (!grid_fits(rows, kThreads)) return fail(BDM_ERR_UNSUPPORTED, "%s: too many rows", what);
    return BDM_OK;
}

// A team's waves and values a lane, and the parts of a row.  One wave a row as long as it holds it (8,192 rows of 2,000
// BF16 logits with 4 alternatives: 12.6 us, 28.3 by four waves), then four; parts of at most 16,384, all alike, which
// leave several workgroups to a CU (4,096 rows of 50,257 with 8: 113 us, 127 in parts of at most 8,192); half as long ones
// where there are few workgroups (a row of 50,257 with 8: 9.5 us, 10.1 otherwise; 64 rows 12.1 and 12.0).
struct Shape {
    int waves, values, splits;
};

Shape shape_of(const bdm_token_args &a) {
    for (const int values : {8, 16, 32})
        if (a.vocab <= kWave * values) return {1, values, 1};
    for (const int values : {16, 32})
        if (a.vocab <= 256 * values) return {4, values, 1};
    const int splits = (a.vocab + 16383) / 16384;
    if (splits > 1 && a.rows * splits < 256) return {4, 32, (a.vocab + 8191) / 8192};
    for (const int values : {48, 56})
        if (a.vocab <= 256 * values * splits) return {4, values, splits};
    return {4, 64, splits};
}

template <typename T, int WAVES, int VALUES>
void launch_scores(const Rows &p, hipStream_t s) {
    constexpr int NV = VALUES / Vec<T>::kSize;
    const int64_t blocks = WAVES == 1 ? (p.a.rows + 3) / 4 : p.a.rows * p.splits;
    if (p.a.alternatives)
        score_kernel<T, WAVES, NV, true><<<unsigned(blocks), kThreads, 0, s>>>(p);
    else
        score_kernel<T, WAVES, NV, false><<<unsigned(blocks), kThreads, 0, s>>>(p);
}

template <typename T>
int launch_scores(const Rows &p, const Shape &shape, hipStream_t s) {
    if (shape.waves == 1)
        shape.values == 8 ? launch_scores<T, 1, 8>(p, s) : shape.values == 16 ? launch_scores<T, 1, 16>(p, s) : launch_scores<T, 1, 32>(p, s);
    else if (shape.values <= 32)
        shape.values == 16 ? launch_scores<T, 4, 16>(p, s) : launch_scores<T, 4, 32>(p, s);
    else
        shape.values == 48 ? launch_scores<T, 4, 48>(p, s) : shape.values == 56 ? launch_scores<T, 4, 56>(p, s) : launch_scores<T, 4, 64>(p, s);
    if (int rc = check_launch("score_kernel")) return rc;
    if (p.splits == 1) return BDM_OK;
    join_kernel<T><<<unsigned(p.a.rows), kThreads, 0, s>>>(p);
    return check_launch("join_kernel");
}

// Whether a call without alternatives streams its rows (8,192 rows of 50,257 BF16: 149 us, 196 from registers; 2,048 of
// 4,099 6.5 and 8.7; 255 of 65,536 10.7 and 12.3): not short rows (8,192 of 4,096: 17.6 us, 15.4 from registers), nor few
// long ones, whose parts work side by side (a row of 131,072: 12.1 us, 5.6 in parts; 255 22.9 and 17.8).  Both bounds are
// rough: some 64 rows of 50,000 to 65,536 tokens would gain by parts (of 65,536: 9.3 us, 7.7 in parts; 128 rows 9.9 and
// 9.3), and so would few hundred of 131,072 and more (256: 22.8 us, 17.9 in parts; 1,024 53 either way; 512 of 262,144 51
// and 53).
bool streams(const bdm_token_args &a) {
    return !a.alternatives && a.vocab > 4096 && (a.rows >= 256 || a.vocab <= 65536);
}

template <typename T, int LANES, int U>
int launch_gradient(const bdm_token_grad_args &a, hipStream_t s) {
    constexpr int kPart = LANES * U * Vec<T>::kSize, kTeams = kThreads / LANES;
    const int parts = (a.vocab + kPart - 1) / kPart;
    const int64_t blocks = (a.rows * parts + kTeams - 1) / kTeams;
    if (!grid_fits(blocks, kThreads)) return fail(BDM_ERR_UNSUPPORTED, "token_log_probs_backward: too many rows");
    if (a.grad_top_log_probs)
        token_gradient_kernel<T, LANES, U, true><<<unsigned(blocks), kThreads, 0, s>>>(a, parts);
    else
        token_gradient_kernel<T, LANES, U, false><<<unsigned(blocks), kThreads, 0, s>>>(a, parts);
    return check_launch("token_gradient_kernel");
}

// A wave a part for short rows (8,192 of 192 BF16 5.2 us, 10.9 by workgroups; of 2,048 12.9 and 17.9; 4,096 of 4,096 13.0
// and 15.3), a workgroup for long ones (4,096 of 6,000: 19.9 us, 21.2 by waves; of 8,192 with 8 alternatives 27.5 either
// way; 8,192 of 50,257 290 and 298).
template <typename T>
int launch_gradient(const bdm_token_grad_args &a, hipStream_t s) {
    return a.vocab <= 4096 ? launch_gradient<T, 64, 4>(a, s) : launch_gradient<T, 256, 4>(a, s);
}

}  // namespace
}  // namespace bdm

using namespace bdm;

extern "C" size_t bdm_token_log_probs_workspace_size(const bdm_token_args *a) {
    if (!a || a->rows <= 0 || a->vocab <= 0 || a->alternatives < 0 || a->vocab > kVocabMax) return 0;
    const size_t splits = streams(*a) ? 1 : size_t(shape_of(*a).splits);
    if (splits == 1) return 0;
    return size_t(a->rows) * splits * (sizeof(float4) + size_t(a->alternatives) * sizeof(uint64_t));
}

extern "C" int bdm_token_log_probs(const bdm_token_args *a, void *workspace, size_t workspace_bytes, void *stream) {
    if (!a) return fail(BDM_ERR_INVALID, "token_log_probs: null args");
    if (int rc = check_rows("token_log_probs", a->rows, a->row_stride, a->vocab, a->dtype, a->alternatives)) return rc;
    if (a->rows == 0) return BDM_OK;
    if (!a->logits || !a->tokens || !a->log_probs || (a->alternatives && (!a->top_log_probs || !a->top_tokens)))
        return fail(BDM_ERR_INVALID, "token_log_probs: null pointer");
    if (streams(*a)) {
        const Rows p{*a, nullptr, nullptr, 1};
        if (a->dtype == BDM_BF16)
            stream_kernel<bf16_t, 4><<<unsigned(a->rows), kThreads, 0, as_stream(stream)>>>(p);
        else
            stream_kernel<float, 4><<<unsigned(a->rows), kThreads, 0, as_stream(stream)>>>(p);
        return check_launch("stream_kernel");
    }
    const Shape shape = shape_of(*a);
    if (!grid_fits(a->rows * shape.splits, kThreads)) return fail(BDM_ERR_UNSUPPORTED, "token_log_probs: too many rows");
    if (shape.splits > 1 && (!workspace || workspace_bytes < bdm_token_log_probs_workspace_size(a) || !aligned(workspace, 16)))
        return fail(BDM_ERR_INVALID, "token_log_probs: workspace too small or not aligned to 16 bytes");
    Rows p{*a, static_cast<float4 *>(workspace), nullptr, shape.splits};
    p.lists = reinterpret_cast<uint64_t *>(p.parts + a->rows * shape.splits);
    return a->dtype == BDM_BF16 ? launch_scores<bf16_t>(p, shape, as_stream(stream))
                                : launch_scores<float>(p, shape, as_stream(stream));
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
        return launch_gradient<bf16_t>(*a, s);
    return launch_gradient<float>(*a, s);
}

extern "C" int bdm_token_loss(const float *log_probs, const int64_t *tokens, int64_t rows, int64_t ignore_index,
                              float *loss, float *inverse_count, void *stream) {
    if (rows < 0) return fail(BDM_ERR_INVALID, "token_loss: bad geometry");
    if ((rows && (!log_probs || !tokens)) || !loss || !inverse_count)
        return fail(BDM_ERR_INVALID, "token_loss: null pointer");
    token_loss_kernel<<<1, kLossThreads, 0, as_stream(stream)>>>(log_probs, tokens, rows, ignore_index, loss, inverse_count);
    return check_launch("token_loss_kernel");
}
