// Layer normalization, forward and backward, also behind a residual add.
//
//   mu = mean x,  v = mean (x - mu)^2,  r = 1 / sqrt(v + eps),  xh = (x - mu) r,  y = xh w + b,
//   dx = r (dy w - mean(dy w) - xh mean(dy w xh)) + dsum,   dw = sum over rows dy xh,   db = sum over rows dy.
// With a residual, x is the rounded sum, written beside y.  The statistics and
// sums are FP32, the variance from the centred values.
//
// A row is held in registers by a team of waves, the next one loaded meanwhile; the backward keeps its columns' parts of
// dw and db there too, over all rows of the team.  Every wave centres its values on its own mean c first, and one
// exchange joins what all sums need: with d = x - c and n the wave's columns,
//   mu = (sum over waves n c + sum d) / width,   sum (x - mu)^2 = sum d^2 + 2 (c - mu) sum d + n (c - mu)^2,
//   sum g (x - mu) = sum g d + (c - mu) sum g       (g = dy w),
// so that rows far from zero lose nothing, and a team of several waves waits once a row.
//
// Bound by HBM where rows are many (32,768 of 1,024 BF16 behind a residual add, 268 MB each way: forward 46 us, backward
// 46 and 4 for the parts' sums, 5.8 TB/s); by the instructions of a row's sums, issued by the two waves a SIMD that the
// registers admit, in the backward of wider BF16 rows (8,192 of 2,048: 27 us, 3.7 TB/s, the SIMDs issue vector
// instructions 73% of the time) and of narrow ones (65,536 of 64: 18 us, 83%); by latency where rows are few (64 of 1,024:
// 4 and 7 us).
#include <type_traits>

#include "bdm_common.h"
#include "epilogue_ops.h"
#include "selection_ops.h"

namespace bdm {
namespace {

constexpr int kMaxWidth = 16384;
constexpr int kSumWaves = 16;

template <int N, typename P>
struct __attribute__((packed, aligned(sizeof(P)))) Packed {
    P at[N];
};

// The columns of a lane: NV vectors of VE, the team's lanes next to each other.  Vector i starts at column `start(i)`:
// the last one of a row early enough to end with it, the columns that the one before holds already not `valid` in it.
template <int LANES, int VE>
struct Columns {
    int thread, width;
    __device__ __forceinline__ int begin(int i) const { return (thread + i * LANES) * VE; }
    __device__ __forceinline__ int start(int i) const { return width < VE ? 0 : min(begin(i), width - VE); }
    __device__ __forceinline__ bool full(int i) const { return begin(i) + VE <= width; }
    __device__ __forceinline__ bool valid(int i, int j) const {
        const int at = start(i) + j;
        return at >= begin(i) && at < width;
    }
    template <typename T>
    __device__ __forceinline__ u32x4 load(const T *row, int i) const {
        if (width >= VE) return reinterpret_cast<const AnyVector<T> *>(row + start(i))->bits;
        // element by element, in a loop that takes few registers
        u32x4 raw{};
#pragma unroll 1
        for (int j = 0; j < width; ++j) {
            const uint32_t bits = __float_as_uint(to_f32(row[j]));
            const int word = VE == 8 ? j / 2 : j;
            const uint32_t part = VE == 8 && j % 2 == 0 ? bits >> 16 : bits;
#pragma unroll
            for (int q = 0; q < 4; ++q) raw[q] |= q == word ? part : 0u;
        }
        return raw;
    }
    // values of vector i, 0 where it has none
    template <typename T>
    __device__ __forceinline__ void widen(u32x4 raw, int i, float (&out)[VE]) const {
        Vec<T>::widen(raw, out);
        clear(i, out);
    }
    __device__ __forceinline__ void clear(int i, float (&out)[VE]) const {
        if (full(i)) return;
#pragma unroll
        for (int j = 0; j < VE; ++j) out[j] = valid(i, j) ? out[j] : 0.f;
    }
    template <typename P>
    __device__ __forceinline__ void parameters(const void *p, int i, float other, float (&out)[VE]) const {
        const P *from = static_cast<const P *>(p);
        if (!p) {
#pragma unroll
            for (int j = 0; j < VE; ++j) out[j] = other;
        } else if (width >= VE) {
            const Packed<VE, P> some = *reinterpret_cast<const Packed<VE, P> *>(from + start(i));
#pragma unroll
            for (int j = 0; j < VE; ++j) out[j] = to_f32(some.at[j]);
        } else {
#pragma unroll
            for (int j = 0; j < VE; ++j) out[j] = 0.f;
#pragma unroll 1
            for (int at = 0; at < width; ++at) {
                const float value = to_f32(from[at]);
#pragma unroll
                for (int j = 0; j < VE; ++j) out[j] = j == at ? value : out[j];
            }
        }
    }
    // FP32 sums of vector i's columns
    __device__ __forceinline__ void sums(float *to, int i, const float (&v)[VE]) const {
        if (full(i)) {
            Packed<VE, float> some;
#pragma unroll
            for (int j = 0; j < VE; ++j) some.at[j] = v[j];
            *reinterpret_cast<Packed<VE, float> *>(to + begin(i)) = some;
        } else {
#pragma unroll
            for (int j = 0; j < VE; ++j)
                if (valid(i, j)) to[start(i) + j] = v[j];
        }
    }
    template <typename T>
    __device__ __forceinline__ void store(T *row, int i, const float (&v)[VE]) const {
        if (full(i)) {
            u32x4 bits;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (VE == 8)
                    bits[j] = pack_bf16x2(v[2 * j], v[2 * j + 1]);
                else
                    bits[j] = __float_as_uint(v[j]);
            }
            reinterpret_cast<AnyVector<T> *>(row + begin(i))->bits = bits;
        } else if (begin(i) < width) {
#pragma unroll
            for (int j = 0; j < VE; ++j)
                if (valid(i, j)) row[start(i) + j] = from_f32<T>(v[j]);
        }
    }
};

template <typename T>
struct Rows {
    const T *x, *residual, *grad_out, *grad_sum;
    const void *weight, *bias;
    T *sum_out, *out;
    float *partials;
    int64_t rows;
    int width;
    float eps;
};

// A team of 16 waves has 128 registers a lane: it loads a row when its turn comes, and the parameters with every row.
constexpr int kLeanLanes = 1024;

template <int CONTROL>
__device__ __forceinline__ float dpp(float x) {
    return __uint_as_float(uint32_t(__builtin_amdgcn_update_dpp(0, int(__float_as_uint(x)), CONTROL, 0xf, 0xf, false)));
}
// The sum over each 16 lanes, in all of them: neighbours, pairs, then the mirrored half and row.
__device__ __forceinline__ float row_total(float x) {
    x += dpp<0xb1>(x);   // quad_perm 1 0 3 2
    x += dpp<0x4e>(x);   // quad_perm 2 3 0 1
    x += dpp<0x141>(x);  // row_half_mirror
    x += dpp<0x140>(x);  // row_mirror
    return x;
}
// The sum over the lanes of a row's team, or over its wave where the team has several.
template <int LANES>
__device__ __forceinline__ float lanes_total(float x) {
    if constexpr (LANES >= kWave) {
        return wave_sum(x);
    } else {
        x = row_total(x);
        if constexpr (LANES == 32) x += __shfl_xor(x, 16, kWave);
        return x;
    }
}

// What a wave gives to its team of a row.
struct Sums {
    float count, centre, d, square, g, gd;
};

// The row's mean as an offset from the wave's own centre, 1 / deviation, mean g and mean g xh.
struct Statistics {
    float offset, scale, g, dot;
};

template <int WAVES, bool GRADIENT>
__device__ __forceinline__ Statistics join(Sums mine, Sums (&shared)[2][WAVES], int turn, int wave, int lane, int width,
                                           float eps) {
    const float inverse = 1.f / float(width);
    Statistics out{};
    if constexpr (WAVES == 1) {
        out.offset = mine.d * inverse;
        out.scale = rsqrtf(fmaxf(mine.square * inverse - out.offset * out.offset, 0.f) + eps);
        out.g = mine.g * inverse;
        out.dot = (mine.gd - out.offset * mine.g) * inverse * out.scale;
    } else {
        // lane i of 16 takes wave i
        static_assert(WAVES <= 16);
        if (lane == 0) shared[turn][wave] = mine;
        __syncthreads();
        const int from = lane % 16;
        Sums s = shared[turn][min(from, WAVES - 1)];
        const float pivot = shared[turn][0].centre;
        if (from >= WAVES) s = Sums{0.f, pivot, 0.f, 0.f, 0.f, 0.f};
        const float mean = row_total(fmaf(s.count, s.centre - pivot, s.d)) * inverse;  // from the pivot
        const float away = (s.centre - pivot) - mean;
        const float square = row_total(s.square + away * (2.f * s.d + s.count * away));
        out.offset = mean - (mine.centre - pivot);
        out.scale = rsqrtf(fmaxf(square * inverse, 0.f) + eps);
        if constexpr (GRADIENT) {
            out.g = row_total(s.g) * inverse;
            out.dot = row_total(s.gd + away * s.g) * inverse * out.scale;
        }
    }
    return out;
}

template <int LANES, int VE, int NV>
__device__ __forceinline__ float columns_of_wave(const Columns<LANES, VE> &c, int wave) {
    constexpr int kMine = LANES < kWave ? LANES : kWave;
    int count = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) count += min(max(c.width - (wave * kWave + i * LANES) * VE, 0), kMine * VE);
    return float(count);
}

// Teams of LANES lanes take the rows in turn; a workgroup of 256 lanes holds several teams of a wave or less, one of
// several waves is a workgroup.
template <typename T, typename P, int LANES, int NV, bool RESIDUAL>
__global__ __launch_bounds__(LANES <= 256 ? 256 : LANES) void layer_norm_kernel(Rows<T> p) {
    constexpr int VE = Vec<T>::kSize, WAVES = LANES <= kWave ? 1 : LANES / kWave, kTeams = WAVES == 1 ? 256 / LANES : 1;
    constexpr bool kLean = LANES == kLeanLanes;
    __shared__ Sums shared[2][WAVES];
    const int lane = int(threadIdx.x) % kWave, wave = WAVES == 1 ? 0 : int(threadIdx.x) / kWave;
    const Columns<LANES, VE> c{int(threadIdx.x) % LANES, p.width};
    const int64_t step = int64_t(gridDim.x) * kTeams;
    int64_t row = int64_t(blockIdx.x) * kTeams + (WAVES == 1 ? int(threadIdx.x) / LANES : 0);
    if (row >= p.rows) return;
    u32x4 x[NV], r[NV];
    const auto load = [&](int64_t at) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            x[i] = c.load(p.x + at * p.width, i);
            if constexpr (RESIDUAL) r[i] = c.load(p.residual + at * p.width, i);
        }
    };
    float weight[NV][VE], bias[NV][VE];
    if constexpr (!kLean) {
        load(row);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            c.template parameters<P>(p.weight, i, 1.f, weight[i]);
            c.template parameters<P>(p.bias, i, 0.f, bias[i]);
        }
    }
    const float count = columns_of_wave<LANES, VE, NV>(c, wave);
    int turn = 0;
    for (; row < p.rows; row += step, turn ^= 1) {
        const int64_t base = row * p.width;
        if constexpr (kLean) load(row);
        float v[NV][VE];
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            c.template widen<T>(x[i], i, v[i]);
            if constexpr (RESIDUAL) {
                float other[VE];
                c.template widen<T>(r[i], i, other);
#pragma unroll
                for (int j = 0; j < VE; ++j) v[i][j] = round_to<T>(v[i][j] + other[j]);
                c.store(p.sum_out + base, i, v[i]);
            }
#pragma unroll
            for (int j = 0; j < VE; ++j) sum += v[i][j];
        }
        if (!kLean && row + step < p.rows) load(row + step);
        Sums s{};
        s.count = count;
        s.centre = lanes_total<LANES>(sum) / fmaxf(count, 1.f);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int j = 0; j < VE; ++j) v[i][j] -= s.centre;
            c.clear(i, v[i]);
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                s.d += v[i][j];
                s.square = fmaf(v[i][j], v[i][j], s.square);
            }
        }
        s.d = lanes_total<LANES>(s.d);
        s.square = lanes_total<LANES>(s.square);
        const Statistics t = join<WAVES, false>(s, shared, turn, wave, lane, p.width, p.eps);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (kLean) {
                c.template parameters<P>(p.weight, i, 1.f, weight[i]);
                c.template parameters<P>(p.bias, i, 0.f, bias[i]);
            }
            float y[VE];
#pragma unroll
            for (int j = 0; j < VE; ++j) y[j] = fmaf((v[i][j] - t.offset) * t.scale, weight[i][j], bias[i][j]);
            c.store(p.out + base, i, y);
        }
    }
}

// Lanes of a backward's workgroup: several teams share one, and its LDS adds up their columns' sums (8,192 rows of 2,048
// BF16: 32 us with one team of two waves, 28 with four).
constexpr int backward_block(int lanes) { return lanes <= kWave ? 256 : lanes <= 512 ? 512 : lanes; }

template <typename T, typename P, int LANES, int NV, bool SUM>
__global__ __launch_bounds__(backward_block(LANES)) void layer_norm_backward_kernel(Rows<T> p) {
    constexpr int VE = Vec<T>::kSize, WAVES = LANES <= kWave ? 1 : LANES / kWave, kBlock = backward_block(LANES);
    constexpr int kTeams = kBlock / LANES, kColumns = LANES * NV * VE;
    constexpr bool kLean = LANES == kLeanLanes;
    __shared__ Sums shared[kTeams][2][WAVES];
    __shared__ float slice[kTeams][kTeams > 1 ? kColumns : 1];
    const int lane = int(threadIdx.x) % kWave, wave = WAVES == 1 ? 0 : int(threadIdx.x) % LANES / kWave;
    const int team = int(threadIdx.x) / LANES;
    const Columns<LANES, VE> c{int(threadIdx.x) % LANES, p.width};
    const int64_t step = int64_t(gridDim.x) * kTeams;
    int64_t row = int64_t(blockIdx.x) * kTeams + team;
    u32x4 x[NV], dy[NV], ds[NV];
    const auto load = [&](int64_t at) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            x[i] = c.load(p.x + at * p.width, i);
            dy[i] = c.load(p.grad_out + at * p.width, i);
            if constexpr (SUM) ds[i] = c.load(p.grad_sum + at * p.width, i);
        }
    };
    if (!kLean && row < p.rows) load(row);
    float weight[NV][VE], dw[NV][VE], db[NV][VE];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        if constexpr (!kLean) c.template parameters<P>(p.weight, i, 1.f, weight[i]);
#pragma unroll
        for (int j = 0; j < VE; ++j) dw[i][j] = db[i][j] = 0.f;
    }
    const float count = columns_of_wave<LANES, VE, NV>(c, wave);
    int turn = 0;
    // the teams of a workgroup take the same turns: those of several waves wait for each other
    for (int64_t first = int64_t(blockIdx.x) * kTeams; first < p.rows; first += step, row += step, turn ^= 1) {
        const bool live = row < p.rows;
        const int64_t base = row * p.width;
        if (kLean && live) load(row);
        float v[NV][VE], g[NV][VE], more[NV][VE];
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            c.template widen<T>(x[i], i, v[i]);
            c.template widen<T>(dy[i], i, g[i]);
            if constexpr (SUM) Vec<T>::widen(ds[i], more[i]);
#pragma unroll
            for (int j = 0; j < VE; ++j) sum += v[i][j];
        }
        if (!kLean && row + step < p.rows) load(row + step);
        Sums s{};
        s.count = count;
        s.centre = lanes_total<LANES>(sum) / fmaxf(count, 1.f);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
#pragma unroll
            for (int j = 0; j < VE; ++j) v[i][j] -= s.centre;
            c.clear(i, v[i]);
            if constexpr (kLean) c.template parameters<P>(p.weight, i, 1.f, weight[i]);
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                const float gw = g[i][j] * weight[i][j];
                s.d += v[i][j];
                s.square = fmaf(v[i][j], v[i][j], s.square);
                s.g += gw;
                s.gd = fmaf(gw, v[i][j], s.gd);
            }
        }
        s.d = lanes_total<LANES>(s.d);
        s.square = lanes_total<LANES>(s.square);
        s.g = lanes_total<LANES>(s.g);
        s.gd = lanes_total<LANES>(s.gd);
        const Statistics t = join<WAVES, true>(s, shared[team], turn, wave, lane, p.width, p.eps);
        if (!live) continue;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if constexpr (kLean) c.template parameters<P>(p.weight, i, 1.f, weight[i]);
            float dx[VE];
#pragma unroll
            for (int j = 0; j < VE; ++j) {
                const float xh = (v[i][j] - t.offset) * t.scale;
                dw[i][j] = fmaf(g[i][j], xh, dw[i][j]);
                db[i][j] += g[i][j];
                dx[j] = (g[i][j] * weight[i][j] - t.g - xh * t.dot) * t.scale;
                if constexpr (SUM) dx[j] += more[i][j];
            }
            c.store(p.out + base, i, dx);
        }
    }
    float *part = p.partials + int64_t(blockIdx.x) * 2 * p.width;
    if constexpr (kTeams == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            c.sums(part, i, dw[i]);
            c.sums(part + p.width, i, db[i]);
        }
    } else {
        // the teams' sums, in their order
        const auto put = [&](const float (&from)[NV][VE], float *to) {
#pragma unroll
            for (int i = 0; i < NV; ++i) c.sums(slice[team], i, from[i]);
            __syncthreads();
            for (int at = threadIdx.x; at < p.width; at += kBlock) {
                float total = slice[0][at];
#pragma unroll
                for (int i = 1; i < kTeams; ++i) total += slice[i][at];
                to[at] = total;
            }
            __syncthreads();
        };
        put(dw, part);
        put(db, part + p.width);
    }
}

// The parts' sums, column by column: wave k of a workgroup's 16 takes the parts k, k + 16, ..., and the waves' sums are
// added in their order.
__global__ __launch_bounds__(kSumWaves * kWave) void layer_norm_param_kernel(const float *partials, int parts, int width,
                                                                             void *dw, void *db, int dtype) {
    __shared__ float slice[kSumWaves][kWave];
    const int lane = int(threadIdx.x) % kWave, wave = int(threadIdx.x) / kWave;
    const int c = int(blockIdx.x) * kWave + lane;
    float total = 0.f;
    if (c < 2 * width) {
#pragma unroll 8
        for (int i = wave; i < parts; i += kSumWaves) total += partials[int64_t(i) * 2 * width + c];
    }
    slice[wave][lane] = total;
    __syncthreads();
    if (wave != 0 || c >= 2 * width) return;
    float sum = slice[0][lane];
    for (int k = 1; k < kSumWaves; ++k) sum += slice[k][lane];
    void *out = c < width ? dw : db;
    if (!out) return;
    const int at = c < width ? c : c - width;
    if (dtype == BDM_BF16)
        static_cast<bf16_t *>(out)[at] = from_f32<bf16_t>(sum);
    else
        static_cast<float *>(out)[at] = sum;
}

int check_rows(const char *what, int64_t rows, int32_t width, int32_t dtype, int32_t param_dtype) {
    if (rows < 0 || width <= 0) return fail(BDM_ERR_INVALID, "%s: bad geometry", what);
    if (width > kMaxWidth) return fail(BDM_ERR_UNSUPPORTED, "%s: width %d > %d", what, width, kMaxWidth);
    if ((dtype != BDM_BF16 && dtype != BDM_F32) || (param_dtype != BDM_BF16 && param_dtype != BDM_F32))
        return fail(BDM_ERR_INVALID, "%s: dtype", what);
    if (rows >= (int64_t(1) << 40)) return fail(BDM_ERR_UNSUPPORTED, "%s: too many rows", what);
    return BDM_OK;
}

// Lanes of a team and vectors of a lane for a width: eight values a lane up to a wave's 512 columns, so that narrow rows
// share a wave (65,536 rows of 64 BF16: 8.7 us forward, 20.8 with a wave a row), then sixteen, which halve the exchanges
// (32,768 rows of 1,024 BF16, backward: 43 us, 49 by two waves with eight values; 4,096 of 8,192: 50 and 61).
template <typename T, typename F>
void with_shape(int width, F f) {
    constexpr int kVectors = 8 / Vec<T>::kSize;
    const auto shape = [&](auto lanes, auto vectors) { f(lanes, vectors); };
    const auto eight = std::integral_constant<int, kVectors>{};
    const auto sixteen = std::integral_constant<int, 2 * kVectors>{};
    if (width <= 128)
        shape(std::integral_constant<int, 16>{}, eight);
    else if (width <= 256)
        shape(std::integral_constant<int, 32>{}, eight);
    else if (width <= 512)
        shape(std::integral_constant<int, 64>{}, eight);
    else if (width <= 1024)
        shape(std::integral_constant<int, 64>{}, sixteen);
    else if (width <= 2048)
        shape(std::integral_constant<int, 128>{}, sixteen);
    else if (width <= 4096)
        shape(std::integral_constant<int, 256>{}, sixteen);
    else if (width <= 8192)
        shape(std::integral_constant<int, 512>{}, sixteen);
    else
        shape(std::integral_constant<int, 1024>{}, sixteen);
}

// Workgroups of `block` lanes for a pass over the rows by teams of `lanes`: as many as there is work for, at most `waves`
// waves.
int64_t blocks_of(int64_t rows, int lanes, int block, int64_t waves) {
    const int64_t teams = block / lanes, blocks = (rows + teams - 1) / teams, most = waves * kWave / block;
    return blocks < most ? blocks : most;
}
constexpr int64_t kForwardWaves = 256 * 32;

// The backward's workgroups, each of which leaves its columns' sums: as many waves as the registers of 16 values a lane
// admit, twice as many with 8 values or without a row loaded ahead (more of 16 wait for the first ones: 8,192 rows of
// 2,048 BF16 28 us with 2,048 waves, 34 with 3,072, 32 with 4,096, 32,768 of 1,024 43, 42 and 48; 2,048 rows of 16,384 83
// with 2,048, 60 with 4,096, 65,536 of 256 29 and 28).
int64_t backward_parts(int64_t rows, int width) {
    int64_t parts = 0;
    with_shape<bf16_t>(width, [&](auto lanes, auto vectors) {
        constexpr bool kMany = decltype(vectors)::value == 1 || decltype(lanes)::value == kLeanLanes;
        parts = blocks_of(rows, decltype(lanes)::value, backward_block(decltype(lanes)::value), kMany ? 4096 : 2048);
    });
    return parts;
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
    const auto run = [&](auto element, auto parameter) {
        using T = decltype(element);
        using P = decltype(parameter);
        const Rows<T> p{static_cast<const T *>(x), static_cast<const T *>(residual), nullptr, nullptr, weight, bias,
                        static_cast<T *>(sum_out), static_cast<T *>(out), nullptr, rows, width, eps};
        with_shape<T>(width, [&](auto lanes, auto vectors) {
            constexpr int kTeam = decltype(lanes)::value, kBlock = kTeam <= kWave ? 256 : kTeam;
            const unsigned blocks = unsigned(blocks_of(rows, kTeam, kBlock, kForwardWaves));
            if (residual)
                layer_norm_kernel<T, P, kTeam, decltype(vectors)::value, true><<<blocks, kBlock, 0, as_stream(stream)>>>(p);
            else
                layer_norm_kernel<T, P, kTeam, decltype(vectors)::value, false><<<blocks, kBlock, 0, as_stream(stream)>>>(p);
        });
    };
    if (dtype == BDM_BF16)
        param_dtype == BDM_BF16 ? run(bf16_t{}, bf16_t{}) : run(bf16_t{}, float{});
    else
        param_dtype == BDM_BF16 ? run(float{}, bf16_t{}) : run(float{}, float{});
    return check_launch("layer_norm_kernel");
}

extern "C" size_t bdm_layer_norm_backward_workspace_size(int64_t rows, int32_t width) {
    if (rows <= 0 || width <= 0) return 0;
    if (width > kMaxWidth) return 0;
    return size_t(backward_parts(rows, width)) * 2 * size_t(width) * sizeof(float);
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
    const int64_t parts = backward_parts(rows, width);
    const auto run = [&](auto element, auto parameter) {
        using T = decltype(element);
        using P = decltype(parameter);
        const Rows<T> p{static_cast<const T *>(x), nullptr, static_cast<const T *>(grad_out), static_cast<const T *>(grad_sum),
                        weight, nullptr, nullptr, static_cast<T *>(grad_x), static_cast<float *>(workspace), rows, width, eps};
        with_shape<T>(width, [&](auto lanes, auto vectors) {
            constexpr int kTeam = decltype(lanes)::value, kBlock = backward_block(kTeam);
            if (grad_sum)
                layer_norm_backward_kernel<T, P, kTeam, decltype(vectors)::value, true><<<unsigned(parts), kBlock, 0, s>>>(p);
            else
                layer_norm_backward_kernel<T, P, kTeam, decltype(vectors)::value, false><<<unsigned(parts), kBlock, 0, s>>>(p);
        });
    };
    if (parts) {
        if (dtype == BDM_BF16)
            param_dtype == BDM_BF16 ? run(bf16_t{}, bf16_t{}) : run(bf16_t{}, float{});
        else
            param_dtype == BDM_BF16 ? run(float{}, bf16_t{}) : run(float{}, float{});
    }
    if (int rc = check_launch("layer_norm_backward_kernel")) return rc;
    if (!grad_weight && !grad_bias) return BDM_OK;
    layer_norm_param_kernel<<<unsigned((2 * width + kWave - 1) / kWave), kSumWaves * kWave, 0, s>>>(
        static_cast<const float *>(workspace), int(parts), width, grad_weight, grad_bias, param_dtype);
    return check_launch("layer_norm_param_kernel");
}
