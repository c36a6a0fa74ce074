// Beam search: the selection over beams and vocabulary, and the dense caches
// of several layers put in the order of the chosen parents.
//
// Selection.  With x the logits of beam k of a prompt, l = log sum exp x and
// s the beam's score, the candidate (k, t) has the total s + x_t - l; an ended
// beam offers one candidate, (eos, s).  The W best totals (divided by
// length^a where lengths are normalized) are wanted, ties to the lower
// k * V + t.  Within a beam the order of the totals is that of the logits, so
// one pass over the logits is enough: it keeps, for each part of a row, the
// maximum, the sum of exponentials and the W best logits (scan), and the
// parts of a prompt's rows are then joined (join).
//
// The scan holds its part in registers.  A lower bound of the W-th best value
// is near the W-th best of the lanes' own maxima, found by bisection with one
// ballot a bit; the few values at or above the bound go to LDS and are ranked
// there by counting.  Where ties or an unlucky layout put more there than it
// holds, the exact W-th value is found instead, and of those equal to it the
// first (equal logits, 64 prompts of 16 beams over 50,257: 85 us).
//
// What bounds it: for large calls in FP32 the read of the logits (64 prompts of
// 16 beams over 50,257, 206 MB: 42.3 us, the scan 32 to 35 of them, a part from
// the cache), in BF16 the vector instructions (40 us, the scan 33.6 of them).
// Both scans issue 14.5 M of these, 15 for each value of a lane, which is 24 us at
// four cycles each; of BF16's 40 us the candidates' compares, ballots and LDS
// atomics are 9, the exponentials 3 (copies without them).  For small calls it is
// the chain of a load, two selections and their barriers (4 beams over 192 tokens:
// 5.5 us).
//
// The exponentials and their sums are FP32 (each exponent relative to its
// part's maximum), everything behind them is FP64: candidates of different
// beams are compared by totals, which lie near each other.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "bdm_common.h"
#include "selection_ops.h"

namespace bdm {
namespace {

constexpr int kBeamMax = 64;       // beams in, and candidates out, per prompt
constexpr int kReorderTensors = 32;  // tensors of one reordering launch

// ------------------------------------------------------------------ a team's part of a row
// A team of WAVES waves holds NV vectors of VE values a lane, and one more: its shared memory.
template <int WAVES>
struct TeamShared {
    static constexpr int kRoom = 256 * WAVES;
    uint64_t list[kRoom];  // ordered value, then ~index: descending order is value, then lowest index
    float high[WAVES], sum[WAVES];
    uint32_t bound[WAVES], share[WAVES];
    int found[WAVES];
    int ties[WAVES][9];
    int count;
};

// How many of the team's values are above `than`, or at least that.
template <int WAVES, int E>
__device__ __forceinline__ int team_count(TeamShared<WAVES> &sh, const float (&x)[E], float than, bool level, int wave,
                                          int lane) {
    int mine = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) mine += popcount(__ballot(level ? x[e] >= than : x[e] > than));
    if constexpr (WAVES > 1) {
        if (lane == 0) sh.found[wave] = mine;
        __syncthreads();
        mine = 0;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) mine += sh.found[i];
        __syncthreads();
    }
    return mine;
}

// The exact `width` best of the team's values to sh.list, where more than it
// holds reach `least`: those above the width-th, then of those equal to it the
// ones of lowest index, which lie in the order of vectors, lanes, places in the
// vector, the odd ones behind all of these.  Where fewer than width
// are above `least` (equal logits, or a mask of the type's lowest value over
// most of the row) it is the width-th itself; else that is bisected.
template <int WAVES, int NV, int VE, typename Index>
__device__ __forceinline__ int team_ties(TeamShared<WAVES> &sh, const float (&x)[NV * VE + 1], Index index, float least,
                                         int width, int wave, int lane) {
    constexpr int E = NV * VE + 1, kGroups = NV + 1;
    static_assert(kGroups <= 9);
    float value = least;
    int above = team_count<WAVES, E>(sh, x, value, false, wave, lane);
    if (above >= width) {
        uint32_t found = 0;
#pragma unroll 1
        for (int bit = 31; bit >= 0; --bit) {
            // patterns beyond the infinities are NaN: no value reaches them
            const uint32_t next = found | (1u << bit);
            if (team_count<WAVES, E>(sh, x, unordered(next), true, wave, lane) >= width) found = next;
        }
        value = unordered(found);
        above = team_count<WAVES, E>(sh, x, value, false, wave, lane);
    }
    const bool odd = x[E - 1] == value;
    int ties[kGroups];
    ties[NV] = popcount(__ballot(odd));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        ties[i] = 0;
#pragma unroll
        for (int j = 0; j < VE; ++j) ties[i] += popcount(__ballot(x[i * VE + j] == value));
    }
    if (lane == 0) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g) sh.ties[wave][g] = ties[g];
    }
    if (wave == 0 && lane == 0) sh.count = 0;
    team_sync<WAVES>();
    auto take = [&](int e) {
        sh.list[atomicAdd(&sh.count, 1)] = uint64_t(ordered(x[e])) << 32 | uint32_t(~index(e));
    };
    int before = above;  // candidates ahead of the group's, in this wave's order
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        int at = before;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            at += w < wave ? sh.ties[w][g] : 0;
            before += sh.ties[w][g];
        }
        if (at >= width) continue;
        if (g == NV) {
            const uint64_t lanes = __ballot(odd);
            if (odd && at + popcount(lanes & ((1ull << lane) - 1)) < width) take(E - 1);
        } else {
#pragma unroll
            for (int j = 0; j < VE; ++j) at += popcount(__ballot(x[g * VE + j] == value) & ((1ull << lane) - 1));
#pragma unroll
            for (int j = 0; j < VE; ++j)
                if (x[g * VE + j] == value && at++ < width) take(g * VE + j);
        }
    }
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (x[e] > value) take(e);
    team_sync<WAVES>();
    return sh.count;
}

// Maximum, sum of exponentials and the `width` best of the team's values
// (load(x) gets them, index(e) is value e's index): sets high and sum in every lane, leaves the
// candidates in sh.list and returns how many there are.  Values of -inf are no
// candidates.  The few parts with too many ties load their values once more:
// kept alive for those, the values and their patterns took 108 registers of a
// lane with 33, and half the waves.
template <int WAVES, int NV, int VE, typename Load, typename Index>
__device__ __forceinline__ int team_scan(TeamShared<WAVES> &sh, Load load, Index index, int width, int wave, int lane,
                                         float &high, float &sum) {
    constexpr int E = NV * VE + 1;
    float x[E];
    load(x);
    float top = x[0];
#pragma unroll
    for (int e = 1; e < E; ++e) top = fmaxf(top, x[e]);
    const uint32_t mine = top > -INFINITY ? ordered(top) : 0u;
    uint32_t bound;
    high = wave_max(top);
    if constexpr (WAVES > 1) {
        // width lanes of one wave, or as many of all of them together, reach the bound
        const Bounds<2> bounds = nth_of_lanes<2>(mine, {{uint32_t(width), uint32_t(width + WAVES - 1) / WAVES}});
        if (lane == 0) {
            sh.high[wave] = high;
            sh.bound[wave] = bounds.at[0];
            sh.share[wave] = bounds.at[1];
        }
        if (threadIdx.x == 0) sh.count = 0;
        __syncthreads();
        bound = sh.share[0];
#pragma unroll
        for (int i = 0; i < WAVES; ++i) bound = min(bound, sh.share[i]);
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            high = fmaxf(high, sh.high[i]);
            bound = max(bound, sh.bound[i]);
        }
    } else {
        bound = nth_of_lanes<1>(mine, {{uint32_t(width)}}).at[0];
    }
    // the sum relative to the part's maximum; a part without a finite value has the sum 0, one with a NaN
    // or +inf (inf - inf) a NaN
    sum = 0.f;
    const float from = high > -INFINITY ? high : 0.f;
#pragma unroll
    for (int e = 0; e < E; ++e) sum += __expf(x[e] - from);
    sum = wave_sum(sum);
    if constexpr (WAVES > 1) {
        if (lane == 0) sh.sum[wave] = sum;
    }
    const float least = bound ? unordered(bound) : -FLT_MAX;
    if constexpr (WAVES > 1) {
        if (top >= least) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if (x[e] >= least) {
                    const int at = atomicAdd(&sh.count, 1);
                    if (at < TeamShared<WAVES>::kRoom)
                        sh.list[at] = uint64_t(ordered(x[e])) << 32 | uint32_t(~index(e));
                }
            }
        }
    } else {
        // without atomics, whose trips one row cannot hide (16 beams over 192 tokens: 9.6 us with them, 9.2 so; in
        // large calls other rows hide them, and waves without candidates pass this by: 40.6 us, 43 so)
        int found = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const bool reaches = x[e] >= least;
            const uint64_t lanes = __ballot(reaches);
            if (lanes) {
                const int at = found + popcount(lanes & ((1ull << lane) - 1));
                if (reaches && at < TeamShared<WAVES>::kRoom)
                    sh.list[at] = uint64_t(ordered(x[e])) << 32 | uint32_t(~index(e));
                found += popcount(lanes);
            }
        }
        if (lane == 0) sh.count = found;
    }
    team_sync<WAVES>();
    const int count = sh.count;
    if constexpr (WAVES > 1) {
        sum = 0.f;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) sum += sh.sum[i];
    }
    if (count <= TeamShared<WAVES>::kRoom) return count;
    team_sync<WAVES>();
    float again[E];
    load(again);
    return team_ties<WAVES, NV, VE>(sh, again, index, least, width, wave, lane);
}

// The team's candidates in descending order, the first `width` of them to out, 0 behind the last.
template <int WAVES>
__device__ __forceinline__ void team_rank(const TeamShared<WAVES> &sh, int count, int width, int wave, int lane,
                                          uint64_t *out) {
    for (int i = wave * kWave + lane; i < count; i += WAVES * kWave) {
        const uint64_t mine = sh.list[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < count; ++j) rank += sh.list[j] > mine;
        if (rank < width) out[rank] = mine;
    }
    for (int i = count + wave * kWave + lane; i < width; i += WAVES * kWave) out[i] = 0;
}

// NV vectors of a row's `vectors`, `step` apart from `begin` on, -inf where the row has none.  All are asked for at
// once, the last one in the place of those (a load under a condition of its own is waited for before the next).
template <typename T, int NV>
__device__ __forceinline__ void load_part(const T *x, int vectors, int begin, int step, float *out) {
    constexpr int VE = Vec<T>::kSize;
    u32x4 raw[NV];
    if (vectors > 0) {
#pragma unroll
        for (int i = 0; i < NV; ++i) raw[i] = reinterpret_cast<const AnyVector<T> *>(x + int64_t(min(begin + i * step, vectors - 1)) * VE)->bits;
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        Vec<T>::widen(raw[i], out + i * VE);
        const bool held = begin + i * step < vectors;
#pragma unroll
        for (int j = 0; j < VE; ++j) out[i * VE + j] = held ? out[i * VE + j] : -INFINITY;
    }
}

struct BeamParams {
    const void *logits;
    const float *scores;
    const uint8_t *finished;
    const int32_t *lengths;
    float *out_scores;
    int64_t *out_tokens, *out_parents;
    uint8_t *out_finished;
    int32_t *out_lengths;
    float2 *parts;    // [rows, splits] maximum and sum
    uint64_t *lists;  // [rows, splits, width] ordered logit, ~token; 0 behind the last
    int64_t batch_stride, beam_stride, eos;
    double penalty;
    int beams, vocab, width, splits;
};

// Whether a beam's logits count: it has not ended and its score is finite.
__device__ __forceinline__ bool beam_live(const BeamParams &p, int64_t row) {
    return !(p.finished && p.finished[row]) && isfinite(p.scores[row]);
}

// One part of one row.  The values behind the row's last whole vector are a
// tail that the first part takes one by one.  33 values a lane: with 17 the bounds and ranks
// weigh twice as much, with 65 of BF16 fewer waves hide each other's waits (64
// prompts of 16 beams over 50,257: 40.5 us, 42.8 with 65; over 131,072, whose
// parts are all full, 75 and 71).
// For wide selections a row's last part weighs: where it fills few of the lanes
// the waves without values have no share of the bound, one wave's own bound
// admits most of the part, and ranking them by counting takes its square (width
// 64, 16 beams, BF16: 25 us over 49,152 or 51,200 tokens, 36 to 54 over 50,257,
// whose last part fills 138 of 256 lanes; FP32 25, whose vectors are smaller).
template <typename T, int NV>
__global__ __launch_bounds__(256) void beam_scan_kernel(BeamParams p) {
    constexpr int VE = Vec<T>::kSize, E = NV * VE + 1;
    __shared__ TeamShared<4> sh;
    const uint32_t row = blockIdx.x / uint32_t(p.splits);
    const int split = int(blockIdx.x % uint32_t(p.splits));
    if (!beam_live(p, row)) return;
    const int wave = int(threadIdx.x) / kWave, lane = int(threadIdx.x) % kWave;
    const T *x = static_cast<const T *>(p.logits) + int64_t(row / uint32_t(p.beams)) * p.batch_stride +
                 int64_t(row % uint32_t(p.beams)) * p.beam_stride;
    const int vectors = p.vocab / VE;
    const int begin = split * NV * 256 + int(threadIdx.x);
    const int odd = vectors * VE + int(threadIdx.x);
    auto load = [&](float(&v)[E]) {
        load_part<T, NV>(x, vectors, begin, 256, v);
        v[E - 1] = split == 0 && odd < p.vocab ? to_f32(x[odd]) : -INFINITY;
    };
    auto index = [&](int e) { return uint32_t(e == E - 1 ? odd : (begin + e / VE * 256) * VE + e % VE); };
    float high, sum;
    const int count = team_scan<4, NV, VE>(sh, load, index, p.width, wave, lane, high, sum);
    const int64_t part = int64_t(row) * p.splits + split;
    if (threadIdx.x == 0) p.parts[part] = make_float2(high, sum);
    uint64_t *out = p.lists + part * p.width;
    team_rank<4>(sh, count, p.width, wave, lane, out);
}

// ------------------------------------------------------------------ joining a prompt's beams
template <int THREADS>
struct JoinShared {
    static constexpr int kRoom = THREADS, kWaves = THREADS / kWave;
    double log_sum[kBeamMax], norm[kBeamMax], score[kBeamMax];
    uint64_t key[kRoom];    // ordered compared value
    uint64_t place[kRoom];  // beam * vocab + token
    double total[kRoom];
    uint64_t chosen[kBeamMax];
    double chosen_total[kBeamMax];
    uint32_t bound[3][kWaves];
    uint2 found[2][kWaves];
    int list[kRoom];  // lists whose best reaches the bound
    int count, reaching;
};

// What a candidate has to reach: a compared value, and among those equal to it a place.
struct JoinBound {
    uint64_t key, place;
};

struct JoinCandidate {
    uint64_t key, place;  // ordered compared value, 0: there is none; beam * vocab + token
    double total;

    __device__ __forceinline__ uint32_t high() const { return uint32_t(key >> 32); }
    __device__ __forceinline__ bool reaches(const JoinBound &b) const {
        return key && (key > b.key || (key == b.key && place <= b.place));
    }
};

// The `width` best of the `count` > width candidates that sh holds, a thread
// each: the others are dropped.  The width-th one is found two bits at a time
// from the top, a step three ballots and a barrier: by the upper half of its
// key, among those equal in that by the lower half, and then by the place (of
// place_bits bits), as far as more than width are left.  Returns what the last
// one reaches.
template <int THREADS>
__device__ JoinBound join_cut(JoinShared<THREADS> &sh, int count, int width, int place_bits) {
    constexpr int kWaves = JoinShared<THREADS>::kWaves;
    const int thread = int(threadIdx.x), wave = thread / kWave, lane = thread % kWave;
    const bool held = wave * kWave < count;  // a wave without candidates only keeps the barriers
    const uint64_t key = thread < count ? sh.key[thread] : 0, place = thread < count ? sh.place[thread] : 0;
    const double total = thread < count ? sh.total[thread] : 0;
    int turn = 0;
    // how many threads satisfy each of three conditions, the waves' counts summed in a row of lanes
    auto counts = [&](bool a, bool b, bool c, int (&sum)[3]) {
        uint2 mine = make_uint2(0, 0);
        if (held) {
            mine.x = uint32_t(popcount(__ballot(a))) | uint32_t(popcount(__ballot(b))) << 16;
            mine.y = uint32_t(popcount(__ballot(c)));
        }
        if (lane == 0) sh.found[turn][wave] = mine;
        __syncthreads();
        uint2 all = sh.found[turn][lane % kWaves];
        if (lane >= kWaves) all = make_uint2(0, 0);
        const uint32_t pair = row_sum(all.x);
        sum[0] = int(pair & 0xffff), sum[1] = int(pair >> 16), sum[2] = int(row_sum(all.y));
        turn ^= 1;
    };
    // the largest bound that `want` of the candidates of `among` reach with `value`; narrows `among` to those equal to
    // it, and `want` to what is left to find between them.  True: no more than `want` of them reach it.
    bool among = thread < count, above = false;
    int want = width;
    auto narrow = [&](uint32_t value, int bits, uint32_t &bound) {
        bound = 0;
        int reach = INT32_MAX, sum[3];
        for (int shift = (bits - 1) & ~1; shift >= 0 && reach > want; shift -= 2) {
            const uint32_t one = 1u << shift, next = bound;
            counts(among && value >= next + one, among && value >= next + 2 * one, among && value >= next + 3 * one, sum);
#pragma unroll
            for (int s = 0; s < 3; ++s)
                if (sum[s] >= want) bound = next + uint32_t(s + 1) * one, reach = sum[s];
        }
        if (reach == want) {
            above |= among && value >= bound;
            return true;
        }
        counts(among && value > bound, false, false, sum);
        want -= sum[0];
        above |= among && value > bound;
        among = among && value == bound;
        return false;
    };
    uint32_t high = 0, low = 0;
    JoinBound bound{0, UINT64_MAX};
    if (!narrow(uint32_t(key >> 32), 32, high) && !narrow(uint32_t(key), 32, low)) {
        // lower places are the better ones
        uint32_t upper = 0, lower = 0;
        bool done = false;
        const uint32_t most = place_bits > 32 ? (1u << (place_bits - 32)) - 1 : 0;
        if (place_bits > 32) done = narrow(most - uint32_t(place >> 32), place_bits - 32, upper);
        if (!done) done = narrow(~uint32_t(place) << (32 - min(place_bits, 32)) >> (32 - min(place_bits, 32)),
                                 min(place_bits, 32), lower);
        above |= among && !done;  // one at most: places differ
        const uint32_t ones = place_bits >= 32 ? UINT32_MAX : (1u << place_bits) - 1;
        bound.place = uint64_t(most - upper) << 32 | (ones - lower);
    }
    bound.key = uint64_t(high) << 32 | low;
    if (thread == 0) sh.count = 0;
    __syncthreads();
    if (above) {
        const int at = atomicAdd(&sh.count, 1);
        sh.key[at] = key;
        sh.place[at] = place;
        sh.total[at] = total;
    }
    __syncthreads();
    return bound;
}

// A beam's score and the divisor of its candidates.
template <int THREADS>
__device__ __forceinline__ void join_beam(const BeamParams &p, JoinShared<THREADS> &sh, int64_t row, int beam) {
    sh.score[beam] = double(p.scores[row]);
    const bool ended = p.finished && p.finished[row];
    sh.norm[beam] = p.penalty != 0.0 ? pow(double(p.lengths[row] + (ended ? 0 : 1)), p.penalty) : 1.0;
}

// The `width` best of a prompt's candidates.  Each of its beams' `lists` lists
// (entry(list, rank): the list's rank-th value, descending, 0 behind the last;
// beam_of(list): its beam, which has the log_sum NaN where it has no totals) and
// each ended beam has candidates in descending order.  A lower bound of the
// width-th best one is found first, from all of them where a thread has few,
// else from the lists' first ones; those that reach it go to LDS.  Where they
// are more than a wave, the width best of what LDS took are cut out, and where
// they are more than LDS holds, the last of these is the next bound: each turn
// leaves fewer.  FEW: a thread always has few.  Called by the whole workgroup, behind a barrier that made
// log_sum, norm and score of every beam visible.
template <int THREADS, bool FEW, typename Entry, typename BeamOf>
__device__ void join_beams(const BeamParams &p, JoinShared<THREADS> &sh, int64_t prompt, int lists, Entry entry,
                           BeamOf beam_of) {
    constexpr int kRoom = JoinShared<THREADS>::kRoom, kWaves = THREADS / kWave;
    constexpr int kKept = 4;  // candidates that a thread keeps
    const int thread = int(threadIdx.x), wave = thread / kWave, lane = thread % kWave;
    // few of the best: one wave has them all; more: neighbours, as the lists of one beam, lie in different waves
    // (16 beams over 49,152 logits at width 32 17.7 us, one wave's bounds 20.1; at width 64 FP32 25.5 and 37.7, BF16 33.2
    // and 59.6; 64 beams at width 17 24.0 and 22.6)
    const bool wide = !FEW && p.width > 16;
    const int slot = wide ? lane * kWaves + wave : thread;
    const int ended = p.finished ? p.beams : 0, all = lists + ended;
    // the candidate of a list value, or an ended beam's own
    auto made = [&](int beam, uint64_t token, double total) {
        const double value = p.penalty != 0.0 ? total / sh.norm[beam] : total;
        return JoinCandidate{isfinite(value) ? ordered(value) : 0, uint64_t(beam) * uint32_t(p.vocab) + token, total};
    };
    auto listed = [&](int list, uint64_t item) {
        const int beam = beam_of(list);
        JoinCandidate c = made(beam, uint32_t(~uint32_t(item)),
                               sh.score[beam] + (double(unordered(uint32_t(item >> 32))) - sh.log_sum[beam]));
        if (!item) c.key = 0;
        return c;
    };
    auto candidate = [&](int list, int rank) {
        if (list < lists) return listed(list, entry(list, rank));
        const int beam = list - lists;
        JoinCandidate c = made(beam, uint64_t(p.eos), sh.score[beam]);
        if (rank || !p.finished[prompt * p.beams + beam]) c.key = 0;
        return c;
    };
    // the bound from each thread's best: width lanes of a wave reach it, or, for the wider ones, a quarter of that
    // in each of four waves, or as many in all of them together
    auto first_bound = [&](uint32_t best) {
        const uint32_t w = uint32_t(p.width);
        uint32_t bound = 0;
        if (thread == 0) sh.count = sh.reaching = 0;
        if (!wide) {
            const Bounds<1> part = nth_of_lanes<1>(best, {{w}});
            if (lane == 0) sh.bound[0][wave] = part.at[0];
            __syncthreads();
#pragma unroll
            for (int i = 0; i < kWaves; ++i) bound = max(bound, sh.bound[0][i]);
        } else {
            const Bounds<3> part = nth_of_lanes<3>(best, {{w, (w + 3) / 4, (w + kWaves - 1) / kWaves}});
            if (lane == 0) {
#pragma unroll
                for (int n = 0; n < 3; ++n) sh.bound[n][wave] = part.at[n];
            }
            __syncthreads();
            uint32_t every = UINT32_MAX;
#pragma unroll
            for (int i = 0; i < kWaves; i += 4) {
                uint32_t group = UINT32_MAX;
#pragma unroll
                for (int j = i; j < i + 4; ++j) {
                    bound = max(bound, sh.bound[0][j]);
                    group = min(group, sh.bound[1][j]);
                    every = min(every, sh.bound[2][j]);
                }
                bound = max(bound, group);
            }
            bound = max(bound, every);
        }
        return JoinBound{uint64_t(bound) << 32, UINT64_MAX};
    };
    auto take = [&](const JoinCandidate &c) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kRoom) {
            sh.key[at] = c.key;
            sh.place[at] = c.place;
            sh.total[at] = c.total;
        }
    };
    // cuts what LDS took down to a wave: by a bound from it, then exactly; whether there was more
    auto cut = [&](JoinBound &bound) {
        __syncthreads();
        const int reached = sh.count;
        if (reached <= kWave) return false;
        JoinCandidate mine{0, 0, 0};
        if (thread < min(reached, kRoom)) mine = JoinCandidate{sh.key[thread], sh.place[thread], sh.total[thread]};
        __syncthreads();
        const JoinBound next = first_bound(mine.high());
        if (next.key > bound.key) bound = next;
        if (mine.reaches(next)) take(mine);
        __syncthreads();
        const int left = sh.count;
        if (left > kWave) bound = join_cut(sh, left, p.width, 64 - __clzll(uint64_t(p.beams) * uint32_t(p.vocab)));
        if (reached <= kRoom) return false;
        __syncthreads();
        if (thread == 0) sh.count = sh.reaching = 0;
        __syncthreads();
        return true;
    };
    uint32_t best = 0;
    const int entries = lists * p.width;
    if (FEW || entries <= kKept * THREADS) {
        // the lists' first ones first, so that the best of many threads are high
        uint64_t item[kKept];
        JoinCandidate kept[kKept + 1];
#pragma unroll
        for (int n = 0; n < kKept; ++n) {
            if (n * THREADS >= entries) break;
            const uint32_t i = uint32_t(min(slot + n * THREADS, entries - 1));
            item[n] = entry(int(i % uint32_t(lists)), int(i / uint32_t(lists)));
        }
#pragma unroll
        for (int n = 0; n <= kKept; ++n) {
            kept[n] = JoinCandidate{0, 0, 0};
            if (n == kKept && slot < ended) kept[n] = candidate(lists + slot, 0);
            if (n < kKept && slot + n * THREADS < entries)
                kept[n] = listed(int(uint32_t(slot + n * THREADS) % uint32_t(lists)), item[n]);
            best = max(best, kept[n].high());
        }
        JoinBound bound = first_bound(best);
        do {
#pragma unroll
            for (int n = 0; n <= kKept; ++n)
                if (kept[n].reaches(bound)) take(kept[n]);
        } while (cut(bound));
    } else {
        const uint32_t ranks = min(uint32_t(p.width), uint32_t(THREADS + lists - 1) / uint32_t(lists));
        for (uint32_t i = slot; i < uint32_t(lists) * ranks; i += THREADS)
            best = max(best, candidate(int(i % uint32_t(lists)), int(i / uint32_t(lists))).high());
        JoinBound bound = first_bound(best);
        do {
            // the lists whose best reaches the bound's key and whose beam its place, whatever the best's own (entries
            // behind it with an equal key can have lower ones), then all of these (more than LDS holds: all of all)
            for (int list = thread; list < all; list += THREADS) {
                JoinCandidate c = candidate(list, 0);
                c.place = uint64_t(list < lists ? beam_of(list) : list - lists) * uint32_t(p.vocab);
                if (c.reaches(bound)) {
                    const int at = atomicAdd(&sh.reaching, 1);
                    if (at < kRoom) sh.list[at] = list;
                }
            }
            __syncthreads();
            const bool held = sh.reaching <= kRoom;
            const uint32_t most = uint32_t(held ? sh.reaching : all) * uint32_t(p.width);
            for (uint32_t i = thread; i < most; i += THREADS) {
                const uint32_t at = i / uint32_t(p.width);
                const JoinCandidate c = candidate(held ? sh.list[at] : int(at), int(i - at * uint32_t(p.width)));
                if (c.reaches(bound)) take(c);
            }
        } while (cut(bound));
    }
    const int count = sh.count;  // a wave of them at most
    for (int i = wave; i < count; i += kWaves) {
        const uint64_t key = sh.key[i], at = sh.place[i], k = sh.key[min(lane, count - 1)],
                       place_of = sh.place[min(lane, count - 1)];
        const int rank = popcount(__ballot(lane < count && (k > key || (k == key && place_of < at))));
        if (lane == 0 && rank < p.width) {
            sh.chosen[rank] = at;
            sh.chosen_total[rank] = sh.total[i];
        }
    }
    __syncthreads();
    if (thread == 0 && count < p.width) {
        // fewer candidates than places: the lowest places that are none of them, with the score -inf
        uint64_t next = 0;
        for (int i = count; i < p.width; ++next) {
            bool taken = false;
            for (int j = 0; j < count; ++j) taken |= sh.chosen[j] == next;
            if (!taken) {
                sh.chosen_total[i] = -INFINITY;
                sh.chosen[i++] = next;
            }
        }
    }
    __syncthreads();
    for (int i = thread; i < p.width; i += THREADS) {
        const uint64_t at = sh.chosen[i];
        const int64_t beam = int64_t(at / uint32_t(p.vocab)), token = int64_t(at % uint32_t(p.vocab));
        const int64_t row = prompt * p.beams + beam, out = prompt * p.width + i;
        const bool ended = p.finished && p.finished[row];
        p.out_scores[out] = float(sh.chosen_total[i]);
        p.out_tokens[out] = token;
        p.out_parents[out] = row;
        if (p.out_finished) p.out_finished[out] = ended || token == p.eos;
        if (p.out_lengths) p.out_lengths[out] = p.lengths[row] + (ended ? 0 : 1);
    }
}

// One workgroup a prompt: the parts of its rows joined.  It reads little, so the
// latency of its loads, FP64 logarithms and barriers bounds it: 8 prompts of 8
// beams in 13 parts 6.6 us, 64 of 16 beams in 7 parts 8.9.
constexpr int kJoinThreads = 1024;

__global__ __launch_bounds__(kJoinThreads) void beam_join_kernel(BeamParams p) {
    __shared__ JoinShared<kJoinThreads> sh;
    const int64_t prompt = blockIdx.x;
    const int wave = int(threadIdx.x) / kWave, lane = int(threadIdx.x) % kWave;
    const int last = int(threadIdx.x) - (kJoinThreads - kWave);  // the last wave: it has the fewest rows
    if (last >= 0 && last < p.beams) join_beam(p, sh, prompt * p.beams + last, last);
    for (int beam = wave; beam < p.beams; beam += kJoinThreads / kWave) {
        const int64_t row = prompt * p.beams + beam;
        if (!beam_live(p, row)) {  // no totals: its lists were not written
            if (lane == 0) sh.log_sum[beam] = NAN;
            continue;
        }
        const float2 *parts = p.parts + row * p.splits;
        float high = -INFINITY;
        for (int i = lane; i < p.splits; i += kWave) high = fmaxf(high, parts[i].x);
        high = wave_max(high);
        double sum = 0;
        for (int i = lane; i < p.splits; i += kWave) {
            const float2 part = parts[i];
            if (part.y != 0.f) sum += double(part.y) * exp(double(part.x) - double(high));
        }
#pragma unroll
        for (int d = kWave / 2; d; d >>= 1) sum += __shfl_xor(sum, d);
        if (lane == 0) sh.log_sum[beam] = double(high) + log(sum);
    }
    __syncthreads();
    const int rows = p.beams * p.splits;
    const uint64_t *lists = p.lists + prompt * rows * p.width;
    join_beams<kJoinThreads, false>(
        p, sh, prompt, rows,
        [&](int list, int rank) { return lists[uint32_t(list) * uint32_t(p.width) + uint32_t(rank)]; },
        [&](int list) { return int(uint32_t(list) / uint32_t(p.splits)); });
}

// Small vocabularies, one launch: one workgroup a prompt, a wave a row.  Bound
// by latency as the join is: 4 beams over 192 tokens 5.3 us.  A wave of its own
// for each of 16 beams, not two beams for each of 8: 12.1 -> 9.9 us over 2048.
constexpr int kRowBeams = 16, kRowWidth = 16;

template <typename T, int NV, int WAVES>
__global__ __launch_bounds__(WAVES *kWave) void beam_rows_kernel(BeamParams p) {
    constexpr int VE = Vec<T>::kSize, E = NV * VE + 1;
    __shared__ TeamShared<1> teams[WAVES];
    __shared__ JoinShared<WAVES * kWave> sh;
    __shared__ uint64_t lists[WAVES * kRowWidth];
    const int64_t prompt = blockIdx.x;
    const int wave = int(threadIdx.x) / kWave, lane = int(threadIdx.x) % kWave;
    TeamShared<1> &team = teams[wave];
    const int64_t row = prompt * p.beams + wave;
    if (wave < p.beams && beam_live(p, row)) {
        const T *x = static_cast<const T *>(p.logits) + prompt * p.batch_stride + wave * p.beam_stride;
        const int vectors = p.vocab / VE, odd = vectors * VE + lane;
        auto load = [&](float(&v)[E]) {
            load_part<T, NV>(x, vectors, lane, kWave, v);
            v[E - 1] = odd < p.vocab ? to_f32(x[odd]) : -INFINITY;
        };
        auto index = [&](int e) { return uint32_t(e == E - 1 ? odd : (e / VE * kWave + lane) * VE + e % VE); };
        float high, sum;
        const int count = team_scan<1, NV, VE>(team, load, index, p.width, 0, lane, high, sum);
        team_rank<1>(team, count, p.width, 0, lane, lists + wave * p.width);
        if (lane == 0) sh.log_sum[wave] = double(high) + log(double(sum));
    } else if (wave < p.beams && lane == 0) {
        sh.log_sum[wave] = NAN;  // no totals: its list is not written
    }
    if (int(threadIdx.x) < p.beams) join_beam(p, sh, prompt * p.beams + threadIdx.x, threadIdx.x);
    __syncthreads();
    join_beams<WAVES * kWave, true>(
        p, sh, prompt, p.beams,
        [&](int list, int rank) { return lists[uint32_t(list) * uint32_t(p.width) + uint32_t(rank)]; },
        [](int list) { return list; });
}

// How a call is cut: whole rows by a wave each (splits 0), or parts of `vectors` 16-byte vectors a thread.
struct BeamPlan {
    int vectors, splits;
};

// One launch for small vocabularies: 4 beams over 192 tokens 5.4 us, 8.8 as
// two; 8 over 2048 7.1 and 9.8; 16 over 2048 9.9 and 11.3 for one prompt, 10.5
// and 14.8 for 64.  Not for more than 16 of a row: a lane's best bounds them
// badly (64 of 16 beams over 2048: 106 us, 33 as two).
// The parts of a row are made smaller until there are 512 of them, two a
// compute unit: 8 prompts of 8 beams over 50,257 BF16 logits take 12.2 us so,
// 12.8 and 13.5 with 256 and 1024.
BeamPlan beam_plan(const bdm_beam_args &a) {
    const int ve = a.dtype == BDM_BF16 ? Vec<bf16_t>::kSize : Vec<float>::kSize;
    if (a.vocab <= 2048 && a.beams <= kRowBeams && a.width <= kRowWidth)
        return {a.vocab <= 512 ? 512 / (kWave * ve) : 2048 / (kWave * ve), 0};
    int vectors = 32 / ve;
    const int64_t rows = a.batch * a.beams;
    while (vectors > 8 / ve && rows * ((a.vocab + vectors * 256 * ve - 1) / (vectors * 256 * ve)) < 512)
        vectors /= 2;
    const int part = vectors * 256 * ve;
    return {vectors, (a.vocab + part - 1) / part};
}

// ------------------------------------------------------------------ reordering
struct ReorderTensor {
    char *data;
    int64_t row_bytes;
    unsigned first_block;  // of the tensor's workgroups of one prompt
};

struct ReorderParams {
    ReorderTensor tensors[kReorderTensors];
    const int64_t *parents;
    int count, beams;
    unsigned blocks;  // workgroups of one prompt
};

// data[i] <- data[parents[i]] within a prompt's beams, in place: a thread owns
// one vector column of all the prompt's rows, so it has every row that it
// moves in registers before it stores the first, and no other thread touches
// the column.  Rows that stay are neither read nor written.  Two beams of one
// parent read the same lines at the same time, from the caches.
// HBM's rate bounds it, and that wants long runs: a workgroup takes 512 vectors
// of each row (4 KiB of a row at a time reached 3.3 TB/s on 64 rows of 4 MiB,
// 8 KiB 5.2, past the caches, as the rows stream, 5.4; a large copy 4.8).
// More rows than registers hold as 16-byte vectors are moved in shorter ones: one
// prompt's rows of 4 MiB in four tensors, host's launch included, 4.1 TB/s for 16
// beams, 4.1 to 4.3 for 17 to 32 (8 bytes), 3.9 to 4.0 for 33 to 64 (4 bytes).
constexpr int kReorderRun = 512;  // vectors of a row

template <typename V, int K>
__global__ __launch_bounds__(256) void reorder_kernel(ReorderParams p) {
    constexpr int U = kReorderRun / 256;
    const int64_t prompt = blockIdx.x / p.blocks;
    const unsigned block = blockIdx.x % p.blocks;
    int which = 0;
    while (which + 1 < p.count && p.tensors[which + 1].first_block <= block) ++which;
    const ReorderTensor t = p.tensors[which];
    const int64_t column = int64_t(block - t.first_block) * kReorderRun + threadIdx.x, columns = t.row_bytes / int64_t(sizeof(V));
    const int64_t first = prompt * p.beams;
    V *base = reinterpret_cast<V *>(t.data + first * t.row_bytes);
    V held[K][U];
    int from[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        from[k] = k;
        if (k < p.beams) {
            const int64_t parent = p.parents[first + k] - first;
            from[k] = int(parent < 0 ? 0 : parent >= p.beams ? p.beams - 1 : parent);
            if (from[k] != k) {
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (column + u * 256 < columns)
                        held[k][u] = __builtin_nontemporal_load(base + from[k] * columns + column + u * 256);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (k < p.beams && from[k] != k) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (column + u * 256 < columns)
                    __builtin_nontemporal_store(held[k][u], base + k * columns + column + u * 256);
        }
    }
}

// `check`: nothing is launched, only what a launch would refuse.
template <typename V>
int launch_reorder(ReorderParams &p, int64_t batch, bool check, hipStream_t stream) {
    unsigned blocks = 0;
    for (int i = 0; i < p.count; ++i) {
        p.tensors[i].first_block = blocks;
        const int64_t need = (p.tensors[i].row_bytes / int64_t(sizeof(V)) + kReorderRun - 1) / kReorderRun;
        if (!grid_fits(need + blocks, 256)) return fail(BDM_ERR_UNSUPPORTED, "reorder_states: rows too long");
        blocks += unsigned(need);
    }
    if (blocks && !grid_fits(batch, 256 * int64_t(blocks))) return fail(BDM_ERR_UNSUPPORTED, "reorder_states: grid too large");
    if (blocks == 0 || check) return BDM_OK;
    p.blocks = blocks;
    const unsigned grid = unsigned(batch * blocks);
    constexpr int kMost = sizeof(V) == 16 ? 16 : sizeof(V) == 8 ? 32 : kBeamMax;  // rows that registers hold
    if (p.beams <= 4)
        reorder_kernel<V, 4><<<grid, 256, 0, stream>>>(p);
    else if (p.beams <= 8)
        reorder_kernel<V, 8><<<grid, 256, 0, stream>>>(p);
    else if (p.beams <= 16)
        reorder_kernel<V, 16><<<grid, 256, 0, stream>>>(p);
    else if (p.beams <= 32)
        reorder_kernel<V, kMost < 32 ? kMost : 32><<<grid, 256, 0, stream>>>(p);
    else
        reorder_kernel<V, kMost><<<grid, 256, 0, stream>>>(p);
    return check_launch("reorder_kernel");
}

template <typename T, int NV>
void launch_scan(const BeamParams &p, int64_t batch, hipStream_t stream) {
    beam_scan_kernel<T, NV><<<unsigned(batch * p.beams * p.splits), 256, 0, stream>>>(p);
}

int check_beam(const bdm_beam_args *a) {
    if (!a) return fail(BDM_ERR_INVALID, "beam_select: null args");
    if (a->batch < 0 || a->beams <= 0 || a->vocab <= 0 || a->width <= 0)
        return fail(BDM_ERR_INVALID, "beam_select: bad geometry");
    if (a->dtype != BDM_BF16 && a->dtype != BDM_F32) return fail(BDM_ERR_INVALID, "beam_select: logits dtype");
    if (a->vocab > 1 << 30) return fail(BDM_ERR_UNSUPPORTED, "beam_select: vocabulary of %d", a->vocab);
    if (a->beams > kBeamMax || a->width > kBeamMax)
        return fail(BDM_ERR_UNSUPPORTED, "beam_select: more than %d beams", kBeamMax);
    if (int64_t(a->width) > int64_t(a->beams) * a->vocab)
        return fail(BDM_ERR_INVALID, "beam_select: width %d exceeds the candidates", a->width);
    return BDM_OK;
}

}  // namespace
}  // namespace bdm

extern "C" size_t bdm_beam_select_workspace_size(const bdm_beam_args *a) {
    using namespace bdm;
    if (check_beam(a) != BDM_OK) return 0;
    const size_t parts = size_t(a->batch) * a->beams * beam_plan(*a).splits;
    return parts * (sizeof(float2) + size_t(a->width) * sizeof(uint64_t));
}

extern "C" int bdm_beam_select(const bdm_beam_args *a, void *workspace, size_t workspace_bytes, void *stream) {
    using namespace bdm;
    const int rc = check_beam(a);
    if (rc != BDM_OK) return rc;
    if (a->batch == 0) return BDM_OK;
    if (!a->logits || !a->scores || !a->out_scores || !a->out_tokens || !a->out_parents)
        return fail(BDM_ERR_INVALID, "beam_select: null pointer");
    if (a->finished && (a->eos < 0 || a->eos >= a->vocab))
        return fail(BDM_ERR_INVALID, "beam_select: ended beams need an eos token of the vocabulary");
    if ((a->length_penalty != 0.0 || a->out_lengths) && !a->lengths)
        return fail(BDM_ERR_INVALID, "beam_select: length normalization needs lengths");
    if (!(a->length_penalty - a->length_penalty == 0.0))
        return fail(BDM_ERR_INVALID, "beam_select: length_penalty must be finite");
    const size_t es = a->dtype == BDM_BF16 ? 2 : 4;
    if (!aligned(a->logits, es)) return fail(BDM_ERR_INVALID, "beam_select: logits not aligned to their type");
    const size_t need = bdm_beam_select_workspace_size(a);
    if (need && (!workspace || workspace_bytes < need)) return fail(BDM_ERR_WORKSPACE, "beam_select: workspace of %zu bytes", need);
    if (need && !aligned(workspace, 8)) return fail(BDM_ERR_INVALID, "beam_select: workspace must be 8-byte aligned");
    const BeamPlan plan = beam_plan(*a);
    if (!grid_fits(a->batch, std::max<int64_t>(kJoinThreads, 256 * int64_t(a->beams) * plan.splits)))
        return fail(BDM_ERR_UNSUPPORTED, "beam_select: grid too large");
    BeamParams p{};
    p.logits = a->logits;
    p.scores = a->scores;
    p.finished = a->finished;
    p.lengths = a->lengths;
    p.out_scores = a->out_scores;
    p.out_tokens = a->out_tokens;
    p.out_parents = a->out_parents;
    p.out_finished = a->out_finished;
    p.out_lengths = a->out_lengths;
    p.lists = static_cast<uint64_t *>(workspace);
    p.parts = reinterpret_cast<float2 *>(p.lists + size_t(a->batch) * a->beams * plan.splits * a->width);
    p.batch_stride = a->batch_stride;
    p.beam_stride = a->beam_stride;
    p.eos = a->eos;
    p.penalty = a->length_penalty;
    p.beams = a->beams;
    p.vocab = a->vocab;
    p.width = a->width;
    p.splits = plan.splits;
    hipStream_t s = as_stream(stream);
    const unsigned prompts = unsigned(a->batch);
    if (plan.splits == 0) {
        auto rows = [&](auto waves) {
            constexpr int W = decltype(waves)::value;
            if (a->dtype == BDM_BF16) {
                if (plan.vectors == 1)
                    beam_rows_kernel<bf16_t, 1, W><<<prompts, W * kWave, 0, s>>>(p);
                else
                    beam_rows_kernel<bf16_t, 4, W><<<prompts, W * kWave, 0, s>>>(p);
            } else {
                if (plan.vectors == 2)
                    beam_rows_kernel<float, 2, W><<<prompts, W * kWave, 0, s>>>(p);
                else
                    beam_rows_kernel<float, 8, W><<<prompts, W * kWave, 0, s>>>(p);
            }
        };
        if (a->beams <= 8)
            rows(std::integral_constant<int, 8>{});
        else
            rows(std::integral_constant<int, 16>{});
        return check_launch("beam_rows_kernel");
    }
    if (a->dtype == BDM_BF16) {
        if (plan.vectors == 4)
            launch_scan<bf16_t, 4>(p, a->batch, s);
        else if (plan.vectors == 2)
            launch_scan<bf16_t, 2>(p, a->batch, s);
        else
            launch_scan<bf16_t, 1>(p, a->batch, s);
    } else {
        if (plan.vectors == 8)
            launch_scan<float, 8>(p, a->batch, s);
        else if (plan.vectors == 4)
            launch_scan<float, 4>(p, a->batch, s);
        else
            launch_scan<float, 2>(p, a->batch, s);
    }
    const int scanned = check_launch("beam_scan_kernel");
    if (scanned != BDM_OK) return scanned;
    beam_join_kernel<<<prompts, kJoinThreads, 0, s>>>(p);
    return check_launch("beam_join_kernel");
}

extern "C" int bdm_reorder_states(void *const *states, const int64_t *row_bytes, int32_t count, const int64_t *parents,
                                  int64_t batch, int32_t beams, void *stream) {
    using namespace bdm;
    if (count < 0 || batch < 0 || beams <= 0) return fail(BDM_ERR_INVALID, "reorder_states: bad geometry");
    if (beams > kBeamMax) return fail(BDM_ERR_UNSUPPORTED, "reorder_states: more than %d beams", kBeamMax);
    if (count == 0 || batch == 0) return BDM_OK;
    if (!states || !row_bytes || !parents) return fail(BDM_ERR_INVALID, "reorder_states: null pointer");
    for (int i = 0; i < count; ++i) {
        if (row_bytes[i] < 0) return fail(BDM_ERR_INVALID, "reorder_states: bad geometry");
        if (row_bytes[i] && !states[i]) return fail(BDM_ERR_INVALID, "reorder_states: null pointer");
    }
    const int launches = (count + kReorderTensors - 1) / kReorderTensors;
    for (int turn = 0; turn < 2 * launches; ++turn) {  // every launch checked before the first one
        const int done = turn % launches * kReorderTensors;
        const bool check = turn < launches;
        ReorderParams p{};
        p.parents = parents;
        p.beams = beams;
        p.count = count - done < kReorderTensors ? count - done : kReorderTensors;
        uintptr_t bits = 0;  // what every base and row length is a multiple of
        for (int i = 0; i < p.count; ++i) {
            p.tensors[i].data = static_cast<char *>(states[done + i]);
            p.tensors[i].row_bytes = row_bytes[done + i];
            bits |= reinterpret_cast<uintptr_t>(states[done + i]) | uintptr_t(row_bytes[done + i]);
        }
        int rc;
        // a thread holds two vectors of each row in registers: 16 bytes of 16 rows are 128 of them, and beyond
        // that the vectors are shorter
        if (bits % 16 == 0 && beams <= 16)
            rc = launch_reorder<u32x4>(p, batch, check, as_stream(stream));
        else if (bits % 8 == 0 && beams <= 32)
            rc = launch_reorder<u32x2>(p, batch, check, as_stream(stream));
        else if (bits % 4 == 0)
            rc = launch_reorder<uint32_t>(p, batch, check, as_stream(stream));
        else if (bits % 2 == 0)
            rc = launch_reorder<uint16_t>(p, batch, check, as_stream(stream));
        else
            rc = launch_reorder<uint8_t>(p, batch, check, as_stream(stream));
        if (rc != BDM_OK) return rc;
    }
    return BDM_OK;
}
