// A paged bank cache: the banks of all sequences and layers in pages of one
// pool, shared between sequences until one of them writes.
//
// table[layer][sequence][bank] is the page of a bank (-1: the sequence holds
// none), references[page] counts its table entries and free_bits has a bit for
// each page with none.  A page is only ever an entry of one layer and bank.
// New pages are the lowest-numbered free ones, taken in the order of the
// requests, and reference counts are integers, so every result is the same
// from run to run whatever the order of the atomics.
//
//   resolve  before a decode step: the pages of the banks that the step reads,
//            and a page of its own for each bank that it writes and shares
//   fork     the table rows in the order of the parents
//   load     dense states into pages, equal banks shared with a base sequence
//   dense    pages into dense states
//   compact  the used pages moved to the front of the pool
#include "bdm_common.h"
#include "pages.h"

namespace bdm {
namespace {

constexpr int kMaxSequences = 512;
constexpr int kMaxSlots = 16;
constexpr int kBlock = 1024;  // the single workgroup of resolve, assign and compact's plan
constexpr int kBlockWaves = kBlock / kWave;

struct Pages {
    char *pool;
    int32_t *table, *references;
    unsigned long long *free_bits;
    int32_t *status;
    int64_t pages, page_bytes;
    int layers, sequences, banks;
};

// A table entry as a page of the pool, or -1.
__device__ __forceinline__ int checked(const Pages &p, int page) { return uint32_t(page) < uint64_t(p.pages) ? page : -1; }

// One reference less; the last one frees the page.
__device__ __forceinline__ void drop_reference(const Pages &p, int page) {
    if (atomicSub(p.references + page, 1) == 1) atomicOr(p.free_bits + page / 64, 1ull << (page % 64));
}

// Sum of the values of the lower lanes.
template <typename N>
__device__ __forceinline__ N wave_before(N value, int lane) {
    N sum = value;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) {
        const N other = __shfl_up(sum, d);
        if (lane >= d) sum += other;
    }
    return sum - value;
}

// Sum of the values of the lower threads of the workgroup; `all`: of all of them.
template <int THREADS, typename N>
__device__ __forceinline__ N block_before(N value, N *waves, N &all) {
    const int wave = int(threadIdx.x) / kWave, lane = int(threadIdx.x) % kWave;
    const N before = wave_before(value, lane);
    if (lane == kWave - 1) waves[wave] = before + value;
    __syncthreads();
    N lower = 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < THREADS / kWave; ++w) {
        const N sum = waves[w];
        if (w < wave) lower += sum;
        all += sum;
    }
    __syncthreads();
    return lower + before;
}

// x of the lane N below in the row of 16 (N < 0: above), `none` where there is no such lane.
template <int N>
__device__ __forceinline__ int in_row(int x, int none) {
    return __builtin_amdgcn_update_dpp(none, x, N > 0 ? 0x110 + N : 0x100 - N, 0xf, 0xf, false);
}

// The free bits of the lanes' pages.  Pages that were taken together are
// released together, so neighbouring lanes share words of the bits: a run of
// them within 16 lanes is one atomic, by its last lane (64 lanes on one word
// took 5 us).  Made by all lanes of a wave together.
struct FreeRun {
    int word;
    uint32_t low, high;
    bool last;

    FreeRun() = default;
    __device__ __forceinline__ FreeRun(bool free, int page) {
        word = free ? page / 64 : -1;
        low = free && !(page & 32) ? 1u << (page & 31) : 0;
        high = free && page & 32 ? 1u << (page & 31) : 0;
        // a lane's bits reach every lane above it in its row that has its word
        join<1>();
        join<2>();
        join<4>();
        join<8>();
        last = free && in_row<-1>(word, -2) != word;
    }

    template <int N>
    __device__ __forceinline__ void join() {
        const int other = in_row<N>(word, -2), more_low = in_row<N>(int(low), 0), more_high = in_row<N>(int(high), 0);
        if (other == word) {
            low |= uint32_t(more_low);
            high |= uint32_t(more_high);
        }
    }

    __device__ __forceinline__ void store(const Pages &p) const {
        if (last) atomicOr(p.free_bits + word, uint64_t(high) << 32 | low);
    }
};

// store(rank, lane, bit) for every set bit of the wave's words, in order;
// `before`: bits of the words ahead.  Few bits a word: each lane goes through its
// own; else the wave takes a word at a time, a lane a bit.
template <typename F>
__device__ __forceinline__ void each_bit(unsigned long long word, int before, F store) {
    const int lane = int(threadIdx.x) % kWave;
    if (!__any(__popcll(word) > 8)) {
        for (; word; word &= word - 1) store(before++, lane, __ffsll(word) - 1);
        return;
    }
    for (uint64_t left = __ballot(word != 0); left; left &= left - 1) {
        const int from = __ffsll(static_cast<unsigned long long>(left)) - 1;
        const uint64_t low = uint32_t(__builtin_amdgcn_readlane(int(uint32_t(word)), from));
        const uint64_t bits = low | uint64_t(uint32_t(__builtin_amdgcn_readlane(int(uint32_t(word >> 32)), from))) << 32;
        const int first = __builtin_amdgcn_readlane(before, from);
        if (bits >> lane & 1) store(first + __popcll(bits & ((1ull << lane) - 1)), from, lane);
    }
}

// `word` without its n lowest set bits (n of them at least).
__device__ __forceinline__ unsigned long long without_lowest(unsigned long long word, int n) {
    int low = 0;  // the largest number of low places with n set bits at most
#pragma unroll
    for (int step = 32; step; step >>= 1)
        if (__popcll(word & ((1ull << (low + step)) - 1)) <= n) low += step;
    // with 63 places taken the last one is left to look at
    if (low == 63 && __popcll(word) <= n) return 0;
    return word >> low << low;
}

// The free pages of THREADS words, found by their rank: a list of them, written
// a bit at a time, took 2 to 3 us of the kernels that take a few hundred.
template <int THREADS>
struct FreeTile {
    int waves[THREADS / kWave];
    int ahead[THREADS];  // free pages of the words below each
    unsigned long long words[THREADS];
};

// Fills the tile with the words from `base` on (`word` is the thread's), behind
// `below` free pages; those of the lowest `need` are free no more.  Returns how
// many there are.  Called by the whole workgroup, which has left the tile.
template <int THREADS>
__device__ __forceinline__ int fill_tile(const Pages &p, FreeTile<THREADS> &tile, int64_t base, unsigned long long word,
                                         int below, int need) {
    int all;
    const int ahead = below + block_before<THREADS>(int(__popcll(word)), tile.waves, all);
    tile.ahead[threadIdx.x] = ahead;
    tile.words[threadIdx.x] = word;
    if (word && ahead < need) {
        const int take = need - ahead;
        p.free_bits[base + threadIdx.x] = __popcll(word) <= take ? 0 : without_lowest(word, take);
    }
    __syncthreads();
    return all;
}

// The free page of a rank that the tile holds.
template <int THREADS>
__device__ __forceinline__ int free_page(const FreeTile<THREADS> &tile, int64_t base, int rank) {
    int low = 0;  // the last word with no more than `rank` pages below it
#pragma unroll
    for (int step = THREADS / 2; step; step >>= 1)
        if (tile.ahead[low + step] <= rank) low += step;
    const unsigned long long rest = without_lowest(tile.words[low], rank - tile.ahead[low]);
    return int((base + low) * 64 + __ffsll(rest) - 1);
}

__device__ __forceinline__ unsigned long long free_word(const Pages &p, int64_t at) {
    return at < (p.pages + 63) / 64 ? p.free_bits[at] : 0;
}

// ------------------------------------------------------------------ resolve
// One workgroup for a step's N * KW written and N * KR read banks: a written
// bank whose page other sequences hold gets a page of its own.  All of the
// sharers that write take new pages, so the page that they read from is stored
// to by none of them in this step; where none is left it is free for the next.
// A chain of dependent loads (bank, table, references, free bits), so it is
// latency that bounds it: 3.1 us for 64 written banks that nobody shares, 5.0
// for 32 that are shared, 6.1 for 512 of 64 sequences, 8.9 for 1,024 of 128.
// Beyond 1,024 it is another matter: eight rounds of requests, all of them whatever
// their number, do not fit the registers (932 bytes of scratch a lane): 98 us for
// 129 sequences of 8 banks, 101 for 256, 107 for 512.
template <int THREADS, int TILES>
__global__ __launch_bounds__(THREADS) void resolve_kernel(Pages p, int layer, const int64_t *write, const int64_t *read,
                                                          int rows, int kw, int kr, int32_t *source, int32_t *target,
                                                          int32_t *read_pages) {
    constexpr int kWaves = THREADS / kWave;
    __shared__ FreeTile<THREADS> tile;
    __shared__ int counts[TILES][kWaves];
    const int thread = int(threadIdx.x), wave = thread / kWave, lane = thread % kWave;
    int32_t *table = p.table + int64_t(layer) * p.sequences * p.banks;
    auto clamped = [&](int64_t index) { return int(index < 0 ? 0 : index >= p.banks ? p.banks - 1 : index); };
    const int writes = rows * kw, reads = rows * kr;
    unsigned long long word = free_word(p, threadIdx.x);  // in flight beside the chain below
    // each link of the chain (bank, page, references) for all requests at once and without a branch, behind which
    // the compiler would wait for it alone; a thread without a request repeats the last
    int page[TILES], before[TILES], bank[TILES], first[TILES], to[TILES];
    bool shared[TILES];
    int64_t asked[TILES][kMaxSlots], read_asked = 0;
    int read_page = -1, repeated = 0;
    // (a step without written, or read, banks looks at the other ones)
    const int64_t *writing = writes ? write : read, *reading = reads ? read : write;
    const int every = writes ? kw : kr, most = max(writes ? writes : reads, 1) - 1;
    const int read_every = reads ? kr : kw, read_at = min(thread, (reads ? reads : writes) - 1);
    read_asked = reading[read_at];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        const int at = min(t * THREADS + thread, most), row = at / every * every;
#pragma unroll
        for (int d = 0; d < kMaxSlots; ++d) asked[t][d] = writing[max(at - d, row)];
    }
    read_page = table[int64_t(read_at / read_every) * p.banks + clamped(read_asked)];
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        const int r = t * THREADS + thread, at = min(r, most);
        bank[t] = clamped(asked[t][0]);
        page[t] = table[int64_t(at / every) * p.banks + bank[t]];
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        const int r = t * THREADS + thread, slot = min(r, most) % every;
        first[t] = r;  // the first slot of the token with this bank
#pragma unroll
        for (int d = 1; d < kMaxSlots; ++d)
            if (d <= slot && clamped(asked[t][d]) == bank[t]) first[t] = r - d;
        page[t] = checked(p, page[t]);
        to[t] = p.references[max(page[t], 0)];
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        const int r = t * THREADS + thread;
        shared[t] = r < writes && page[t] >= 0 && first[t] == r && to[t] > 1;
        repeated |= r < writes && first[t] != r;
        const uint64_t mask = __ballot(shared[t]);
        before[t] = __popcll(mask & ((1ull << lane) - 1));
        if (lane == 0) counts[t][wave] = __popcll(mask);
        to[t] = shared[t] ? -1 : page[t];
        if (r < writes) source[r] = page[t];
    }
    if (thread < reads) read_pages[thread] = checked(p, read_page);
    for (int r = thread + THREADS; r < reads; r += THREADS)
        read_pages[r] = checked(p, table[int64_t(r / kr) * p.banks + clamped(read[r])]);
    repeated = __syncthreads_or(repeated);
    int need = 0;
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            if (w == wave) before[t] += need;
            need += counts[t][w];
        }
    }
    // the before[t]-th lowest free page for each
    int found = 0;
    for (int64_t base = 0; base * 64 < p.pages && found < need; base += THREADS) {
        if (base) {
            __syncthreads();
            word = free_word(p, base + thread);
        }
        const int all = fill_tile(p, tile, base, word, found, need);
#pragma unroll
        for (int t = 0; t < TILES; ++t)
            if (shared[t] && before[t] >= found && before[t] < found + all) to[t] = free_page(tile, base, before[t]);
        found += all;
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        const int r = t * THREADS + thread;
        if (shared[t]) {
            if (to[t] >= 0) {
                table[int64_t(r / kw) * p.banks + bank[t]] = to[t];
                p.references[to[t]] = 1;
                drop_reference(p, page[t]);
            } else {
                atomicOr(p.status, 1);
            }
        }
        if (r < writes && first[t] == r) target[r] = to[t];
    }
    if (!repeated) return;
    // slots that repeat a bank store where its first slot does
    __threadfence_block();
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TILES; ++t) {
        const int r = t * THREADS + thread;
        if (r < writes && first[t] != r) target[r] = target[first[t]];
    }
}

// ------------------------------------------------------------------ fork
struct ReleaseMask {
    uint64_t bits[kMaxSequences / 64];
};

// table[:, i] <- table[:, parents[i]].  A workgroup owns `span` banks of a
// layer and holds their column of every row that moves, is continued elsewhere
// or ends in LDS.  The references of a page change by what each of its rows
// gains or loses, (children of the row) - 1, at least -1: the count is zero
// behind the page's last row only, so whoever leaves zero frees the page.  A
// thread has kForkRows loads, then atomics, in flight: one at a time, each a
// trip to the L2, 64 rows took 13 us.
// The rows of a thread are neighbours, as beams of one prompt are, and where they
// share a page their changes are one (none for a prompt whose beams all share it).
// Latency bounds it too (parents, table, reference counts, free bits): one layer
// of 4 rows of 1,024 banks takes 4.3 us from a graph (5.1 by the profiler), of 64
// rows of 256 5.4 (6.9), 16 layers of 64 rows of 1,024 banks (8.4 MB of table in
// and out) 8.1 (10).
constexpr int kForkRows = 8;
constexpr int kForkInts = 8192;  // LDS of a column tile: sequences * span

// Rows [base, end) of the changed ones in one column, R of them at most: into the tile, and what they change of the
// references.  Each step for all rows at once: a load or atomic that the next row waited for was a trip of its own.
template <int R>
__device__ __forceinline__ void fork_rows(const Pages &p, const int32_t *column, const int *rows, const int *children,
                                          int *tile, int base, int end, int span, int mine, bool held) {
    int page[R], change[R], old[R];
#pragma unroll
    for (int u = 0; u < R; ++u) page[u] = column[int64_t(rows[max(min(base + u, end - 1), 0)]) * p.banks];
#pragma unroll
    for (int u = 0; u < R; ++u) {
        page[u] = checked(p, page[u]);
        change[u] = 0;
        if (base + u < end) {
            if (held && page[u] >= 0) change[u] = children[rows[base + u]] - 1;
            tile[(base + u) * span + mine] = page[u];
        }
    }
#pragma unroll
    for (int u = 1; u < R; ++u)
#pragma unroll
        for (int w = 0; w < u; ++w)
            if (page[w] == page[u]) {
                change[w] += change[u];
                change[u] = 0;
            }
#pragma unroll
    for (int u = 0; u < R; ++u) {
        old[u] = 0;
        if (change[u] < 0) old[u] = atomicAdd(p.references + page[u], change[u]);
    }
#pragma unroll
    for (int u = 0; u < R; ++u)
        if (change[u] > 0) atomicAdd(p.references + page[u], change[u]);
    bool free[R], any = false;
#pragma unroll
    for (int u = 0; u < R; ++u) {
        free[u] = change[u] < 0 && old[u] + change[u] == 0;
        any |= free[u];
    }
    if (!__any(any)) return;
    FreeRun runs[R];
#pragma unroll
    for (int u = 0; u < R; ++u) runs[u] = FreeRun(free[u], page[u]);
#pragma unroll
    for (int u = 0; u < R; ++u) runs[u].store(p);
}

__global__ __launch_bounds__(256) void fork_kernel(Pages p, const int64_t *parents, int count, ReleaseMask released,
                                                   int span) {
    constexpr int kParts = kMaxSequences / 256;
    __shared__ int tile[kForkInts];
    __shared__ int parent[kMaxSequences], children[kMaxSequences];
    __shared__ int rows[kMaxSequences], place[kMaxSequences], counts[kParts][4];
    const int tiles = (p.banks + span - 1) / span;
    const int layer = blockIdx.x / tiles;
    const int mine = int(threadIdx.x) % span, bank = blockIdx.x % tiles * span + mine;
    for (int i = threadIdx.x; i < p.sequences; i += 256) {
        int64_t from = released.bits[i / 64] >> (i % 64) & 1 ? -1 : i;
        if (parents && i < count) from = parents[i];
        parent[i] = int(from < 0 ? -1 : from >= p.sequences ? p.sequences - 1 : from);
        children[i] = 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.sequences; i += 256)
        if (parent[i] >= 0) atomicAdd(&children[parent[i]], 1);
    __syncthreads();
    // the rows that move, are continued elsewhere or end, in order
    const int wave = int(threadIdx.x) / kWave, lane = int(threadIdx.x) % kWave;
    uint64_t changes[kParts];
#pragma unroll
    for (int c = 0; c < kParts; ++c) {
        const int i = c * 256 + int(threadIdx.x);
        changes[c] = __ballot(i < p.sequences && (children[i] != 1 || parent[i] != i));
        if (lane == 0) counts[c][wave] = __popcll(changes[c]);
    }
    __syncthreads();
    int changed = 0;
#pragma unroll
    for (int c = 0; c < kParts; ++c) {
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int i = c * 256 + int(threadIdx.x);
            if (w == wave && changes[c] >> lane & 1) {
                place[i] = changed + __popcll(changes[c] & ((1ull << lane) - 1));
                rows[place[i]] = i;
            }
            changed += counts[c][w];
        }
    }
    if (!changed) return;
    __syncthreads();
    int32_t *column = p.table + int64_t(layer) * p.sequences * p.banks + min(bank, p.banks - 1);
    // every lane takes every turn: the lanes of a wave read each other's below
    const int threads = 256 / span, each = min((changed + threads - 1) / threads, kForkRows);
    for (int turn = 0; turn < changed; turn += threads * each) {
        const int base = turn + int(threadIdx.x) / span * each;
        if (each == 1)
            fork_rows<1>(p, column, rows, children, tile, base, changed, span, mine, bank < p.banks);
        else if (each == 2)
            fork_rows<2>(p, column, rows, children, tile, base, min(changed, base + each), span, mine, bank < p.banks);
        else if (each <= 4)
            fork_rows<4>(p, column, rows, children, tile, base, min(changed, base + each), span, mine, bank < p.banks);
        else
            fork_rows<kForkRows>(p, column, rows, children, tile, base, min(changed, base + each), span, mine, bank < p.banks);
    }
    __syncthreads();
    if (bank >= p.banks) return;
    for (int at = int(threadIdx.x) / span; at < changed; at += threads) {
        const int i = rows[at], from = parent[i];
        if (from != i) column[int64_t(i) * p.banks] = from < 0 ? -1 : tile[place[from] * span + mine];
    }
}

// ------------------------------------------------------------------ load and dense
struct Rows {
    int16_t at[kMaxSequences];  // sequence of each dense row
};

__device__ __forceinline__ bool bits_differ(uint4 a, uint4 b) {
    return ((a.x ^ b.x) | (a.y ^ b.y) | (a.z ^ b.z) | (a.w ^ b.w)) != 0;
}
__device__ __forceinline__ bool bits_differ(uint2 a, uint2 b) { return ((a.x ^ b.x) | (a.y ^ b.y)) != 0; }
__device__ __forceinline__ bool bits_differ(uint32_t a, uint32_t b) { return a != b; }

// Whether a dense bank differs from the base sequence's page of it; the old
// page is dropped, an equal base page taken.  A wave a bank; the books of a
// workgroup's banks are kept together, whose old pages mostly share a word of
// the free bits (one bank a workgroup, the atomics on these took 4 of 12 us).
// The read of the prompt and of the equal banks' pages bounds it: 8 prompts of
// 256 banks of 16 KiB, 40 % of them equal, 9.2 us; 2 of 1,024 banks of 1 KiB 3.5.
constexpr int kCompareWaves = 8;

template <typename V>
__global__ __launch_bounds__(kCompareWaves *kWave) void compare_kernel(Pages p, int layer, Rows rows, int base,
                                                                       uint32_t banks, const char *states,
                                                                       uint8_t *differs) {
    __shared__ int unequal[kCompareWaves];
    const int wave = int(threadIdx.x) / kWave, lane = int(threadIdx.x) % kWave;
    int32_t *table = p.table + int64_t(layer) * p.sequences * p.banks;
    const int count = int(p.page_bytes / int64_t(sizeof(V)));
    // what the books need of the workgroup's banks, in flight beside the comparison: lane i's is bank i's
    const uint32_t at = blockIdx.x * kCompareWaves + min(lane, kCompareWaves - 1);
    int32_t *entry = table;
    int old = -1, taken = -1;
    if (wave == 0) {
        const uint32_t kept = min(at, banks - 1), row = kept / uint32_t(p.banks), bank = kept - row * uint32_t(p.banks);
        entry = table + int64_t(rows.at[row]) * p.banks + bank;
        old = *entry;
        taken = table[int64_t(max(base, 0)) * p.banks + bank];
    }
    const uint32_t mine = blockIdx.x * kCompareWaves + wave;
    if (mine < banks) {
        const int shared = base < 0 ? -1 : checked(p, table[int64_t(base) * p.banks + mine % uint32_t(p.banks)]);
        const V *x = reinterpret_cast<const V *>(states + mine * p.page_bytes);
        const V *y = reinterpret_cast<const V *>(p.pool + max(shared, 0) * p.page_bytes);
        bool other = shared < 0;
        // a written bank shows it in its first vectors; the others of an equal one are loaded 8 at a time
        if (!other) other = __any(lane < count && bits_differ(x[min(lane, count - 1)], y[min(lane, count - 1)]));
        for (int i = kWave + lane; i - lane < count && !other; i += 8 * kWave) {
            V a[8], b[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int v = min(i + u * kWave, count - 1);
                a[u] = x[v];
                b[u] = y[v];
            }
            bool found = false;
#pragma unroll
            for (int u = 0; u < 8; ++u) found |= bits_differ(a[u], b[u]);
            other = __any(found);
        }
        if (lane == 0) unequal[wave] = other;
    }
    __syncthreads();
    if (wave) return;
    bool free = false;
    old = checked(p, old);
    if (lane < kCompareWaves && at < banks) {
        const bool other = unequal[lane];
        taken = other ? -1 : checked(p, taken);
        if (old != taken) {
            if (taken >= 0) atomicAdd(p.references + taken, 1);
            if (old >= 0) free = atomicSub(p.references + old, 1) == 1;
            *entry = taken;
        }
        differs[at] = uint8_t(other);
    }
    if (__any(free)) FreeRun(free, old).store(p);
}

// Pages for the banks that differ, in their order: target[i], or -1.  One
// workgroup, since a bank's page follows from how many differ before it: the
// latency of its counts and searches bounds it (2,048 banks 6.1 us; 32,768, 2,048
// a round, 53).
constexpr int kEach = 2;  // banks of a thread: 8 took 3 us more for 2,048

__global__ __launch_bounds__(kBlock) void assign_kernel(Pages p, int layer, Rows rows, int64_t banks,
                                                        const uint8_t *differs, int32_t *target) {
    __shared__ FreeTile<kBlock> tile;
    __shared__ int waves[kBlockWaves];
    __shared__ int16_t row_at[kMaxSequences];
    auto flags = [&](int64_t first) {
        if (first >= banks) return 0;
        const int two = *reinterpret_cast<const uint16_t *>(differs + first);  // the workspace has room behind the last
        return (two & 0xff ? 1 : 0) | (first + 1 < banks && two >> 8 ? 2 : 0);
    };
    unsigned long long word = free_word(p, threadIdx.x);  // in flight beside the count
    const int16_t row_of = rows.at[threadIdx.x % kMaxSequences];
    const int mine = flags(int64_t(threadIdx.x) * kEach);
    int count = __popc(mine);
    for (int64_t base = kBlock * kEach; base < banks; base += kBlock * kEach) count += __popc(flags(base + threadIdx.x * kEach));
    row_at[threadIdx.x % kMaxSequences] = row_of;
    int need;
    block_before<kBlock>(count, waves, need);
    if (!need) {
        for (int64_t i = threadIdx.x; i < banks; i += kBlock) target[i] = -1;
        return;
    }
    int32_t *table = p.table + int64_t(layer) * p.sequences * p.banks;
    // requests and free pages both ascend: a tile of one beside a tile of the other
    int64_t words = 0;
    int below = 0, held = fill_tile(p, tile, words, word, 0, need), done = 0;
    for (int64_t base = 0; base < banks; base += kBlock * kEach) {
        const int64_t first = base + threadIdx.x * kEach;
        const int f = base ? flags(first) : mine;
        int all;
        const int rank = done + block_before<kBlock>(int(__popc(f)), waves, all);
        int page[kEach] = {-1, -1};
        while (true) {
#pragma unroll
            for (int i = 0; i < kEach; ++i) {
                const int at = rank + (i ? f & 1 : 0);
                if (f >> i & 1 && at >= below && at < below + held) page[i] = free_page(tile, words, at);
            }
            if (done + all <= below + held || (words + kBlock) * 64 >= p.pages) break;
            below += held;
            words += kBlock;
            __syncthreads();
            held = fill_tile(p, tile, words, free_word(p, words + threadIdx.x), below, need);
        }
        done += all;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if (first + i >= banks) break;
            if (page[i] >= 0) {
                const uint32_t at = uint32_t(first + i), row = at / uint32_t(p.banks);
                p.references[page[i]] = 1;
                table[int64_t(row_at[row]) * p.banks + (at - row * uint32_t(p.banks))] = page[i];
            } else if (f >> i & 1) {
                atomicOr(p.status, 1);
            }
            target[first + i] = page[i];
        }
    }
}

template <typename V>
__device__ __forceinline__ void copy_page(const char *from, char *to, int64_t bytes) {
    const int count = int(bytes / int64_t(sizeof(V)));
    const V *x = reinterpret_cast<const V *>(from);
    V *y = reinterpret_cast<V *>(to);
    for (int i = threadIdx.x; i < count; i += blockDim.x) y[i] = x[i];
}

// A workgroup a bank, here and in dense_kernel: plain copies, bound by HBM or,
// as far as they fit, by the caches (2,048 banks of 16 KiB to dense states 10 us,
// 6.7 TB/s of reads and writes).
template <typename V>
__global__ __launch_bounds__(256) void store_kernel(Pages p, const char *states, const int32_t *target) {
    const int64_t at = blockIdx.x;
    const int page = target[at];
    if (page < 0) return;
    copy_page<V>(states + at * p.page_bytes, p.pool + page * p.page_bytes, p.page_bytes);
}

template <typename V>
__global__ __launch_bounds__(256) void dense_kernel(Pages p, int layer, Rows rows, char *states) {
    const int64_t at = blockIdx.x;
    const int row = int(blockIdx.x / uint32_t(p.banks)), bank = int(blockIdx.x % uint32_t(p.banks));
    const int page = checked(p, p.table[(int64_t(layer) * p.sequences + rows.at[row]) * p.banks + bank]);
    char *out = states + at * p.page_bytes;
    if (page >= 0) {
        copy_page<V>(p.pool + page * p.page_bytes, out, p.page_bytes);
    } else {
        const int count = int(p.page_bytes / int64_t(sizeof(V)));
        for (int i = threadIdx.x; i < count; i += blockDim.x) reinterpret_cast<V *>(out)[i] = V{};
    }
}

// ------------------------------------------------------------------ compact
struct CompactPlan {
    int32_t used, moves;
};

// With U pages in use, the k-th used page at or above U goes to the k-th free
// page below it: the lists of both, ascending, and where each moved page went.
// One workgroup goes through the words of the free bits; two block-wide sums,
// one behind the other, bound it (8 sequences of 1,024 banks 5.6 us).
__global__ __launch_bounds__(kBlock) void compact_plan_kernel(Pages p, CompactPlan *plan, int32_t *from, int32_t *to,
                                                              int32_t *moved) {
    __shared__ int counts[kBlockWaves];
    __shared__ uint64_t waves[kBlockWaves];
    const int64_t words = (p.pages + 63) / 64;
    // the pages of a word that lie below a border
    auto below = [](int64_t word, int64_t border) {
        const int64_t left = border - word * 64;
        return left >= 64 ? ~0ull : left <= 0 ? 0ull : (1ull << left) - 1;
    };
    const unsigned long long word = free_word(p, threadIdx.x);
    int mine = 0;
    for (int64_t at = threadIdx.x; at < words; at += kBlock)
        mine += __popcll(~(at < kBlock ? word : p.free_bits[at]) & below(at, p.pages));
    int used;
    block_before<kBlock>(mine, counts, used);
    uint64_t done = 0;  // movers in the upper half, holes in the lower
    for (int64_t base = 0; base < words; base += kBlock) {
        const int64_t at = base + threadIdx.x, first = base + threadIdx.x / kWave * kWave;
        const unsigned long long bits = base == 0 ? word : at < words ? p.free_bits[at] : 0;
        const unsigned long long low = below(at, used), hole = bits & low, mover = ~bits & below(at, p.pages) & ~low;
        uint64_t all;
        const uint64_t rank = done + block_before<kBlock>(uint64_t(__popcll(mover)) << 32 | uint32_t(__popcll(hole)), waves, all);
        done += all;
        each_bit(hole, int(uint32_t(rank)), [&](int k, int lane, int bit) { to[k] = int32_t((first + lane) * 64 + bit); });
        each_bit(mover, int(rank >> 32), [&](int k, int lane, int bit) { from[k] = int32_t((first + lane) * 64 + bit); });
        const unsigned long long left = below(at, p.pages) & ~low;
        if (at < words && left != bits) p.free_bits[at] = left;
    }
    __syncthreads();
    const int moves = int(done >> 32);
    for (int i = threadIdx.x; i < moves; i += kBlock) moved[from[i]] = to[i];
    if (threadIdx.x == 0) {
        plan->used = used;
        plan->moves = moves;
    }
}

// The moves, a workgroup a page, and the table's entries renamed beside them:
// both only touch pages and entries of their own.  The copies bound it (64
// sequences of banks of 16 KiB, 8 of them replaced: 8.3 us).
template <typename V>
__global__ __launch_bounds__(256) void compact_kernel(Pages p, const CompactPlan *plan, const int32_t *from,
                                                      const int32_t *to, const int32_t *moved) {
    const int moves = plan->moves, used = plan->used;
    if (!moves) return;
    for (int i = blockIdx.x; i < moves; i += gridDim.x) {
        const int a = from[i], b = to[i];
        copy_page<V>(p.pool + a * p.page_bytes, p.pool + b * p.page_bytes, p.page_bytes);
        if (threadIdx.x == 0) {
            p.references[b] = p.references[a];
            p.references[a] = 0;
        }
    }
    const int64_t entries = int64_t(p.layers) * p.sequences * p.banks;
    for (int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x; i < entries; i += int64_t(gridDim.x) * 256) {
        const int page = p.table[i];
        if (page >= used && page < p.pages) p.table[i] = moved[page];
    }
}

// ------------------------------------------------------------------ host side
int check_pages(const bdm_pages *p, Pages &out) {
    if (!p) return fail(BDM_ERR_INVALID, "pages: null args");
    if (p->pages <= 0 || p->layers <= 0 || p->sequences <= 0 || p->banks <= 0 || p->heads <= 0 || p->bank_size <= 0 ||
        p->head_width <= 0)
        return fail(BDM_ERR_INVALID, "pages: bad geometry");
    if (p->dtype != BDM_BF16 && p->dtype != BDM_F32) return fail(BDM_ERR_INVALID, "pages: dtype");
    if (p->sequences > kMaxSequences)
        return fail(BDM_ERR_UNSUPPORTED, "pages: more than %d sequences", kMaxSequences);
    if (p->pages > int64_t(INT32_MAX) - 64) return fail(BDM_ERR_UNSUPPORTED, "pages: more than 2^31 pages");
    const int64_t elements = int64_t(p->heads) * p->bank_size * p->head_width;
    if (elements > int64_t(INT32_MAX) / 4) return fail(BDM_ERR_UNSUPPORTED, "pages: page too large");
    if (int64_t(p->sequences) * p->banks > int64_t(INT32_MAX)) return fail(BDM_ERR_UNSUPPORTED, "pages: table too large");
    if (!p->pool || !p->table || !p->references || !p->free_bits || !p->status)
        return fail(BDM_ERR_INVALID, "pages: null pointer");
    if (!aligned(p->pool, 16) || !aligned(p->free_bits, 8))
        return fail(BDM_ERR_INVALID, "pages: the pool must be 16-byte aligned");
    out.pool = static_cast<char *>(p->pool);
    out.table = p->table;
    out.references = p->references;
    out.free_bits = reinterpret_cast<unsigned long long *>(p->free_bits);
    out.status = p->status;
    out.pages = p->pages;
    out.page_bytes = elements * (p->dtype == BDM_BF16 ? 2 : 4);
    out.layers = p->layers;
    out.sequences = p->sequences;
    out.banks = p->banks;
    return BDM_OK;
}

int check_rows(const bdm_pages *p, int layer, const int32_t *sequences, int count, Rows &rows) {
    if (layer < 0 || layer >= p->layers) return fail(BDM_ERR_INVALID, "pages: layer %d", layer);
    if (count < 0 || count > p->sequences || (count && !sequences))
        return fail(BDM_ERR_INVALID, "pages: bad sequence list");
    bool seen[kMaxSequences] = {};
    for (int i = 0; i < count; ++i) {
        if (sequences[i] < 0 || sequences[i] >= p->sequences || seen[sequences[i]])
            return fail(BDM_ERR_INVALID, "pages: sequence %d out of range or twice in one call", sequences[i]);
        seen[sequences[i]] = true;
        rows.at[i] = int16_t(sequences[i]);
    }
    return BDM_OK;
}

// The widest vector that every page of the pool and of `dense` starts on a multiple of.
template <typename F>
int with_vector(int64_t page_bytes, const void *dense, F run) {
    const uintptr_t bits = uintptr_t(page_bytes) | reinterpret_cast<uintptr_t>(dense);
    if (bits % 16 == 0) return run(uint4{});
    if (bits % 8 == 0) return run(uint2{});
    if (bits % 4 == 0) return run(uint32_t{});
    return run(uint16_t{});
}

// Threads that a page of `count` vectors keeps busy.
int page_threads(int64_t count) {
    const int64_t waves = (count + kWave - 1) / kWave;
    return int(waves >= 4 ? 256 : waves * kWave);
}

size_t round16(size_t n) { return (n + 15) / 16 * 16; }

}  // namespace
}  // namespace bdm

extern "C" int bdm_pages_fork(const bdm_pages *pages, const int64_t *parents, const int32_t *released, int32_t count,
                              void *stream) {
    using namespace bdm;
    Pages p;
    Rows rows;
    int rc = check_pages(pages, p);
    if (rc != BDM_OK) return rc;
    if (parents && released) return fail(BDM_ERR_INVALID, "pages_fork: parents or a list of released sequences");
    if (count < 0 || count > p.sequences) return fail(BDM_ERR_INVALID, "pages_fork: %d of %d sequences", count, p.sequences);
    if (count == 0) return BDM_OK;
    if (!parents) rc = check_rows(pages, 0, released, count, rows);
    if (rc != BDM_OK) return rc;
    ReleaseMask mask{};
    for (int i = 0; !parents && i < count; ++i) mask.bits[rows.at[i] / 64] |= 1ull << (rows.at[i] % 64);
    // 128 bytes of a table row where that fills the card (16 layers, 64 rows, 1,024 banks: 8.1 us, 11.3 with 64 bytes;
    // 8 layers 7.2 and 6.8), else 64 with more rows in flight at once (one layer, 256 banks: 5.4 us, 7.0 with 128)
    const bool wide = p.sequences * 32 <= kForkInts && int64_t(p.layers) * p.banks >= 256 * 32;
    const int span = wide ? 32 : kForkInts / kMaxSequences;
    const int64_t grid = int64_t(p.layers) * ((p.banks + span - 1) / span);
    if (!grid_fits(grid, 256)) return fail(BDM_ERR_UNSUPPORTED, "pages_fork: grid too large");
    fork_kernel<<<unsigned(grid), 256, 0, as_stream(stream)>>>(p, parents, count, mask, span);
    return check_launch("fork_kernel");
}

extern "C" size_t bdm_pages_load_workspace_size(const bdm_pages *pages, int32_t count) {
    using namespace bdm;
    if (!pages || count <= 0 || pages->banks <= 0) return 0;
    const size_t banks = size_t(count) * pages->banks;
    return round16(banks) + round16(banks * sizeof(int32_t));
}

extern "C" int bdm_pages_load(const bdm_pages *pages, int32_t layer, const int32_t *sequences, int32_t count,
                              int32_t base, const void *states, void *workspace, size_t workspace_bytes, void *stream) {
    using namespace bdm;
    Pages p;
    Rows rows;
    int rc = check_pages(pages, p);
    if (rc == BDM_OK) rc = check_rows(pages, layer, sequences, count, rows);
    if (rc != BDM_OK) return rc;
    if (base >= p.sequences) return fail(BDM_ERR_INVALID, "pages_load: base %d", base);
    for (int i = 0; i < count; ++i)
        if (sequences[i] == base) return fail(BDM_ERR_INVALID, "pages_load: the base is loaded itself");
    if (count == 0) return BDM_OK;
    const int64_t banks = int64_t(count) * p.banks;
    if (!states) return fail(BDM_ERR_INVALID, "pages_load: null pointer");
    if (!aligned(states, pages->dtype == BDM_BF16 ? 2 : 4))
        return fail(BDM_ERR_INVALID, "pages_load: states not aligned to their type");
    if (!workspace || workspace_bytes < bdm_pages_load_workspace_size(pages, count))
        return fail(BDM_ERR_WORKSPACE, "pages_load: workspace of %zu bytes", bdm_pages_load_workspace_size(pages, count));
    if (!aligned(workspace, 16)) return fail(BDM_ERR_INVALID, "pages_load: workspace must be 16-byte aligned");
    uint8_t *differs = static_cast<uint8_t *>(workspace);
    int32_t *target = reinterpret_cast<int32_t *>(differs + round16(banks));
    const char *data = static_cast<const char *>(states);
    hipStream_t s = as_stream(stream);
    return with_vector(p.page_bytes, states, [&](auto vector) {
        using V = decltype(vector);
        const int threads = page_threads(p.page_bytes / int64_t(sizeof(V)));
        if (!grid_fits(banks, threads)) return fail(BDM_ERR_UNSUPPORTED, "pages_load: grid too large");  // store_kernel's
        compare_kernel<V><<<unsigned((banks + kCompareWaves - 1) / kCompareWaves), kCompareWaves * kWave, 0, s>>>(
            p, layer, rows, base, uint32_t(banks), data, differs);
        int code = check_launch("compare_kernel");
        if (code != BDM_OK) return code;
        assign_kernel<<<1, kBlock, 0, s>>>(p, layer, rows, banks, differs, target);
        code = check_launch("assign_kernel");
        if (code != BDM_OK) return code;
        store_kernel<V><<<unsigned(banks), threads, 0, s>>>(p, data, target);
        return check_launch("store_kernel");
    });
}

extern "C" int bdm_pages_dense(const bdm_pages *pages, int32_t layer, const int32_t *sequences, int32_t count,
                               void *states, void *stream) {
    using namespace bdm;
    Pages p;
    Rows rows;
    int rc = check_pages(pages, p);
    if (rc == BDM_OK) rc = check_rows(pages, layer, sequences, count, rows);
    if (rc != BDM_OK) return rc;
    if (count == 0) return BDM_OK;
    if (!states) return fail(BDM_ERR_INVALID, "pages_dense: null pointer");
    if (!aligned(states, pages->dtype == BDM_BF16 ? 2 : 4))
        return fail(BDM_ERR_INVALID, "pages_dense: states not aligned to their type");
    const int64_t banks = int64_t(count) * p.banks;
    hipStream_t s = as_stream(stream);
    return with_vector(p.page_bytes, states, [&](auto vector) {
        using V = decltype(vector);
        const int threads = page_threads(p.page_bytes / int64_t(sizeof(V)));
        if (!grid_fits(banks, threads)) return fail(BDM_ERR_UNSUPPORTED, "pages_dense: grid too large");
        dense_kernel<V><<<unsigned(banks), threads, 0, s>>>(
            p, layer, rows, static_cast<char *>(states));
        return check_launch("dense_kernel");
    });
}

extern "C" size_t bdm_pages_compact_workspace_size(const bdm_pages *pages) {
    using namespace bdm;
    if (!pages || pages->pages <= 0) return 0;
    return 16 + 3 * round16(size_t(pages->pages) * sizeof(int32_t));
}

extern "C" int bdm_pages_compact(const bdm_pages *pages, void *workspace, size_t workspace_bytes, void *stream) {
    using namespace bdm;
    Pages p;
    const int rc = check_pages(pages, p);
    if (rc != BDM_OK) return rc;
    if (!workspace || workspace_bytes < bdm_pages_compact_workspace_size(pages))
        return fail(BDM_ERR_WORKSPACE, "pages_compact: workspace of %zu bytes", bdm_pages_compact_workspace_size(pages));
    if (!aligned(workspace, 16)) return fail(BDM_ERR_INVALID, "pages_compact: workspace must be 16-byte aligned");
    CompactPlan *plan = static_cast<CompactPlan *>(workspace);
    const size_t each = round16(size_t(p.pages) * sizeof(int32_t)) / sizeof(int32_t);
    int32_t *from = static_cast<int32_t *>(workspace) + 4, *to = from + each, *moved = to + each;
    hipStream_t s = as_stream(stream);
    compact_plan_kernel<<<1, kBlock, 0, s>>>(p, plan, from, to, moved);
    const int code = check_launch("compact_plan_kernel");
    if (code != BDM_OK) return code;
    return with_vector(p.page_bytes, nullptr, [&](auto vector) {
        using V = decltype(vector);
        compact_kernel<V><<<2048, 256, 0, s>>>(p, plan, from, to, moved);
        return check_launch("compact_kernel");
    });
}

extern "C" size_t bdm_pages_decode_workspace_size(const bdm_pages *pages, int32_t write_banks, int32_t read_banks) {
    if (!pages || pages->sequences <= 0 || write_banks < 0 || read_banks < 0) return 0;
    return size_t(pages->sequences) * (2 * size_t(write_banks) + read_banks) * sizeof(int32_t);
}

extern "C" int bdm_pages_decode(const bdm_pages *pages, int32_t layer, const bdm_decode_args *a, void *workspace,
                                size_t workspace_bytes, void *stream) {
    using namespace bdm;
    Pages p;
    const int rc = check_pages(pages, p);
    if (rc != BDM_OK) return rc;
    if (!a) return fail(BDM_ERR_INVALID, "pages_decode: null args");
    if (layer < 0 || layer >= p.layers) return fail(BDM_ERR_INVALID, "pages_decode: layer %d", layer);
    if (a->batch < 0 || a->batch > p.sequences || a->bank_count != p.banks || a->heads != pages->heads ||
        a->bank_size != pages->bank_size || a->head_width != pages->head_width || a->state_dtype != pages->dtype)
        return fail(BDM_ERR_INVALID, "pages_decode: the step's geometry is not the pages'");
    if (a->write_banks < 0 || a->read_banks < 0 || a->write_banks + a->read_banks == 0)
        return fail(BDM_ERR_INVALID, "pages_decode: bad geometry");
    if (a->write_banks > kMaxSlots || a->read_banks > kMaxSlots)
        return fail(BDM_ERR_UNSUPPORTED, "pages_decode: more than %d selected banks", kMaxSlots);
    if ((a->write_banks && !a->write_indices) || (a->read_banks && !a->read_indices))
        return fail(BDM_ERR_INVALID, "pages_decode: null pointer");
    if (a->batch == 0) return BDM_OK;
    const size_t need = bdm_pages_decode_workspace_size(pages, a->write_banks, a->read_banks);
    if (!workspace || workspace_bytes < need) return fail(BDM_ERR_WORKSPACE, "pages_decode: workspace of %zu bytes", need);
    if (!aligned(workspace, 16)) return fail(BDM_ERR_INVALID, "pages_decode: workspace must be 16-byte aligned");
    bdm_decode_args args = *a;
    args.state = p.pool;
    const int step = check_decode_pages(&args);  // before the tables change
    if (step != BDM_OK) return step;
    const int rows = int(a->batch), writes = rows * a->write_banks;
    int32_t *source = static_cast<int32_t *>(workspace), *target = source + writes, *read = target + writes;
    hipStream_t s = as_stream(stream);
    auto resolve = [&](auto kernel, int threads) {
        kernel<<<1, threads, 0, s>>>(p, layer, a->write_indices, a->read_indices, rows, a->write_banks, a->read_banks,
                                     source, target, read);
    };
    if (writes <= 256)
        resolve(resolve_kernel<256, 1>, 256);
    else if (writes <= 512)
        resolve(resolve_kernel<512, 1>, 512);
    else if (writes <= kBlock)
        resolve(resolve_kernel<kBlock, 1>, kBlock);
    else
        resolve(resolve_kernel<kBlock, kMaxSequences * kMaxSlots / kBlock>, kBlock);
    const int code = check_launch("resolve_kernel");
    if (code != BDM_OK) return code;
    return launch_decode_pages(args, PageTables{p.pool, source, target, read}, s);
}
