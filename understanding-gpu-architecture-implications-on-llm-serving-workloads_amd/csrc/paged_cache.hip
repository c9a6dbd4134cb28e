// What fills a paged key-value cache and what keeps it short, for gfx950 (MI355X): rotary embedding of a fused projection with its keys and values
// filed into their pages, and eviction by accumulated attention weight. Memory-bound, or bound by their chains of memory round trips.
#include <algorithm>

#include "paged.h"

namespace mi355 {

namespace pcache {
constexpr int THREADS = 256;
}

// Token (b, t) of a fused projection [q_heads | Hkv key heads | Hkv value heads] of 128: queries rotated in place, rotated keys and the values to row
// seq_lens[b] - new + t of the sequence; keep_keys: the rotated keys also where they were read. A thread owns 8 values of the
// lower half of a head and their 8 partners; 8 threads a head, 32 heads a workgroup. The arithmetic is that of rope_kernel (glue.hip). Bound by
// HBM for prompts (4 x 2048 rows, 60 % of them tokens, 32/8 heads: 29 us, 5.35 TB/s), by its chain of loads for a step (64 tokens: 3.2 us).
template <typename T>
__global__ __launch_bounds__(pcache::THREADS) void rope_paged_kernel(PagedKv kv, T* qkv, int S, Divisor by_s, int q_heads, int keep_keys, long x_batch,
                                                                     long x_row, const float* __restrict__ cos_t, const float* __restrict__ sin_t,
                                                                     const int* __restrict__ positions, long pos_batch, int n_pos) {
    using V8 = typename Elem<T>::v8;
    const int head = blockIdx.y * 32 + (threadIdx.x >> 3);
    if (head >= q_heads + 2 * kv.Hkv) return;
    const int b = divide(blockIdx.x, by_s), t = blockIdx.x - b * S;
    const int n_new = paged_new(kv, b, S);
    if (t >= n_new) return;
    const int i0 = (threadIdx.x & 7) * 8;
    T* xp = qkv + b * x_batch + t * x_row + (long)head * 128 + i0;
    V8 lo = *(const V8*)xp;
    V8 hi = *(const V8*)(xp + 64);
    const int place = positions[b * pos_batch + t];
    if (head < q_heads + kv.Hkv) {
        const int pos = min(max(place, 0), n_pos - 1);
        const float* cp = cos_t + (long)pos * 64 + i0;
        const float* sp = sin_t + (long)pos * 64 + i0;
        const float4v c0 = *(const float4v*)cp, c1 = *(const float4v*)(cp + 4);
        const float4v s0 = *(const float4v*)sp, s1 = *(const float4v*)(sp + 4);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float c = j < 4 ? c0[j] : c1[j - 4];
            const float sn = j < 4 ? s0[j] : s1[j - 4];
            const float x = (float)lo[j], y = (float)hi[j];
            lo[j] = (T)(x * c - y * sn);
            hi[j] = (T)(y * c + x * sn);
        }
        if (head < q_heads || keep_keys) {
            *(V8*)xp = lo;
            *(V8*)(xp + 64) = hi;
        }
        if (head < q_heads) return;
    }
    // a token in front of the cache's first row (a length smaller than its tokens) or behind its last, or of a page outside the pool, is not filed
    const int key = kv.seq_lens[b] - n_new + t;
    if (key < 0 || key >= kv.max_len) return;
    const int i = divide(key, kv.by_page);
    const int page = kv.table[(long)b * kv.table_stride + i];
    if ((uint32_t)page >= (uint32_t)kv.n_pages) return;
    const int slot = key - i * kv.page_size;
    char* op = kv.pages + (long)page * kv.page_bytes + (long)(head - q_heads) * kv.head_bytes + (uint32_t)slot * kv.row_bytes + 2 * i0;
    *(V8*)op = lo;
    *(V8*)(op + 128) = hi;
    if (head < q_heads + kv.Hkv && i0 == 0) {   // what eviction goes by
        const long at = ((long)page * kv.Hkv + (head - q_heads)) * kv.page_size + slot;
        if (kv.weights != nullptr) kv.weights[at] = 0.f;
        if (kv.key_positions != nullptr) kv.key_positions[at] = place;
    }
}

// ---- eviction ------------------------------------------------------------------------------------------------------------
//
// A kv head of a sequence longer than the budget keeps the `budget` keys of the largest rank: those whose position is within `recent` of its
// largest one first, then by weight, ties to the lowest slot. Kept keys behind the budget fill the slots of the dropped ones in
// front of it, in order: attention does not care how keys lie, their positions travel with them, and only as many rows move
// as are dropped (closing ranks would move most of the cache for one dropped key). A slot of a page outside the pool holds no key and takes none: one
// in front of the budget counts as kept, so that nothing moves there, one behind it is dropped before all keys.
namespace evict {
constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr int BINS = 2048, COPIES = 2;        // of the histogram, even and odd lanes' own
constexpr int kCompared = 64;                 // so many keys are compared with one another
constexpr int kMostChunks = 8;                // of 4 keys whose ranks stay in a thread's registers (32768 keys)
constexpr int kMovesHere = 256;               // up to this many moves are made by the selecting workgroup
constexpr int MOVES = 32;                     // of a workgroup of the moving kernel, 8 at a time side by side

// a weight as a whole number of the same order; the slots of pages outside the pool lowest (0), then NaN, then minus infinity
__device__ __forceinline__ uint32_t rank_of(float w) {
    const uint32_t u = __builtin_bit_cast(uint32_t, w == 0.f ? 0.f : w);   // (-0 is 0)
    if (w != w) return 1u;
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
// the lowest n bits, n cut to 0 .. 32
__device__ __forceinline__ uint32_t low_bits(int n) { return n >= 32 ? 0xffffffffu : n > 0 ? (1u << n) - 1u : 0u; }
constexpr uint32_t kRecent = 0xffffffffu;     // above plus infinity (0xff800000)
}  // namespace evict

struct Evict {
    int budget, recent, cap;   // cap: the most moves of a (sequence, kv head)
    int* counts;               // [pair]
    int* moves;                // [pair][2][cap]: slots of the dropped keys, of those that take them
    uint4* ranks;              // [pair][2][max_len / 4]: ranks and positions, where registers do not hold them
    int* lens_out;
    Divisor by_hkv;
};

namespace evict {

// sum of one value a thread over the threads in front of this one; `sums` is free again behind the caller's next barrier
__device__ __forceinline__ int block_before(int x, int (&sums)[WAVES], int& total) {
    const int incl = wave_inclusive_sum(x), wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if ((threadIdx.x & 63) == 63) sums[wave] = incl;
    __syncthreads();
    static_assert(WAVES == 16, "the waves' sums are summed up in a row of lanes");
    const int waves = row_inclusive_sum(sums[threadIdx.x & 15]);
    total = __builtin_amdgcn_readlane(waves, 15);
    return incl - x + (wave > 0 ? __builtin_amdgcn_readlane(waves, wave - 1) : 0);
}

// Moves n0, n0 + step, .. of those listed: 32 threads a move, four in flight each
template <typename List>
__device__ __forceinline__ void move_keys(const PagedKv& kv, int b, int hkv, List to, List from, int n0, int step, int count) {
    const int* table = kv.table + (long)b * kv.table_stride;
    const int l32 = threadIdx.x & 31;
    const long head = (long)(hkv + (l32 >> 4) * kv.Hkv) * kv.head_bytes + (l32 & 15) * 16;
    constexpr int N = 4;
    if (n0 >= count) return;
    int d[N], s[N], dp[N], sp[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int n = min(n0 + step * k, count - 1);   // (the last move again behind the end: not stored)
        d[k] = to[n];
        s[k] = from[n];
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const int di = divide(d[k], kv.by_page), si = divide(s[k], kv.by_page);
        dp[k] = table[di];
        sp[k] = table[si];
        d[k] -= di * kv.page_size;
        s[k] -= si * kv.page_size;
    }
    int4v row[N];
    int other[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        // a page outside the pool has no keys: nothing comes from it, nothing goes there
        if (n0 + step * k >= count || (uint32_t)dp[k] >= (uint32_t)kv.n_pages || (uint32_t)sp[k] >= (uint32_t)kv.n_pages) dp[k] = -1;
        if (dp[k] < 0) continue;
        row[k] = *(const int4v*)(kv.pages + (long)sp[k] * kv.page_bytes + head + (uint32_t)s[k] * kv.row_bytes);
        const long sa = ((long)sp[k] * kv.Hkv + hkv) * kv.page_size + s[k];
        if (l32 == 0) other[k] = __builtin_bit_cast(int, kv.weights[sa]);
        if (l32 == 16) other[k] = kv.key_positions[sa];
    }
#pragma unroll
    for (int k = 0; k < N; ++k) {
        if (dp[k] < 0) continue;
        *(int4v*)(kv.pages + (long)dp[k] * kv.page_bytes + head + (uint32_t)d[k] * kv.row_bytes) = row[k];
        const long da = ((long)dp[k] * kv.Hkv + hkv) * kv.page_size + d[k];
        if (l32 == 0) kv.weights[da] = __builtin_bit_cast(float, other[k]);
        if (l32 == 16) kv.key_positions[da] = other[k];
    }
}

}  // namespace evict

// One workgroup per (sequence, kv head). A thread owns 4 * chunks slots side by side (4 lie in one page and are read with one access), so that
// what has to be counted in the order of the slots is one sum over the threads. Their ranks stay in M chunks of registers or, M == 0, in
// the workspace, where only their thread reads them again. Bound by its chain of about a dozen steps, a memory round trip or a pass over
// the workgroup each (128 workgroups, 2176 keys each, 13.4 us with a copy of 2.5: length and loads 0.8 us, ranks and their range 0.8, the recent ones 0.6, histogram
// 1.0, comparing 0.8, what is kept 0.9, lists 0.3, 120 moves 2.3). In registers the keys' comparisons become bits of one word, which took 8192 keys from 24.4 to
// 21.3 us; adding the waves' sums up in a row of lanes, not by every thread, 0.5 us; three passes of 11, 11 and 10 bits instead of range and comparison 0.4.
// Through the workspace 4 x 8 kv heads of 65536 keys to 8192 take 224 us (the bytes 52).
template <int M>
__global__ __launch_bounds__(evict::THREADS) void evict_select_kernel(PagedKv kv, Evict a) {
    using namespace evict;
    __shared__ __attribute__((aligned(16))) int hist[BINS * COPIES];
    __shared__ int sums[4][WAVES];
    __shared__ int found[3], extent[2][WAVES], near, standing[kCompared];
    __shared__ int list[2][kMovesHere];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int b = divide(blockIdx.x, a.by_hkv), hkv = blockIdx.x - b * kv.Hkv;
    const int len = __builtin_amdgcn_readfirstlane(paged_len(kv, b));
    if (hkv == 0 && tid == 0) a.lens_out[b] = min(len, a.budget);
    if (len <= a.budget) {
        if (tid == 0) a.counts[blockIdx.x] = 0;
        return;
    }
    const int* table = kv.table + (long)b * kv.table_stride;
    const int chunks = (len + 4 * THREADS - 1) / (4 * THREADS);   // <= M, where that is given
    const int j0 = tid * 4 * chunks;   // (up to 4096 behind the last key)
    constexpr int REGS = M > 0 ? M : 1;
    uint4 rank[REGS], position[REGS];
    uint4* kept_ranks = a.ranks + (long)blockIdx.x * 2 * ((kv.max_len + 3) / 4 + THREADS);
    uint4* kept_positions = kept_ranks + (kv.max_len + 3) / 4 + THREADS;
#pragma unroll
    for (int i = 0; i < BINS * COPIES / THREADS; ++i) hist[i * THREADS + tid] = 0;

    // Positions and the weights' ranks; the largest position. `there`: a bit for each key of a chunk that the sequence has, in a page of the pool
    const auto there_of = [&](int j, int page) -> uint32_t {
        return (uint32_t)page < (uint32_t)kv.n_pages && (uint32_t)j < (uint32_t)len ? (len - j >= 4 ? 15u : (1u << (len - j)) - 1u) : 0u;
    };
    const auto get = [&](const uint4& v, int e) { return e == 0 ? v.x : e == 1 ? v.y : e == 2 ? v.z : v.w; };
    int newest = INT32_MIN;
    uint32_t lowest = 0xffffffffu, highest = 0;   // ranks
    const auto load = [&](int c, uint4& r, uint4& p) {
        const int j = min(j0 + 4 * c, kv.max_len - 4), i = divide(j, kv.by_page);
        const int page = table[i];
        const uint32_t there = c < chunks && j == j0 + 4 * c ? there_of(j, page) : 0u;
        const long at = ((long)(there ? page : 0) * kv.Hkv + hkv) * kv.page_size + (j - i * kv.page_size);
        p = *(const uint4*)(kv.key_positions + at);
        const float4v w = *(const float4v*)(kv.weights + at);
        uint32_t x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            x[e] = (there >> e) & 1 ? rank_of(w[e]) : 0u;
            newest = (there >> e) & 1 ? max(newest, (int)get(p, e)) : newest;
            const bool has = c < chunks && j0 + 4 * c + e < len;   // (in a page of the pool or not)
            lowest = has ? min(lowest, x[e]) : lowest;
            highest = max(highest, x[e]);
            if (M > 0) x[e] = has ? x[e] : kRecent;   // (what the sequence does not have is outside every range)
        }
        r = uint4{x[0], x[1], x[2], x[3]};
        return there;
    };
    uint32_t present = 0;   // of the chunks in registers, 4 bits each
    if constexpr (M > 0) {
#pragma unroll
        for (int c = 0; c < M; ++c) present |= load(c, rank[c], position[c]) << (4 * c);
    } else {
        for (int c = 0; c < chunks; ++c) {
            uint4 r, p;
            load(c, r, p);
            kept_ranks[c * THREADS + tid] = r;
            kept_positions[c * THREADS + tid] = p;
        }
    }
    newest = wave_max(newest);
    const int below = wave_max((int)(~lowest ^ 0x80000000u)), above = wave_max((int)(highest ^ 0x80000000u));
    if (lane == 0) sums[0][wave] = newest, extent[0][wave] = below, extent[1][wave] = above;
    if (tid == 0) near = 0;
    if (tid < kCompared) standing[tid] = 0;
    __syncthreads();
    newest = row_max(sums[0][lane & 15]);
    const int bottom = row_max(extent[0][lane & 15]), top = row_max(extent[1][lane & 15]);
    const long old = (long)newest - a.recent;   // positions up to here are not recent
    int recent = 0;
    // (`none`: slots in front of the budget that hold no key)
    const auto mark = [&](uint32_t there, uint32_t none, uint4& r, const uint4& p) {
        uint32_t x[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const bool is = (there >> e) & 1 ? (int)get(p, e) > old : (none >> e) & 1;
            x[e] = is ? kRecent : get(r, e);
            recent += is;
        }
        r = uint4{x[0], x[1], x[2], x[3]};
    };
    // f(key, rank) for this thread's keys in order (from the workspace)
    const auto each = [&](auto&& f) {
        for (int c = 0; c < chunks && j0 + 4 * c < len; ++c) {
            const uint4 r = kept_ranks[c * THREADS + tid];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (j0 + 4 * c + e < len) f(j0 + 4 * c + e, get(r, e));
        }
    };
    // a bit for each of them (in registers) of which f(rank) holds
    const auto bits_of = [&](auto&& f) {
        uint32_t m = 0;
#pragma unroll
        for (int c = 0; c < REGS; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) m |= f(get(rank[c], e)) ? 1u << (4 * c + e) : 0u;
        return m;
    };
    if constexpr (M > 0) {
#pragma unroll
        for (int c = 0; c < M; ++c) mark((present >> (4 * c)) & 15, 0, rank[c], position[c]);
        const uint32_t none = low_bits(min(len - j0, 4 * chunks)) & low_bits(a.budget - j0) & ~present;
        if (__builtin_amdgcn_ballot_w64(none != 0) != 0) {
#pragma unroll
            for (int c = 0; c < M; ++c) mark(0, (none >> (4 * c)) & 15, rank[c], position[c]);
        }
    } else {
        for (int c = 0; c < chunks; ++c) {
            const int j = j0 + 4 * c;
            if (j >= len) break;
            uint4 r = kept_ranks[c * THREADS + tid];
            const int page = table[divide(j, kv.by_page)];
            const uint32_t there = there_of(j, page);
            const uint4 at = kept_positions[c * THREADS + tid];
            mark(there, 0, r, at);
            if (there != 15u) mark(0, low_bits(min(len, a.budget) - j) & ~there, r, at);
            kept_ranks[c * THREADS + tid] = r;
        }
    }
    int all_recent;
    block_before(recent, sums[1], all_recent);

    // The rank of the last kept key, and how many keys of it are kept (`want`, the first ones). The recent ones are counted above (in the
    // histogram they would all fall on one counter); of the others the want-th largest: a histogram of their range in 2048 equal bins (of the ranks'
    // upper 11 bits a few are all that occur, and their counters are waited for), and of its bin, where that holds more than 64 keys, the same
    // again; 64 keys are compared with one another.
    uint32_t last = kRecent;
    int want = a.budget;
    if (all_recent < a.budget) {
        want -= all_recent;
        uint32_t base = ~((uint32_t)bottom ^ 0x80000000u), range = ((uint32_t)top ^ 0x80000000u) - base;   // ranks base .. base + range
        int shift = max(21 - __builtin_clz(range | 1), 0);
        for (int pass = 0;; ++pass) {
            const auto count_one = [&](uint32_t r) {
                if (r - base <= range) atomicAdd(&hist[((r - base) >> shift) * COPIES + (lane & (COPIES - 1))], 1);
            };
            if constexpr (M > 0) {
#pragma unroll
                for (int c = 0; c < M; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) count_one(get(rank[c], e));
            } else {
                each([&](int, uint32_t r) { count_one(r); });
            }
            __syncthreads();
            // thread t: the bins 2047 - 2t and 2046 - 2t; sums from the top
            int4v* at = (int4v*)(hist + (BINS - 2 - 2 * tid) * COPIES);
            const int4v both = *at;
            *at = int4v{0, 0, 0, 0};
            const int h0 = both[2] + both[3], h1 = both[0] + both[1];
            int unused;
            const int before = block_before(h0 + h1, sums[2 + (pass & 1)], unused);
            if (before < want && want <= before + h0) found[0] = BINS - 1 - 2 * tid, found[1] = want - before, found[2] = h0;
            else if (before + h0 < want && want <= before + h0 + h1) found[0] = BINS - 2 - 2 * tid, found[1] = want - before - h0, found[2] = h1;
            __syncthreads();
            base += (uint32_t)found[0] << shift;
            want = found[1];
            const int count = found[2];
            last = base;
            if (shift == 0) break;
            range = (1u << shift) - 1;
            if (count <= kCompared) {
                if constexpr (M > 0) {
                    if (bits_of([&](uint32_t r) { return r - base <= range; }) != 0) {
#pragma unroll
                        for (int c = 0; c < M; ++c)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                if (get(rank[c], e) - base <= range) list[0][atomicAdd(&near, 1)] = (int)get(rank[c], e);
                    }
                } else {
                    each([&](int, uint32_t r) {
                        if (r - base <= range) list[0][atomicAdd(&near, 1)] = (int)r;
                    });
                }
                __syncthreads();
                // each wave compares them all with four of them: how many are larger, how many equal (16 bits each)
                const uint32_t mine = (uint32_t)list[0][min(lane, count - 1)];
                int place = 0;
#pragma unroll
                for (int i = 0; i < kCompared / WAVES; ++i) {
                    const int at = wave * (kCompared / WAVES) + i;
                    const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)mine, at);
                    place += at >= count ? 0 : other > mine ? 1 : other == mine ? 1 << 16 : 0;
                }
                if (place != 0) atomicAdd(&standing[lane], place);
                __syncthreads();
                place = standing[lane];
                const int larger = place & 0xffff, equal = place >> 16;
                // (the same of all lanes that hold it, and of all waves)
                const int who = __builtin_ctzll(__builtin_amdgcn_ballot_w64(larger < want && want <= larger + equal));
                last = (uint32_t)__builtin_amdgcn_readlane((int)mine, who);
                want -= __builtin_amdgcn_readlane(larger, who);
                break;
            }
            shift = max(shift - 11, 0);
        }
    }
    // Kept are the larger ranks and the first `want` of this one; of the slots in front of the budget those that are not kept are holes, and kept keys
    // behind it move. `mine`: how many of this thread's own of this rank are kept.
    const bool here = a.cap <= kMovesHere;
    int* to = a.moves + (long)blockIdx.x * 2 * a.cap;
    int* from = to + a.cap;
    int total, unused;
    if constexpr (M > 0) {
        const uint32_t have = low_bits(min(len - j0, 4 * chunks)), front = low_bits(a.budget - j0);
        const uint32_t equal = bits_of([&](uint32_t r) { return r == last; }) & have;
        uint32_t keep = bits_of([&](uint32_t r) { return r > last; }) & have;
        int mine = want - block_before(__builtin_popcount(equal), sums[0], unused);
        for (uint32_t left = equal; left != 0 && mine > 0; left &= left - 1, --mine) keep |= left & -left;
        uint32_t holes = ~keep & have & front, movers = keep & ~front;
        // at most 16384 of each: one sum for both
        const int before = block_before(__builtin_popcount(holes) | __builtin_popcount(movers) << 16, sums[1], total);
        total &= 0xffff;
        int* hole = (here ? list[0] : to) + (before & 0xffff);
        int* mover = (here ? list[1] : from) + (before >> 16);
        for (; holes != 0; holes &= holes - 1) *hole++ = j0 + __builtin_ctz(holes);
        for (; movers != 0; movers &= movers - 1) *mover++ = j0 + __builtin_ctz(movers);
    } else {
        int ties = 0;
        each([&](int, uint32_t r) { ties += r == last; });
        const int tie0 = block_before(ties, sums[0], unused);
        const auto keeps = [&](uint32_t r, int& tie) {
            const bool keep = r > last || (r == last && tie < want);
            tie += r == last;
            return keep;
        };
        int holes = 0, movers = 0, tie = tie0;
        each([&](int j, uint32_t r) {
            const bool keep = keeps(r, tie);
            holes += !keep && j < a.budget;
            movers += keep && j >= a.budget;
        });
        int hole = block_before(holes, sums[1], total), mover = block_before(movers, sums[2], unused);
        tie = tie0;
        each([&](int j, uint32_t r) {
            const bool keep = keeps(r, tie);
            if (!keep && j < a.budget) (here ? list[0] : to)[hole++] = j;
            if (keep && j >= a.budget) (here ? list[1] : from)[mover++] = j;
        });
    }
    if (tid == 0) a.counts[blockIdx.x] = here ? 0 : total;
    if (!here) return;
    __syncthreads();
    for (int n = 0; n < total; n += 4 * THREADS / 32) move_keys(kv, b, hkv, list[0], list[1], n + (tid >> 5), THREADS / 32, total);
}

// Grid (moves / 32, pairs), for more moves than the selecting workgroup makes (32 pairs, ~1500 moves each: 8.9 us; with one move in flight a thread 16)
__global__ __launch_bounds__(256) void evict_move_kernel(PagedKv kv, Evict a) {
    const int count = a.counts[blockIdx.y];
    const int b = divide(blockIdx.y, a.by_hkv), hkv = blockIdx.y - b * kv.Hkv;
    const int* to = a.moves + (long)blockIdx.y * 2 * a.cap;
    evict::move_keys(kv, b, hkv, to, to + a.cap, blockIdx.x * evict::MOVES + (threadIdx.x >> 5), 8, count);
}

hipError_t rope_paged_dispatch(const mi355_paged_kv& c, void* qkv, int S, int q_heads, int keep_keys, long x_batch, long x_row, const float* cos_t,
                               const float* sin_t, const int* positions, long pos_batch, int n_pos, hipStream_t stream) {
    const PagedKv kv = paged_from(c);
    const dim3 grid((unsigned)(kv.B * S), (unsigned)((q_heads + 2 * kv.Hkv + 31) / 32));
    const auto launch = [&](auto type) {
        using T = decltype(type);
        rope_paged_kernel<T><<<grid, dim3(pcache::THREADS), 0, stream>>>(kv, (T*)qkv, S, divisor_of(S), q_heads, keep_keys, x_batch, x_row, cos_t, sin_t,
                                                                         positions, pos_batch, n_pos);
    };
    if (c.dtype == MI355_DTYPE_BF16) launch(bf16_t{});
    else launch(half_t{});
    return hipGetLastError();
}

static int evict_cap(int max_len, int budget) { return std::max(0, std::min(budget, max_len - budget)); }

// ints: the counts and lists, then (16-byte aligned) the ranks and positions of long sequences
static size_t evict_lists(size_t pairs, int cap) { return (pairs + pairs * 2 * cap + 3) / 4 * 4; }

size_t evict_workspace(const mi355_paged_kv& c, int budget) {
    const int max_len = c.max_pages * c.page_size;
    const size_t pairs = (size_t)c.B * c.Hkv;
    const bool long_ones = max_len > evict::kMostChunks * 4 * evict::THREADS;
    return 4 * evict_lists(pairs, evict_cap(max_len, budget)) + (long_ones ? 16 * pairs * 2 * ((size_t)(max_len + 3) / 4 + evict::THREADS) : 0);
}

hipError_t evict_dispatch(const mi355_paged_kv& c, int budget, int recent, int* lens_out, void* workspace, hipStream_t stream) {
    using namespace evict;
    const PagedKv kv = paged_from(c);
    const int pairs = kv.B * kv.Hkv;
    Evict a = {};
    a.budget = budget;
    a.recent = recent;
    a.cap = evict_cap(kv.max_len, budget);
    a.counts = (int*)workspace;
    a.moves = a.counts + pairs;
    a.ranks = (uint4*)((int*)workspace + evict_lists(pairs, a.cap));
    a.lens_out = lens_out;
    a.by_hkv = divisor_of(kv.Hkv);
    const dim3 grid(pairs), block(THREADS);
    const int chunks = (int)(((long)kv.max_len + 4 * THREADS - 1) / (4 * THREADS));
    if (chunks <= 1) evict_select_kernel<1><<<grid, block, 0, stream>>>(kv, a);
    else if (chunks <= 2) evict_select_kernel<2><<<grid, block, 0, stream>>>(kv, a);
    else if (chunks <= 4) evict_select_kernel<4><<<grid, block, 0, stream>>>(kv, a);
    else if (chunks <= kMostChunks) evict_select_kernel<kMostChunks><<<grid, block, 0, stream>>>(kv, a);
    else evict_select_kernel<0><<<grid, block, 0, stream>>>(kv, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.cap <= kMovesHere) return e;
    evict_move_kernel<<<dim3((a.cap + MOVES - 1) / MOVES, pairs), dim3(256), 0, stream>>>(kv, a);
    return hipGetLastError();
}

}  // namespace mi355
