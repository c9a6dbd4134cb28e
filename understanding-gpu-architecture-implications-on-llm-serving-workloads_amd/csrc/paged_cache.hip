// What fills a paged key-value cache and what keeps it short, for gfx950 (MI355X): rotary embedding of a fused projection with its keys and values
// filed into their pages, and eviction by accumulated attention weight. Memory-bound, or bound by their chains of memory round trips.
#include <algorithm>
#include <type_traits>

#include "paged.h"

namespace mi355 {

namespace pcache {
constexpr int THREADS = 256;
}

// Token (b, t) of a fused projection [q_heads | Hkv key heads | Hkv value heads] of 128: queries rotated in place, rotated keys and the values to row
// seq_lens[b] - new + t of the sequence; keep_keys: the rotated keys also where they were read. A thread owns 8 values of the
// lower half of a head and their 8 partners; 8 threads a head, 32 heads a workgroup. The arithmetic is that of rope_kernel (glue.hip).
template <typename T>
__global__ __launch_bounds__(pcache::THREADS) void rope_paged_kernel(PagedKv kv, T* qkv, int S, Divisor by_s, int q_heads, int keep_keys, long x_batch,
                                                                     long x_row, const float* __restrict__ cos_t, const float* __restrict__ sin_t,
                                                                     const int* __restrict__ positions, long pos_batch, int n_pos) {
    using V8 = typename Elem<T>::v8;
    const int head = blockIdx.y * 32 + (threadIdx.x >> 3);
    if (head >= q_heads + 2 * kv.Hkv) return;
    const int b = divide(blockIdx.x, by_s), t = blockIdx.x - b * S;
    const int i0 = (threadIdx.x & 7) * 8;
    T* xp = qkv + b * x_batch + t * x_row + (long)head * 128 + i0;
    V8 lo = *(const V8*)xp;
    V8 hi = *(const V8*)(xp + 64);
    const int n_new = paged_new(kv, b, S);
    if (t >= n_new) return;
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
// as are dropped (closing ranks would move most of the cache for one dropped key).
namespace evict {
constexpr int THREADS = 1024, WAVES = THREADS / 64;
constexpr int BINS = 2048;                    // of 11, 11 and 10 bits
constexpr int kLdsKeys = 36864;               // ranks kept in LDS up to this many keys (144 KiB), behind that in the workspace
constexpr int MOVES = 64;                     // of a workgroup of the moving kernel

// a weight as a whole number of the same order; NaN and the slots of pages outside the pool lowest, minus infinity next
__device__ __forceinline__ uint32_t rank_of(float w) {
    const uint32_t u = __builtin_bit_cast(uint32_t, w == 0.f ? 0.f : w);   // (-0 is 0)
    if (w != w) return 0u;
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
constexpr uint32_t kRecent = 0xffffffffu;     // above plus infinity (0xff800000)
}  // namespace evict

struct Evict {
    int budget, recent, cap;   // cap: the most moves of a (sequence, kv head)
    int* counts;               // [pair]
    int* moves;                // [pair][2][cap]: slots of the dropped keys, of those that take them
    uint32_t* ranks;           // [pair][max_len], where they do not fit LDS
    int* lens_out;
    Divisor by_hkv;
};

// One workgroup per (sequence, kv head)
template <bool IN_LDS>
__global__ __launch_bounds__(evict::THREADS) void evict_select_kernel(PagedKv kv, Evict a) {
    using namespace evict;
    __shared__ int hist[BINS];
    __shared__ int wave_sums[WAVES], wave_sums2[WAVES];
    __shared__ int found[2];
    extern __shared__ uint32_t lds_ranks[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int b = divide(blockIdx.x, a.by_hkv), hkv = blockIdx.x - b * kv.Hkv;
    const int len = paged_len(kv, b);
    if (hkv == 0 && tid == 0) a.lens_out[b] = min(len, a.budget);
    if (len <= a.budget) {
        if (tid == 0) a.counts[blockIdx.x] = 0;
        return;
    }
    uint32_t* ranks = IN_LDS ? lds_ranks : a.ranks + (long)blockIdx.x * kv.max_len;
    const int* table = kv.table + (long)b * kv.table_stride;
    const auto place = [&](int j) -> long {   // of the account of key j; -1: its page is outside the pool
        const int i = divide(j, kv.by_page);
        const int page = table[i];
        return (uint32_t)page < (uint32_t)kv.n_pages ? ((long)page * kv.Hkv + hkv) * kv.page_size + (j - i * kv.page_size) : -1L;
    };

    // the largest position
    int newest = INT32_MIN;
    for (int j = tid; j < len; j += THREADS) {
        const long at = place(j);
        if (at >= 0) newest = max(newest, kv.key_positions[at]);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) newest = max(newest, __shfl_xor(newest, off, 64));
    if (lane == 0) wave_sums[wave] = newest;
    __syncthreads();
    for (int w = 0; w < WAVES; ++w) newest = max(newest, wave_sums[w]);
    const long old = (long)newest - a.recent;   // positions up to here are not recent
    // the ranks
    for (int j = tid; j < len; j += THREADS) {
        const long at = place(j);
        ranks[j] = at < 0 ? 0u : kv.key_positions[at] > old ? kRecent : rank_of(kv.weights[at]);
    }
    // the budget-th largest: 11 bits, 11, then 10; `want` of those whose upper bits are `prefix`
    uint32_t prefix = 0;
    int want = a.budget;
    for (int pass = 0; pass < 3; ++pass) {
        const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        const int above = pass == 0 ? 32 : pass == 1 ? 21 : 10;   // bits that are known
        const uint32_t mask = pass == 2 ? 1023u : 2047u;
        __syncthreads();
        hist[tid] = 0;
        hist[tid + THREADS] = 0;
        __syncthreads();
        for (int j = tid; j < len; j += THREADS) {
            const uint32_t r = ranks[j];
            if (pass == 0 || (r >> above) == prefix) atomicAdd(&hist[(r >> shift) & mask], 1);
        }
        __syncthreads();
        // thread t: the bins 2047 - 2t and 2046 - 2t; sums from the top
        const int h0 = hist[BINS - 1 - 2 * tid], h1 = hist[BINS - 2 - 2 * tid];
        int incl = wave_inclusive_sum(h0 + h1);
        if (lane == 63) wave_sums2[wave] = incl;
        __syncthreads();
        for (int w = 0; w < wave; ++w) incl += wave_sums2[w];
        const int before = incl - h0 - h1;
        if (before < want && want <= before + h0) found[0] = BINS - 1 - 2 * tid, found[1] = want - before;
        else if (before + h0 < want && want <= incl) found[0] = BINS - 2 - 2 * tid, found[1] = want - before - h0;
        __syncthreads();
        prefix = pass == 0 ? (uint32_t)found[0] : (prefix << (pass == 1 ? 11 : 10)) | (uint32_t)found[0];
        want = found[1];
    }
    // `want` of the keys of rank `prefix` are kept, the first ones. A wave owns a run of slots and goes through it three times:
    // how many such keys, how many holes and moving keys, then the lists.
    const int run = (((len + WAVES - 1) / WAVES) + 63) & ~63;
    const int j0 = min(wave * run, len), j1 = min(j0 + run, len);
    int ties = 0;
    for (int j = j0; j < j1; j += 64) ties += __popcll(__builtin_amdgcn_ballot_w64(j + lane < j1 && ranks[j + lane] == prefix));
    __syncthreads();
    if (lane == 0) wave_sums[wave] = ties;
    __syncthreads();
    int tie0 = 0;
    for (int w = 0; w < wave; ++w) tie0 += wave_sums[w];
    const auto kept = [&](int j, int& tie) {   // of key j + lane; `tie`: such keys in front of this call's
        const bool there = j + lane < j1;
        const uint32_t r = there ? ranks[j + lane] : 0u;
        const uint64_t equal = __builtin_amdgcn_ballot_w64(there && r == prefix);
        const int mine = tie + __popcll(equal & ((1ULL << lane) - 1));
        tie += __popcll(equal);
        return there && (r > prefix || (r == prefix && mine < want));
    };
    int holes = 0, movers = 0, tie = tie0;
    for (int j = j0; j < j1; j += 64) {
        const bool keep = kept(j, tie);
        holes += __popcll(__builtin_amdgcn_ballot_w64(j + lane < j1 && !keep && j + lane < a.budget));
        movers += __popcll(__builtin_amdgcn_ballot_w64(keep && j + lane >= a.budget));
    }
    if (lane == 0) wave_sums2[wave] = holes;
    __syncthreads();
    if (lane == 0) wave_sums[wave] = movers;
    __syncthreads();
    int hole0 = 0, mover0 = 0, total = 0;
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) hole0 += wave_sums2[w], mover0 += wave_sums[w];
        total += wave_sums2[w];
    }
    if (tid == 0) a.counts[blockIdx.x] = total;
    int* to = a.moves + (long)blockIdx.x * 2 * a.cap;
    int* from = to + a.cap;
    tie = tie0;
    for (int j = j0; j < j1; j += 64) {
        const bool keep = kept(j, tie);
        const bool hole = j + lane < j1 && !keep && j + lane < a.budget, mover = keep && j + lane >= a.budget;
        const uint64_t hm = __builtin_amdgcn_ballot_w64(hole), mm = __builtin_amdgcn_ballot_w64(mover);
        const uint64_t below = (1ULL << lane) - 1;
        if (hole) to[hole0 + __popcll(hm & below)] = j + lane;
        if (mover) from[mover0 + __popcll(mm & below)] = j + lane;
        hole0 += __popcll(hm);
        mover0 += __popcll(mm);
    }
}

// Grid (moves / 64, pairs): 32 threads move a key, its value, its weight and its position
__global__ __launch_bounds__(256) void evict_move_kernel(PagedKv kv, Evict a) {
    using namespace evict;
    const int count = a.counts[blockIdx.y];
    const int b = divide(blockIdx.y, a.by_hkv), hkv = blockIdx.y - b * kv.Hkv;
    const int* table = kv.table + (long)b * kv.table_stride;
    const int* to = a.moves + (long)blockIdx.y * 2 * a.cap;
    const int l32 = threadIdx.x & 31;
    for (int n = blockIdx.x * MOVES + (threadIdx.x >> 5); n < min(count, (int)(blockIdx.x + 1) * MOVES); n += 8) {
        const int d = to[n], s = to[a.cap + n];
        const int di = divide(d, kv.by_page), si = divide(s, kv.by_page);
        const int dp = table[di], sp = table[si];
        if ((uint32_t)dp >= (uint32_t)kv.n_pages || (uint32_t)sp >= (uint32_t)kv.n_pages) continue;
        const int ds = d - di * kv.page_size, ss = s - si * kv.page_size;
        const long head = (long)(hkv + (l32 >> 4) * kv.Hkv) * kv.head_bytes + (l32 & 15) * 16;
        *(int4v*)(kv.pages + (long)dp * kv.page_bytes + head + (uint32_t)ds * kv.row_bytes) =
            *(const int4v*)(kv.pages + (long)sp * kv.page_bytes + head + (uint32_t)ss * kv.row_bytes);
        const long da = ((long)dp * kv.Hkv + hkv) * kv.page_size + ds, sa = ((long)sp * kv.Hkv + hkv) * kv.page_size + ss;
        if (l32 == 0) kv.weights[da] = kv.weights[sa];
        if (l32 == 16) kv.key_positions[da] = kv.key_positions[sa];
    }
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

size_t evict_workspace(const mi355_paged_kv& c, int budget) {
    const int max_len = c.max_pages * c.page_size;
    const size_t pairs = (size_t)c.B * c.Hkv;
    return 4 * (pairs + pairs * 2 * evict_cap(max_len, budget) + (max_len > evict::kLdsKeys ? pairs * max_len : 0));
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
    a.ranks = (uint32_t*)(a.moves + (size_t)pairs * 2 * a.cap);
    a.lens_out = lens_out;
    a.by_hkv = divisor_of(kv.Hkv);
    if (kv.max_len > kLdsKeys) {
        evict_select_kernel<false><<<dim3(pairs), dim3(THREADS), 0, stream>>>(kv, a);
    } else {
        static DynamicLdsOnce once;
        const hipError_t e = once.ensure(reinterpret_cast<const void*>(evict_select_kernel<true>), kLdsKeys * 4);
        if (e != hipSuccess) return e;
        evict_select_kernel<true><<<dim3(pairs), dim3(THREADS), (size_t)kv.max_len * 4, stream>>>(kv, a);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.cap == 0) return e;
    evict_move_kernel<<<dim3((a.cap + MOVES - 1) / MOVES, pairs), dim3(256), 0, stream>>>(kv, a);
    return hipGetLastError();
}

}  // namespace mi355
