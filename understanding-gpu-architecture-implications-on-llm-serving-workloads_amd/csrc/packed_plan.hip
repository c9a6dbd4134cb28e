// Block tables and slot maps of a packed batch, built from the lengths of its requests on the GPU, for gfx950 (MI355X).
//
// Sequence b has len keys and gets n = new_lens[b] tokens, which are rows off_b .. off_b + n - 1 of the batch, off_b = sum of the new_lens in front of it. It
//     fits      where len + n keys have room in its row of the table and off_b + n rows in the batch
//     lacks     the columns len / page .. (len + n - 1) / page of its row that hold no page (where it fits; none for n = 0)
//     is taken  where it fits and lacks nothing, or what it and the sequences in front of it lack is no more than the ring of free pages holds
// Those that are taken get their pages in the order of (sequence, column) from the front of the ring, and their tokens positions and slots (page * page size + row of
// the page). Behind that the pages that no key of a sequence lies in, from column ceil(len' / page) on, go to the ring's end in the same order.
//
// Bound by launches and chains of memory round trips, not by bytes (a table of 256 x 1024 entries is 1 MB): one kernel counts per sequence (a workgroup each), the
// second adds up the counts of all sequences in every workgroup, 256 at a time, and writes its own sequence's part. Places of the ring that are read and that
// are written differ (it holds `count` pages from `first` on and no more than n_pages in all), so nothing waits for anything but the launch in front. us: a step of 64
// sequences of up to 512 pages 3.1 + 4.2, 64 prompts and 192 running sequences of up to 1024 pages 3.7 + 5.6 (lane sums through LDS, and the table read behind the
// counts: 5.8 and 8.0 for the second).
#include <algorithm>

#include "paged.h"

namespace mi355 {

namespace plan {
constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int TAIL = 4096;   // rows behind the last sequence, of a workgroup
}

struct Plan {
    int* table;
    long table_stride;
    int* seq_lens;
    const int* new_lens;
    int* next_positions;   // may be nullptr
    int* ring;
    int* span;
    int *offsets, *positions, *slots, *taken;
    int* counts;           // workspace: first and count of the ring, 2 unused, then [B] x {len, new, lacks, back if taken}, [B] x back if not
    int B, columns, n_pages, page_size, rows, tails;
    Divisor by_page;
};

namespace plan {

__device__ __forceinline__ bool holds(const Plan& p, int page) { return (uint32_t)page < (uint32_t)p.n_pages; }
__device__ __forceinline__ int pages_of(const Plan& p, int keys) { return divide(keys + p.page_size - 1, p.by_page); }

// Inclusive sum over a wave (x >= 0), cut to `most` at every step: with that the sum of any number of terms fits an int.
__device__ __forceinline__ int cut_inclusive_sum(int x, int most) {
    const auto add = [&](int y) { x = min(x + y, most); };
    add(__builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true));   // (the steps of wave_inclusive_sum)
    add(__builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true));
    add(__builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true));
    add(__builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true));
    add(__builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
    add(__builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
    return x;
}
// What the waves in front of this one have, and all of them. `incl`: inclusive sums over this wave, of which the last lane's is its own.
// `sums` is free again behind the caller's next barrier but one.
template <int N>
__device__ __forceinline__ void over_waves(const int (&incl)[N], int most, int (&sums)[WAVES][N], int (&front)[N], int (&all)[N]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane == 63) {
#pragma unroll
        for (int i = 0; i < N; ++i) sums[wave][i] = incl[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        front[i] = all[i] = 0;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            if (w == wave) front[i] = all[i];
            all[i] = min(all[i] + sums[w][i], most);
        }
    }
}
// Sum over the threads in front of this one, and over all
__device__ __forceinline__ int before_and_all(int x, int most, int (&sums)[WAVES][1], int& all) {
    const int incl[1] = {cut_inclusive_sum(x, most)};
    int front[1], whole[1];
    over_waves(incl, most, sums, front, whole);
    all = whole[0];
    const int left = __builtin_amdgcn_update_dpp(0, incl[0], 0x138, 0xf, 0xf, true);   // wave_shr:1, of the lane in front
    return min(left + front[0], most);
}

// What the sequences in front of some sequence took
struct Before {
    int rows, lacks, used, back;   // `used`: pages taken
};

}  // namespace plan

// One workgroup a sequence
__global__ __launch_bounds__(plan::THREADS) void plan_count_kernel(Plan p) {
    using namespace plan;
    __shared__ int sums[3][WAVES];
    const int b = blockIdx.x, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int len = min(max(p.seq_lens[b], 0), p.columns * p.page_size);
    const int n = min(max(p.new_lens[b], 0), p.rows + 1);   // (more than there are rows: cut, for the sums)
    const bool room = n <= p.columns * p.page_size - len;
    const int c0 = divide(len, p.by_page), kept = pages_of(p, len), c1 = room && n > 0 ? pages_of(p, len + n) : kept;
    const int* row = p.table + (long)b * p.table_stride;
    int lacks = 0, back1 = 0, back0 = 0;
    constexpr int AHEAD = 4;
    for (int c = c0 + threadIdx.x; c < p.columns; c += AHEAD * THREADS) {
        int page[AHEAD];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) page[i] = c + i * THREADS < p.columns ? row[c + i * THREADS] : -1;
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int at = c + i * THREADS;
            const bool held = holds(p, page[i]);
            lacks += !held && at < c1 && room && n > 0;
            back1 += held && at >= c1;
            back0 += held && at >= kept;
        }
    }
    lacks = __builtin_amdgcn_readlane(wave_inclusive_sum(lacks), 63);
    back1 = __builtin_amdgcn_readlane(wave_inclusive_sum(back1), 63);
    back0 = __builtin_amdgcn_readlane(wave_inclusive_sum(back0), 63);
    if (lane == 0) sums[0][wave] = lacks, sums[1][wave] = back1, sums[2][wave] = back0;
    __syncthreads();
    if (threadIdx.x != 0) return;
    lacks = back1 = back0 = 0;
    for (int w = 0; w < WAVES; ++w) lacks += sums[0][w], back1 += sums[1][w], back0 += sums[2][w];
    *(int4v*)(p.counts + 4 + 4 * (long)b) = int4v{len, n, room ? lacks : -1, back1};   // (-1: no room)
    p.counts[4 + 4 * (long)p.B + b] = back0;
    if (b == 0) {
        const int first = p.span[0], count = p.span[1];
        p.counts[0] = (uint32_t)first < (uint32_t)p.n_pages ? first : 0;
        p.counts[1] = min(max(count, 0), p.n_pages);
    }
}

// Workgroups 0 .. B - 1: a sequence each; behind them the rows that are no sequence's, and the ring's new span
__global__ __launch_bounds__(plan::THREADS) void plan_write_kernel(Plan p) {
    using namespace plan;
    __shared__ int sums[3][WAVES][1], pairs[WAVES][2];
    __shared__ int found[8];
    __shared__ int pages[THREADS];
    const int tid = threadIdx.x, lane = tid & 63, target = min((int)blockIdx.x, p.B);   // (B: the sums over all)
    // the first entries of this sequence's row are requested beside the counts
    constexpr int AHEAD = 4;
    const int own = min((int)blockIdx.x, p.B - 1);
    int* row = p.table + (long)own * p.table_stride;
    const int c0 = divide(min(max(p.seq_lens[own], 0), p.columns * p.page_size), p.by_page);
    const int next_position = p.next_positions != nullptr ? p.next_positions[own] : -1;
    int ahead[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) ahead[i] = c0 + i * THREADS + tid < p.columns ? row[c0 + i * THREADS + tid] : -1;
    const int first = p.counts[0], count = p.counts[1], most_rows = p.rows + 1;
    Before sum = {0, 0, 0, 0};
    for (int b0 = 0; b0 < p.B && b0 <= target; b0 += THREADS) {
        const int b = b0 + tid;
        int4v c = {0, 0, 0, 0};
        int back0 = 0;
        if (b < p.B) {
            c = *(const int4v*)(p.counts + 4 + 4 * (long)b);
            back0 = p.counts[4 + 4 * (long)p.B + b];
        }
        int all;
        const int off = min(sum.rows + before_and_all(c[1], most_rows, sums[0], all), most_rows);
        sum.rows = min(sum.rows + all, most_rows);
        const bool fits = c[2] >= 0 && off + c[1] <= p.rows;
        const int lacks = fits ? c[2] : 0;
        const int front = sum.lacks + before_and_all(lacks, INT32_MAX, sums[1], all);
        sum.lacks += all;
        const bool taken = fits && (lacks == 0 || front + lacks <= count);
        const int used = sum.used + before_and_all(taken ? lacks : 0, INT32_MAX, sums[2], all);
        sum.used += all;
        const int back = sum.back + before_and_all(taken ? c[3] : back0, INT32_MAX, sums[0], all);
        sum.back += all;
        if (b == target && target < p.B) {
            found[0] = off, found[1] = used, found[2] = back, found[3] = c[0], found[4] = c[1], found[5] = taken;
        }
        __syncthreads();
    }
    if ((int)blockIdx.x >= p.B) {
        const int tail = blockIdx.x - p.B;
        if (tail == 0 && tid == 0) {
            const int begin = first + sum.used;
            p.offsets[p.B] = min(sum.rows, p.rows);
            p.span[0] = begin >= p.n_pages ? begin - p.n_pages : begin;
            p.span[1] = count - sum.used + min(sum.back, p.n_pages - count);
        }
        for (int r = max(sum.rows, tail * TAIL) + tid; r < min(p.rows, (tail + 1) * TAIL); r += THREADS) p.positions[r] = p.slots[r] = -1;
        return;
    }
    const int b = blockIdx.x, off = found[0], used0 = found[1], back0 = found[2], len = found[3], n = found[4];
    const bool taken = found[5] != 0;
    const int len1 = taken ? len + n : len;
    const int next = p.next_positions != nullptr ? next_position : len;
    if (tid == 0) {
        p.offsets[b] = min(off, p.rows);
        p.taken[b] = taken ? n : 0;
        p.seq_lens[b] = len1;   // (everyone has passed a barrier since the old ones were read)
        if (p.next_positions != nullptr) p.next_positions[b] = next + len1 - len;
    }
    if (!taken)
        for (int r = off + tid; r < min(off + n, p.rows); r += THREADS) p.positions[r] = p.slots[r] = -1;
    const int c1 = pages_of(p, len1);
    int used = used0, back = back0;
    for (int base = c0; base < p.columns; base += THREADS) {
        const int c = base + tid;
        int page = ahead[0];
#pragma unroll
        for (int i = 1; i < AHEAD; ++i) ahead[i - 1] = ahead[i];
        ahead[AHEAD - 1] = c + AHEAD * THREADS < p.columns ? row[c + AHEAD * THREADS] : -1;
        const bool held = holds(p, page), wanted = !held && c < c1 && len1 > len, behind = held && c >= c1;
        const uint64_t all_wanted = __builtin_amdgcn_ballot_w64(wanted), all_behind = __builtin_amdgcn_ballot_w64(behind);
        const int wave_has[2] = {__builtin_popcountll(all_wanted), __builtin_popcountll(all_behind)};
        int in_front[2], in_all[2];
        over_waves(wave_has, THREADS, pairs, in_front, in_all);
        const uint64_t lanes_below = ((uint64_t)1 << lane) - 1;
        const int i = used + in_front[0] + __builtin_popcountll(all_wanted & lanes_below), j = back + in_front[1] + __builtin_popcountll(all_behind & lanes_below);
        used += in_all[0];
        back += in_all[1];
        if (wanted) {
            const int at = first + i;
            page = p.ring[at >= p.n_pages ? at - p.n_pages : at];
            row[c] = page;
        }
        if (behind) {
            if (j < p.n_pages - count) {   // (the ring has no more places where a page is held twice)
                const int at = first + count + j;
                p.ring[at >= p.n_pages ? at - p.n_pages : at] = page;
            }
            row[c] = -1;
        }
        if (base < c1 && len1 > len) {   // the tokens of these pages
            pages[tid] = page;
            __syncthreads();
            const int t0 = max(base * p.page_size - len, 0), t1 = min((int)min((long)(base + THREADS) * p.page_size - len, (long)n), n);
            for (int t = t0 + tid; t < t1; t += THREADS) {
                const int key = len + t, column = divide(key, p.by_page), at = pages[column - base];
                p.positions[off + t] = next + t;
                p.slots[off + t] = holds(p, at) ? at * p.page_size + (key - column * p.page_size) : -1;
            }
        }
        __syncthreads();
    }
}

size_t packed_plan_workspace(int B) { return 4 * ((size_t)4 + 5 * (size_t)B); }

hipError_t packed_plan_dispatch(int* table, long table_stride, int* seq_lens, const int* new_lens, int* next_positions, int* ring, int* span, int B, int columns,
                                int n_pages, int page_size, int rows, int* offsets, int* positions, int* slots, int* taken, void* workspace, hipStream_t stream) {
    Plan p = {};
    p.table = table;
    p.table_stride = table_stride;
    p.seq_lens = seq_lens;
    p.new_lens = new_lens;
    p.next_positions = next_positions;
    p.ring = ring;
    p.span = span;
    p.offsets = offsets, p.positions = positions, p.slots = slots, p.taken = taken;
    p.counts = (int*)workspace;
    p.B = B, p.columns = columns, p.n_pages = n_pages, p.page_size = page_size, p.rows = rows;
    p.tails = std::max(1, (rows + plan::TAIL - 1) / plan::TAIL);
    p.by_page = divisor_of(page_size);
    plan_count_kernel<<<dim3(B), dim3(plan::THREADS), 0, stream>>>(p);
    if (hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    plan_write_kernel<<<dim3(B + p.tails), dim3(plan::THREADS), 0, stream>>>(p);
    return hipGetLastError();
}

}  // namespace mi355
