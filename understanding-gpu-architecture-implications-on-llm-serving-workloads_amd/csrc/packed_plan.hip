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
// are written differ (it holds `count` pages from `first` on and no more than n_pages in all), so nothing waits for anything but the launch in front.
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

// Sum over the threads in front of this one and over all (x >= 0), cut to `most` at every step: with that the sum of any number of terms fits an int.
// `sums` is free again behind the caller's next barrier.
__device__ __forceinline__ int before_and_all(int x, int most, int (&sums)[WAVES], int& all) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int incl = x;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int y = __shfl_up(incl, off, 64);
        incl = lane >= off ? min(incl + y, most) : incl;
    }
    const int left = __shfl_up(incl, 1, 64);   // of the lanes in front
    if (lane == 63) sums[wave] = incl;
    __syncthreads();
    int front = lane > 0 ? left : 0;
    all = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w == wave) front = min(front + all, most);
        all = min(all + sums[w], most);
    }
    return front;
}

// What the sequences in front of some sequence took
struct Before {
    int rows, lacks, used, back;   // `used`: pages taken
};
struct Own {
    int len, n, lacks, taken;
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
    __shared__ int sums[4][WAVES];
    __shared__ int found[8];
    __shared__ int pages[THREADS];
    const int tid = threadIdx.x, target = min((int)blockIdx.x, p.B);   // (B: the sums over all)
    const int first = p.counts[0], count = p.counts[1], most_rows = p.rows + 1;
    Before sum = {0, 0, 0, 0};
    Own own = {0, 0, 0, 0};
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
        const int back = sum.back + before_and_all(taken ? c[3] : back0, INT32_MAX, sums[3], all);
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
    const int next = p.next_positions != nullptr ? p.next_positions[b] : len;
    if (tid == 0) {
        p.offsets[b] = min(off, p.rows);
        p.taken[b] = taken ? n : 0;
        p.seq_lens[b] = len1;
    }
    if (!taken)
        for (int r = off + tid; r < min(off + n, p.rows); r += THREADS) p.positions[r] = p.slots[r] = -1;
    __syncthreads();   // (everyone has the position)
    if (tid == 0 && p.next_positions != nullptr) p.next_positions[b] = next + len1 - len;

    int* row = p.table + (long)b * p.table_stride;
    const int c0 = divide(len, p.by_page), c1 = pages_of(p, len1);
    int used = used0, back = back0;
    for (int base = c0; base < p.columns; base += THREADS) {
        const int c = base + tid;
        int page = c < p.columns ? row[c] : -1;
        const bool held = holds(p, page), wanted = !held && c < c1 && len1 > len, behind = held && c >= c1;
        int n_wanted, n_behind;
        const int i = used + before_and_all(wanted, THREADS, sums[0], n_wanted), j = back + before_and_all(behind, THREADS, sums[1], n_behind);
        used += n_wanted;
        back += n_behind;
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
