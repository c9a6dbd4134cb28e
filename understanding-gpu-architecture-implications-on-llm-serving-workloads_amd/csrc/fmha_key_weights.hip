// What the rows of a prompt attended to, per key of a paged cache, for gfx950 (MI355X):
//
//   weights[page][kv head][slot of j] += sum over the query heads h of the kv head and the rows i of exp(scale q_hi k_j - LSE_hi)
//
// over the rows i < new (or the last `last_rows` of them) that see the key, j <= i + len - new. LSE is what the attention left: no
// maximum is searched and no probability is written, so the work is one product (MFMA) and an exponential a (row, key).
//
// Bound by issue: of the 2340 cycles that a SIMD takes per 64 keys x 64 rows (2 x 32/8 heads, 4096 rows, causal: 154 us, 890 TFLOP/s), the matrix
// pipe is busy 1024 and the vector unit 1400 (a multiply-add, an exponential and an addition a score, 224 instructions), and the two
// hardly overlap: a software pipeline of product and exponentials took 162 us, 32x32x16 instructions (2 waves to a SIMD instead of 3) 177.
//
// A workgroup owns 256 keys of one (sequence, kv head), which stay in its waves' registers as the A operand of S^T = K Q^T;
// tiles of 64 rows of a query head pass through LDS, three stages, and each wave adds its scores' exponentials up in registers: the sum over the
// columns of an accumulator tile is left for the end, where 16 lanes add theirs. The rows of all heads that see the keys are cut into
// ranges of equally many tiles, a workgroup each (in a causal triangle the first keys have many, the last ones few), and a second kernel adds
// the ranges up in order, so that the same call gives the same bits.
#include <algorithm>
#include <type_traits>

#include "paged.h"

namespace mi355 {

namespace kw {
constexpr int D = 128;
constexpr int BLOCK = 256;                    // keys of a workgroup
constexpr int ROWS = 64;                      // of a tile
constexpr int STAGE_BYTES = ROWS * D * 2;     // 16 KiB
constexpr int NSTAGE = 3;                     // one being worked on, two on their way
constexpr int kMinTiles = 4, kMaxTiles = 16;  // of a range
constexpr int kWorkgroups = 700;              // a little less than run at the same time (three to a CU)
}  // namespace kw

struct KeyWeights {
    const void* Q;
    const float* LSE;
    float* part;      // [range][pair][max_blocks * BLOCK], or nullptr: one range, added to the pages at once
    long q_batch, q_head, q_row;
    int Hq, Sq, group, last_rows, ranges, range_tiles, max_blocks;   // most ranges of a block of keys, tiles of a range
    float scale_log2;
    int pairs;
    Divisor by_hkv, by_pairs, by_blocks, by_group;
};

// sum over the 16 lanes of a row, in every lane (rotations within the row: no trip through LDS)
__device__ __forceinline__ float sum_of_16(float x) {
    const auto turned = [](float v, auto by) {
        return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x120 + decltype(by)::value, 0xf, 0xf, true));
    };
    x += turned(x, std::integral_constant<int, 8>{});
    x += turned(x, std::integral_constant<int, 4>{});
    x += turned(x, std::integral_constant<int, 2>{});
    x += turned(x, std::integral_constant<int, 1>{});
    return x;
}

// Row i sees the keys up to i + len - n_new (a sequence shorter than its rows: its first rows see nothing). Tiles are counted from the last rows,
// which see most, to the first that see any key of the block at block0, the heads of a tile's rows one after the other.
__device__ __forceinline__ int key_weights_first(const KeyWeights& a, int n_new) { return a.last_rows > 0 ? max(n_new - a.last_rows, 0) : 0; }
__device__ __forceinline__ int key_weights_tiles(const KeyWeights& a, int len, int n_new, int block0) {
    return a.group * max((n_new - max(key_weights_first(a, n_new), block0 - (len - n_new)) + kw::ROWS - 1) / kw::ROWS, 0);
}

// Grid: one workgroup per (block of keys, pair, range), placed so that an XCD (workgroups go to the 8 of them in turn) has all blocks of
// keys of a (pair, range) one behind the other: they read the same rows, which then come from its L2. The (pair, range)s go to the XCDs
// there and back, since the later ranges of a causal triangle have fewer blocks.
template <typename T, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void key_weights_kernel(PagedKv kv, KeyWeights a) {
    using namespace kw;
    using V8 = typename Elem<T>::v8;
    constexpr int KEYS = BLOCK / WAVES, NKB = KEYS / 16;   // keys of a wave, blocks of 16 of them
    constexpr int COPIES = 16 / WAVES;                     // of 4 rows, of a wave and tile
    __shared__ __attribute__((aligned(1024))) char smem[NSTAGE * STAGE_BYTES];
    __shared__ float refs[kMaxTiles * ROWS];   // the exponents' offsets of the range's rows
    __shared__ int taken_out;                  // whether the LSE of one of them is -inf
    MI355_LDS char* lds = (MI355_LDS char*)smem;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int g = lane >> 4, c16 = lane & 15;
    const int xcd = blockIdx.x & 7, turn = divide(blockIdx.x >> 3, a.by_blocks);
    const int block0 = ((int)(blockIdx.x >> 3) - turn * a.max_blocks) * BLOCK;
    const int both = turn * 8 + (turn & 1 ? 7 - xcd : xcd);
    const int range = divide(both, a.by_pairs), pair = both - range * a.pairs;
    const int b = divide(pair, a.by_hkv), hkv = pair - b * kv.Hkv;
    if (range >= a.ranges) return;
    const int len = __builtin_amdgcn_readfirstlane(paged_len(kv, b));
    const int n_new = __builtin_amdgcn_readfirstlane(paged_new(kv, b, a.Sq));
    if (block0 >= len) return;
    const int shift = len - n_new, first = key_weights_first(a, n_new);
    const int tiles = key_weights_tiles(a, len, n_new, block0);
    const int t_begin = range * a.range_tiles, t_end = min(t_begin + a.range_tiles, tiles);
    if (range > 0 && t_begin >= tiles) return;

    const int key0 = block0 + wave * KEYS;
    float4v acc[NKB];
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb) acc[kb] = float4v{0.f, 0.f, 0.f, 0.f};
    if (t_begin < t_end) {
        const T* Q = (const T*)a.Q + b * a.q_batch;
        const float* LSE = a.LSE + (long)b * a.Hq * a.Sq;
        // tile t: rows row .. row + 63 of a query head; rows in front of the first that counts repeat it and count for nothing. The waves
        // share its copies (where all are there, to offsets worked out once).
        const uint32_t q_row_bytes = (uint32_t)(a.q_row * 2);
        uint32_t offset[COPIES];
#pragma unroll
        for (int c = 0; c < COPIES; ++c) {
            const int r = 4 * (COPIES * wave + c) + (lane >> 4);
            offset[c] = (uint32_t)r * q_row_bytes + (((lane & 15) ^ (r & 15)) << 4);
        }
        auto issue = [&](int t, int slot) {
            const int back = divide(t, a.by_group), hq = hkv * a.group + t - back * a.group, row = n_new - (back + 1) * ROWS;
            const int at = max(row, first), missing = at - row;
            const char* base = (const char*)(Q + (long)hq * a.q_head + (long)at * a.q_row);
            MI355_LDS char* st = lds + slot * STAGE_BYTES + wave * (COPIES * 1024);
            if (missing == 0) {
#pragma unroll
                for (int c = 0; c < COPIES; ++c) copy16_global_to_lds(base, offset[c], st + c * 1024);
            } else {
#pragma unroll
                for (int c = 0; c < COPIES; ++c) {
                    const int r = 4 * (COPIES * wave + c) + (lane >> 4);
                    copy16_global_to_lds(base, (uint32_t)max(r - missing, 0) * q_row_bytes + (((lane & 15) ^ (r & 15)) << 4), st + c * 1024);
                }
            }
        };
        const int q_base = c16 * 256 + ((g ^ c16) << 4);   // xor (ks << 6), + 16 cb rows
        issue(t_begin, 0);
        if (t_begin + 1 < t_end) issue(t_begin + 1, 1);
        // All rows' offsets up front (a load among the copies would be waited for together with them). A row whose LSE is -inf (or that is none)
        // adds nothing: 2^(x - inf) = 0. That holds for a finite x alone, so a range with such an LSE takes the body with comparisons below (a row that is
        // none repeats the first one, whose own term is not finite either where this one is not)
        // (a flag of each wave's own, which needs no barrier in front of the loop: 2 x 32/8 heads, 4096 rows 156.3 us, this way 153.7, without a flag 155.7)
        if (threadIdx.x == 0) taken_out = 0;
        __syncthreads();
        for (int r = threadIdx.x; r < (t_end - t_begin) * ROWS; r += WAVES * 64) {
            const int t = t_begin + r / ROWS, back = divide(t, a.by_group), hq = hkv * a.group + t - back * a.group;
            const int row = n_new - (back + 1) * ROWS + r % ROWS;
            const float lse = row >= first ? LSE[(long)hq * a.Sq + row] : -INFINITY;
            refs[r] = lse == -INFINITY ? -INFINITY : -lse * 1.4426950408889634f;
            if (row >= first && lse == -INFINITY) taken_out = 1;
        }
        // this wave's keys: lane holds K[16 kb + c16][32 ks + 8 g .. +7]; keys behind the last repeat it, those of a page outside the
        // pool read its first one (neither is written out)
        V8 kf[NKB][4];
        const int* table = kv.table + (long)b * kv.table_stride;
        const char* heads = kv.pages + (long)hkv * kv.head_bytes;
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb) {
            const int key = min(key0 + 16 * kb + c16, len - 1);
            const int i = divide(key, kv.by_page);
            int page = table[i];
            page = (uint32_t)page < (uint32_t)kv.n_pages ? page : 0;
            const char* p = heads + (long)page * kv.page_bytes + (uint32_t)(key - i * kv.page_size) * kv.row_bytes + 16 * g;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) kf[kb][ks] = *(const V8*)(p + 64 * ks);
        }
        int slot = 0;
        __syncthreads();
        // a tile from this row on needs no comparisons
        const int plain_from = __builtin_amdgcn_readfirstlane(taken_out) != 0 ? INT32_MAX : key0 + KEYS - 1 - shift;
        for (int t = t_begin; t < t_end; ++t) {
            if (t + 1 < t_end) wait_vmcnt<COPIES>();   // everything but the newest tile has landed
            else wait_vmcnt<0>();
            __syncthreads();   // everybody's copies; the stage of the tile before is free
            if (t + 2 < t_end) issue(t + 2, slot == 0 ? 2 : slot - 1);
            const int row = n_new - (divide(t, a.by_group) + 1) * ROWS;
            MI355_LDS char* st = lds + slot * STAGE_BYTES;
            const float* ref_of = refs + (t - t_begin) * ROWS;
            slot = slot == NSTAGE - 1 ? 0 : slot + 1;
            // 16 rows against this wave's 64 keys, four times. MASKED: the tile holds rows that do not see all of them, or add nothing (a body of its
            // own: the comparisons would double the vector instructions of the others)
            const auto tile = [&](auto mask) {
#pragma unroll
                for (int cb = 0; cb < 4; ++cb) {
                    V8 qf[4];
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        qf[ks] = Elem<T>::frag(lds_read_b128(st + (q_base ^ (ks << 6)) + 16 * cb * 256));
                    const float ref = ref_of[16 * cb + c16];
                    float4v s[NKB];
#pragma unroll
                    for (int kb = 0; kb < NKB; ++kb) s[kb] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                        for (int kb = 0; kb < NKB; ++kb) s[kb] = Elem<T>::mfma16(kf[kb][ks], qf[ks], s[kb]);
                    // of this lane's keys 16 kb + e, those up to here count
                    const int seen = ref == -INFINITY ? -1 : row + 16 * cb + c16 + shift - key0 - 4 * g;
#pragma unroll
                    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][e], a.scale_log2, ref));
                            if constexpr (decltype(mask)::value) p = 16 * kb + e > seen ? 0.f : p;
                            acc[kb][e] += p;
                        }
                }
            };
            if (row >= plain_from) tile(std::false_type{});
            else if (row + ROWS - 1 + shift >= key0) tile(std::true_type{});   // (a tile none of whose rows sees these keys is passed over)
        }
#pragma unroll
        for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[kb][e] = sum_of_16(acc[kb][e]);
    }
    // lane c16 = 4 kb + e of a group writes its key 16 kb + 4 g + e (with fewer keys the upper lanes have none)
    float out = 0.f;
#pragma unroll
    for (int kb = 0; kb < NKB; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e) out = c16 == 4 * kb + e ? acc[kb][e] : out;
    const int key = key0 + 16 * (c16 >> 2) + 4 * g + (c16 & 3);
    if (c16 >= 4 * NKB || key >= len) return;
    if (a.part != nullptr) {
        a.part[((long)range * a.pairs + pair) * ((long)a.max_blocks * BLOCK) + key] = out;
        return;
    }
    const int i = divide(key, kv.by_page);
    const int page = kv.table[(long)b * kv.table_stride + i];
    if ((uint32_t)page < (uint32_t)kv.n_pages)
        kv.weights[((long)page * kv.Hkv + hkv) * kv.page_size + (key - i * kv.page_size)] += out;
}

// Adds the ranges' sums to the pages: grid (blocks of keys, pairs), a thread per key (its 256 are a workgroup's of the kernel above)
__global__ __launch_bounds__(256) void key_weights_sum_kernel(PagedKv kv, KeyWeights a) {
    const int b = divide(blockIdx.y, a.by_hkv), hkv = blockIdx.y - b * kv.Hkv;
    const int key = blockIdx.x * 256 + threadIdx.x;
    if (key >= paged_len(kv, b)) return;
    const int i = divide(key, kv.by_page);
    const int page = kv.table[(long)b * kv.table_stride + i];
    if ((uint32_t)page >= (uint32_t)kv.n_pages) return;
    const long stride = (long)gridDim.y * a.max_blocks * kw::BLOCK;
    const float* p = a.part + (long)blockIdx.y * a.max_blocks * kw::BLOCK + key;
    // the ranges of this block of keys, as their workgroups counted them
    const int tiles = key_weights_tiles(a, paged_len(kv, b), paged_new(kv, b, a.Sq), blockIdx.x * 256);
    const int ranges = max((tiles + a.range_tiles - 1) / a.range_tiles, 1);
    float sum = 0.f;
    for (int z0 = 0; z0 < ranges; z0 += 8) {   // eight in flight
        float x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = p[min(z0 + k, ranges - 1) * stride];
#pragma unroll
        for (int k = 0; k < 8; ++k) sum += z0 + k < ranges ? x[k] : 0.f;
    }
    kv.weights[((long)page * kv.Hkv + hkv) * kv.page_size + (key - i * kv.page_size)] += sum;
}

struct KeyWeightsPlan {
    int max_blocks, ranges, range_tiles;
};
static KeyWeightsPlan key_weights_plan(const mi355_paged_kv& c, int Hq, int Sq, int last_rows) {
    using namespace kw;
    KeyWeightsPlan p;
    p.max_blocks = (c.max_pages * c.page_size + BLOCK - 1) / BLOCK;
    const int max_len = c.max_pages * c.page_size, rows = last_rows > 0 ? std::min(last_rows, Sq) : Sq;
    const long most = (long)(Hq / c.Hkv) * ((rows + ROWS - 1) / ROWS);
    // about as many workgroups as run at the same time, where that leaves them few enough tiles; of the tiles, those that the causal triangle
    // of the longest sequence leaves
    const long seen = (long)((__int128)most * c.B * c.Hkv * p.max_blocks * (2L * max_len - std::min(rows, max_len)) / (2L * max_len));
    p.range_tiles = (int)std::max<long>(kMinTiles, std::min<long>(kMaxTiles, (seen + kWorkgroups - 1) / kWorkgroups));
    p.ranges = (int)((most + p.range_tiles - 1) / p.range_tiles);
    return p;
}

// Workgroups of a launch: all blocks of keys of each (pair, range), which are dealt to the XCDs eight at a time
long key_weights_workgroups(const mi355_paged_kv& c, int Hq, int Sq, int last_rows) {
    const KeyWeightsPlan p = key_weights_plan(c, Hq, Sq, last_rows);
    return ((long)c.B * c.Hkv * p.ranges + 7) / 8 * 8 * p.max_blocks;
}

size_t key_weights_workspace(const mi355_paged_kv& c, int Hq, int Sq, int last_rows) {
    const KeyWeightsPlan p = key_weights_plan(c, Hq, Sq, last_rows);
    return p.ranges == 1 ? 0 : sizeof(float) * (size_t)p.ranges * c.B * c.Hkv * p.max_blocks * kw::BLOCK;
}

hipError_t key_weights_dispatch(const mi355_paged_kv& c, const void* Q, const float* LSE, int Hq, int Sq, const long* q_strides, int last_rows,
                                float scale, void* workspace, hipStream_t stream) {
    using namespace kw;
    const PagedKv kv = paged_from(c);
    KeyWeights a = {};
    a.Q = Q;
    a.LSE = LSE;
    a.q_batch = q_strides[0], a.q_head = q_strides[1], a.q_row = q_strides[2];
    a.Hq = Hq;
    a.Sq = Sq;
    a.group = Hq / kv.Hkv;
    a.last_rows = last_rows;
    const KeyWeightsPlan p = key_weights_plan(c, Hq, Sq, last_rows);
    a.max_blocks = p.max_blocks;
    a.ranges = p.ranges;
    a.range_tiles = p.range_tiles;
    a.part = a.ranges > 1 ? (float*)workspace : nullptr;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.pairs = kv.B * kv.Hkv;
    a.by_hkv = divisor_of(kv.Hkv);
    a.by_pairs = divisor_of(a.pairs);
    a.by_blocks = divisor_of(a.max_blocks);
    a.by_group = divisor_of(a.group);
    const dim3 grid((unsigned)key_weights_workgroups(c, Hq, Sq, last_rows));
    // Eight waves of 32 keys where a CU has one or two workgroups (us, eight / four waves: 64 rows of 32/8 heads over 8191 keys 10.2 / 10.5, 1024
    // rows 16.8 / 17.0), four of 64, which read the rows' tiles half as often, where more share one (2 x 32/8 heads, 4096 rows 157.4 / 153.1).
    const bool few = (long)a.max_blocks * a.pairs * a.ranges <= 512;
    const auto launch = [&](auto type) {
        using T = decltype(type);
        if (few) key_weights_kernel<T, 8><<<grid, dim3(512), 0, stream>>>(kv, a);
        else key_weights_kernel<T, 4><<<grid, dim3(256), 0, stream>>>(kv, a);
    };
    if (c.dtype == MI355_DTYPE_BF16) launch(bf16_t{});
    else launch(half_t{});
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.ranges > 1) {
        key_weights_sum_kernel<<<dim3(a.max_blocks, kv.B * kv.Hkv), dim3(256), 0, stream>>>(kv, a);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace mi355
