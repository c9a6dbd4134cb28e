// What the rows of a prompt attended to, per key of a paged cache, for gfx950 (MI355X):
//
//   weights[page][kv head][slot of j] += sum over the query heads h of the kv head and the rows i of exp(scale q_hi k_j - LSE_hi)
//
// over the rows i < new (or the last `last_rows` of them) that see the key, j <= i + len - new. LSE is what the attention left: no
// maximum is searched and no probability is written, so the work is one product (MFMA) and an exponential a (row, key).
//
// A workgroup owns 256 keys of one (sequence, kv head), 64 a wave, which stay in registers as the A operand of S^T = K Q^T;
// tiles of 64 rows of a query head pass through LDS, two stages, and each wave adds its scores' exponentials up in registers: the sum over the
// columns of an accumulator tile is left for the end, where 16 lanes add theirs. The rows of all heads that see the keys are cut into
// `splits` equal ranges, a workgroup each, and a second kernel adds the ranges up in order, so that the same call gives the same bits.
#include <algorithm>

#include "paged.h"

namespace mi355 {

namespace kw {
constexpr int D = 128;
constexpr int WAVES = 4, NTHREADS = WAVES * 64;
constexpr int KEYS = 64;                      // of a wave
constexpr int BLOCK = WAVES * KEYS;           // of a workgroup
constexpr int ROWS = 64;                      // of a tile
constexpr int STAGE_BYTES = ROWS * D * 2;     // 16 KiB
constexpr int kMinTiles = 4;                  // of a range
constexpr int kWorkgroups = 2048;             // wanted: a causal triangle in equal ranges leaves them very different, the longest first
}  // namespace kw

struct KeyWeights {
    const void* Q;
    const float* LSE;
    float* part;      // [range][pair][max_blocks * BLOCK], or nullptr: one range, added to the pages at once
    long q_batch, q_head, q_row;
    int Hq, Sq, group, last_rows, splits, max_blocks;
    float scale_log2;
    Divisor by_hkv;
};

// Grid (blocks of keys, pairs, ranges)
template <typename T>
__global__ __launch_bounds__(kw::NTHREADS, 2) void key_weights_kernel(PagedKv kv, KeyWeights a) {
    using namespace kw;
    using V8 = typename Elem<T>::v8;
    __shared__ __attribute__((aligned(1024))) char smem[2 * STAGE_BYTES];
    MI355_LDS char* lds = (MI355_LDS char*)smem;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int g = lane >> 4, c16 = lane & 15;
    const int b = divide(blockIdx.y, a.by_hkv), hkv = blockIdx.y - b * kv.Hkv;
    const int len = __builtin_amdgcn_readfirstlane(paged_len(kv, b));
    const int n_new = __builtin_amdgcn_readfirstlane(paged_new(kv, b, a.Sq));
    const int block0 = blockIdx.x * BLOCK;
    if (block0 >= len) return;
    const int shift = len - n_new;   // row i sees the keys up to i + shift (a sequence shorter than its rows: shift < 0)
    const int row0 = max(a.last_rows > 0 ? max(n_new - a.last_rows, 0) : 0, block0 - shift);   // first row that sees any of these keys
    const int per_head = row0 < n_new ? (n_new - row0 + ROWS - 1) / ROWS : 0;
    const int tiles = per_head * a.group;
    const int t_begin = (int)((long)tiles * blockIdx.z / a.splits), t_end = (int)((long)tiles * (blockIdx.z + 1) / a.splits);

    const int key0 = block0 + wave * KEYS;
    float4v acc[4];
#pragma unroll
    for (int kb = 0; kb < 4; ++kb) acc[kb] = float4v{0.f, 0.f, 0.f, 0.f};
    if (t_begin < t_end) {
        // this wave's keys: lane holds K[16 kb + c16][32 ks + 8 g .. +7]; keys behind the last repeat it, those of a page outside the
        // pool read its first one (neither is written out)
        V8 kf[4][4];
        const int* table = kv.table + (long)b * kv.table_stride;
        const char* heads = kv.pages + (long)hkv * kv.head_bytes;
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
            const int key = min(key0 + 16 * kb + c16, len - 1);
            const int i = divide(key, kv.by_page);
            int page = table[i];
            page = (uint32_t)page < (uint32_t)kv.n_pages ? page : 0;
            const char* p = heads + (long)page * kv.page_bytes + (uint32_t)(key - i * kv.page_size) * kv.row_bytes + 16 * g;
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) kf[kb][ks] = *(const V8*)(p + 64 * ks);
        }
        const T* Q = (const T*)a.Q + b * a.q_batch;
        const float* LSE = a.LSE + (long)b * a.Hq * a.Sq;
        float lse[4];
        // tile t: rows row .. row + 63 of a query head; rows behind the last token repeat it and count for nothing. Each wave copies 16 rows.
        auto issue = [&](int t, int slot) {
            const int head = (int)((uint32_t)t / (uint32_t)per_head), row = row0 + (t - head * per_head) * ROWS;
            const int hq = hkv * a.group + head;
            const char* base = (const char*)(Q + (long)hq * a.q_head + (long)row * a.q_row);
            const int last = n_new - 1 - row;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int r = 16 * wave + 4 * c + (lane >> 4);
                copy16_global_to_lds(base, (uint32_t)min(r, last) * (uint32_t)(a.q_row * 2) + (((lane & 15) ^ (r & 15)) << 4),
                                     lds + slot * STAGE_BYTES + (16 * wave + 4 * c) * 256);
            }
#pragma unroll
            for (int cb = 0; cb < 4; ++cb) {
                const int r = 16 * cb + c16;
                lse[cb] = r <= last ? LSE[(long)hq * a.Sq + row + r] : -INFINITY;
            }
        };
        issue(t_begin, 0);
        for (int t = t_begin; t < t_end; ++t) {
            const int slot = (t - t_begin) & 1;
            float ref[4];
            wait_vmcnt<0>();
            // a row that sees no key (or is none) adds nothing: 2^(x - inf) = 0
#pragma unroll
            for (int cb = 0; cb < 4; ++cb) ref[cb] = lse[cb] == -INFINITY ? -INFINITY : -lse[cb] * 1.4426950408889634f;
            __syncthreads();
            if (t + 1 < t_end) issue(t + 1, slot ^ 1);
            const int row = row0 + (t % per_head) * ROWS;
            MI355_LDS char* st = lds + slot * STAGE_BYTES;
            const bool masked = row + shift < key0 + KEYS - 1;
#pragma unroll
            for (int cb = 0; cb < 4; ++cb) {
                V8 qf[4];
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
                    qf[ks] = Elem<T>::frag(lds_read_b128(st + (16 * cb + c16) * 256 + (((4 * ks + g) ^ c16) << 4)));
                float4v s[4];
#pragma unroll
                for (int kb = 0; kb < 4; ++kb) s[kb] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                    for (int kb = 0; kb < 4; ++kb) s[kb] = Elem<T>::mfma16(kf[kb][ks], qf[ks], s[kb]);
                const int seen = row + 16 * cb + c16 + shift - key0 - 4 * g;   // of this lane's keys 16 kb + e, those up to here are seen
#pragma unroll
                for (int kb = 0; kb < 4; ++kb)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][e], a.scale_log2, ref[cb]));
                        if (masked && 16 * kb + e > seen) p = 0.f;
                        acc[kb][e] += p;
                    }
            }
        }
#pragma unroll
        for (int kb = 0; kb < 4; ++kb)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
#pragma unroll
                for (int off = 8; off >= 1; off >>= 1) acc[kb][e] += __shfl_xor(acc[kb][e], off, 64);
            }
    }
    // lane c16 = 4 kb + e of a group writes its key 16 kb + 4 g + e
    float out = 0.f;
#pragma unroll
    for (int kb = 0; kb < 4; ++kb)
#pragma unroll
        for (int e = 0; e < 4; ++e) out = c16 == 4 * kb + e ? acc[kb][e] : out;
    const int key = key0 + 16 * (c16 >> 2) + 4 * g + (c16 & 3);
    if (key >= len) return;
    if (a.part != nullptr) {
        a.part[((long)blockIdx.z * gridDim.y + blockIdx.y) * ((long)a.max_blocks * BLOCK) + key] = out;
        return;
    }
    const int i = divide(key, kv.by_page);
    const int page = kv.table[(long)b * kv.table_stride + i];
    if ((uint32_t)page < (uint32_t)kv.n_pages)
        kv.weights[((long)page * kv.Hkv + hkv) * kv.page_size + (key - i * kv.page_size)] += out;
}

// Adds the ranges' sums to the pages: grid (blocks of keys, pairs), a thread per key
__global__ __launch_bounds__(256) void key_weights_sum_kernel(PagedKv kv, KeyWeights a) {
    const int b = divide(blockIdx.y, a.by_hkv), hkv = blockIdx.y - b * kv.Hkv;
    const int key = blockIdx.x * 256 + threadIdx.x;
    if (key >= paged_len(kv, b)) return;
    const int i = divide(key, kv.by_page);
    const int page = kv.table[(long)b * kv.table_stride + i];
    if ((uint32_t)page >= (uint32_t)kv.n_pages) return;
    const long stride = (long)gridDim.y * a.max_blocks * kw::BLOCK;
    const float* p = a.part + (long)blockIdx.y * a.max_blocks * kw::BLOCK + key;
    float sum = 0.f;
    for (int z = 0; z < a.splits; ++z) sum += p[z * stride];
    kv.weights[((long)page * kv.Hkv + hkv) * kv.page_size + (key - i * kv.page_size)] += sum;
}

static int key_weights_splits(const mi355_paged_kv& c, int Hq, int Sq, int last_rows, int max_blocks) {
    using namespace kw;
    const int rows = last_rows > 0 ? std::min(last_rows, Sq) : Sq;
    const long most = (long)(Hq / c.Hkv) * ((rows + ROWS - 1) / ROWS);
    const long wanted = kWorkgroups / ((long)c.B * c.Hkv * max_blocks);
    return (int)std::max(1L, std::min(wanted, most / kMinTiles));
}

size_t key_weights_workspace(const mi355_paged_kv& c, int Hq, int Sq, int last_rows) {
    const int max_blocks = (c.max_pages * c.page_size + kw::BLOCK - 1) / kw::BLOCK;
    const int splits = key_weights_splits(c, Hq, Sq, last_rows, max_blocks);
    return splits == 1 ? 0 : sizeof(float) * (size_t)splits * c.B * c.Hkv * max_blocks * kw::BLOCK;
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
    a.max_blocks = (kv.max_len + BLOCK - 1) / BLOCK;
    a.splits = key_weights_splits(c, Hq, Sq, last_rows, a.max_blocks);
    a.part = a.splits > 1 ? (float*)workspace : nullptr;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.by_hkv = divisor_of(kv.Hkv);
    const dim3 grid(a.max_blocks, kv.B * kv.Hkv, a.splits);
    if (c.dtype == MI355_DTYPE_BF16) key_weights_kernel<bf16_t><<<grid, dim3(NTHREADS), 0, stream>>>(kv, a);
    else key_weights_kernel<half_t><<<grid, dim3(NTHREADS), 0, stream>>>(kv, a);
    hipError_t e = hipGetLastError();
    if (e == hipSuccess && a.splits > 1) {
        key_weights_sum_kernel<<<dim3(a.max_blocks, kv.B * kv.Hkv), dim3(256), 0, stream>>>(kv, a);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace mi355
