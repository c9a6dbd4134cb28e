// Attention of one new token (or a few) of every sequence over a paged key-value cache, for gfx950 (MI355X).
//
//   s = scale q k^T over the keys j <= i + len - new of the sequence (row i of `new` tokens, which are its last ones)
//   O = softmax(s) V,  LSE = log sum exp s,  and where the cache keeps account: weights[page][kv head][slot] += sum over the query heads of the
//   kv head and the rows of exp(s - LSE)
//
// Bound by the one read of K and V from HBM (512 bytes a key and kv head for 4 * 128 flops a query row). The lengths of a batch differ and
// are known to the device only, so the cut of the work is made there: the key tiles (32 keys) of all (sequence, kv head) pairs
// lie one behind the other on one axis, and each of a fixed number of workgroups takes an equal piece of it, whatever pairs
// the piece touches. A part of a pair leaves an unnormalised partial result (O~ [128], m, l a column, fp32); a second kernel joins the
// parts of a pair and, beside that, adds to the account from the scores that the first one left. Where a pair is walked by one workgroup it writes O and LSE itself.
//
// Inside a part: the query rows of all heads of the kv head are the columns of S^T = K Q^T (MFMA 16x16x32), so K and V are read
// once per kv head (64 sequences of up to 8192 keys, 64/8 heads: 5.66 TB/s in the kernel, 207 us; matrix pipes busy 4 % of the time). The waves take the part's tiles in turn; each streams its own through two private LDS stages with
// direct-to-LDS copies, no barriers, and keeps a running maximum and sum; the next part's first tiles are requested in front of the last ones'
// arithmetic. 16 keys lie in one page: a lane works out the
// address of one such half tile of the next 64, and the scalar unit picks them up one after the other.
#include <algorithm>
#include <type_traits>

#include "paged.h"

namespace mi355 {

namespace pdec {
typedef float float2v __attribute__((ext_vector_type(2)));
typedef unsigned short ushort2v __attribute__((ext_vector_type(2)));
constexpr int D = 128;
constexpr int TK = 32;                       // keys per tile
constexpr int ROW_BYTES = D * 2;             // 256
constexpr int TILE_BYTES = TK * ROW_BYTES;   // 8 KiB
constexpr int STAGE_BYTES = 2 * TILE_BYTES;  // K + V
constexpr int WAVES = 4, NSTAGE = 2;
constexpr int NTHREADS = WAVES * 64;
constexpr int WAVE_BYTES = NSTAGE * STAGE_BYTES;
constexpr int LDS_BYTES = WAVES * WAVE_BYTES;   // 128 KiB
constexpr int kMeetBytes = 31 << 10;           // the rest of a CU's 160 KiB, less what the compiler may want
// columns of a kv head whose scores are kept for the account: those of one workgroup. us, kept / worked out again from K (which is what more columns take), 64 heads on 8:
// 64 sequences of up to 8192 keys, 32 columns 409 / 554, 8 columns 293 / 519; 8 of 4096 keys, 32 columns 44.6 / 75.9; one of 8191, 32 columns 24.2 / 34.9
constexpr int kMostScores = 32;
constexpr int COPIES = 2 * (TILE_BYTES / 1024);
constexpr int WINDOW = 32;                   // tiles whose addresses a wave holds at a time (64 half tiles, one a lane)
constexpr float kLazyLog2 = 8.f;             // rescale only when a column maximum grows by more than 2^8
constexpr int PART_STRIDE = D + 4;           // floats per (part, column): O~[128], m, l, 2 pad (keeps rows 16-byte aligned)
constexpr int kWorkgroups = 256;             // one per CU
constexpr int kMinTiles = 4;                 // of a workgroup: one per wave
constexpr int kDirectLen = 512;              // up to this many keys a workgroup per (sequence, kv head) walks them all (paged_plan)

__device__ __forceinline__ int swz_k(int row) { return row & 15; }
__device__ __forceinline__ int swz_v(int row) { return (row & 7) << 1; }
__device__ __forceinline__ float quad_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    return fmaxf(x, __shfl_xor(x, 32, 64));
}
__device__ __forceinline__ float quad_sum(float x) {
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}
}  // namespace pdec

struct PagedAttn {
    const void* Q;
    void* O;
    float* LSE;       // may be nullptr
    float* part;      // [workgroup + pair][column of a block][PART_STRIDE] per block of columns
    float* scores;    // [pair][max_tiles][ncols][32], where the cache keeps account
    long q_batch, q_head, q_row, o_batch, o_head, o_row;
    long part_block;  // floats of `part` per block of columns
    int Hq, Sq, group, ncols, col_block;   // columns of a kv head, and of a workgroup
    int workgroups, min_tiles, direct, max_tiles;
    int apart;        // the waves' results meet behind the stages
    float scale_log2;
    int chunks;       // of 256 keys, of the longest sequence
    Divisor by_sq, by_hkv, by_ncols, by_chunks;
};

namespace pdec {

// Where the work is cut: `quota` tiles a workgroup over the axis of all pairs' tiles.
struct Cut {
    int total, quota;
};
// One sequence on that axis: its number, its length, its tiles and those of the sequences in front of it (per kv head).
struct Where {
    int b, len, tiles, before;
};
__device__ __forceinline__ int tiles_of(int len) { return (len + TK - 1) / TK; }

// The lengths of up to 64 sequences at a time, one a lane. With up to 64 of them both functions work on the same registers.
struct Lengths {
    const PagedKv& kv;
    int lane, len, incl;   // of sequence `first + lane`
    int first;
    __device__ __forceinline__ Lengths(const PagedKv& kv_) : kv(kv_), lane(threadIdx.x & 63), first(-1) {}
    __device__ __forceinline__ void load(int b0) {
        if (first == b0) return;
        first = b0;
        const int b = b0 + lane;
        len = b < kv.B ? paged_len(kv, b) : 0;
        incl = wave_inclusive_sum(tiles_of(len));
    }
    __device__ __forceinline__ Cut cut(const PagedAttn& a) {
        int total = 0;
        for (int b0 = 0; b0 < kv.B; b0 += 64) {
            load(b0);
            total += __builtin_amdgcn_readlane(incl, 63);
        }
        total *= kv.Hkv;
        return {total, max((int)((uint32_t)(total + a.workgroups - 1) / (uint32_t)a.workgroups), a.min_tiles)};
    }
    __device__ __forceinline__ Where pick(int i, int before) const {
        const int n = __builtin_amdgcn_readlane(len, i), t = tiles_of(n);
        return {first + i, n, t, before + __builtin_amdgcn_readlane(incl, i) - t};
    }
    // the sequence that tile f of the axis belongs to (f < total)
    __device__ __forceinline__ Where find(int f) {
        int before = 0;
        for (int b0 = 0;; b0 += 64) {
            load(b0);
            const uint64_t past = __builtin_amdgcn_ballot_w64(f < (before + incl) * kv.Hkv);
            if (past != 0) return pick(__builtin_ctzll(past), before);
            before += __builtin_amdgcn_readlane(incl, 63);
            if (b0 + 64 >= kv.B) return {kv.B - 1, 0, 0, before};   // (not reached for f < total)
        }
    }
    // sequence b
    __device__ __forceinline__ Where at(int b) {
        int before = 0;
        for (int b0 = 0;; b0 += 64) {
            load(b0);
            if (b < b0 + 64) return pick(b - b0, before);
            before += __builtin_amdgcn_readlane(incl, 63);
        }
    }
};

}  // namespace pdec

// Grid: (workgroups, blocks of columns). NB: blocks of 16 columns of a workgroup. SCORES: the scores are kept for the
// account.
template <typename T, int NB, bool SCORES>
__global__ __launch_bounds__(pdec::NTHREADS) void fmha_paged_kernel(PagedKv kv, PagedAttn a) {
    using namespace pdec;
    using V8 = typename Elem<T>::v8;
    extern __shared__ __attribute__((aligned(1024))) char smem_raw[];
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    MI355_LDS char* wbase = (MI355_LDS char*)smem_raw + wave * WAVE_BYTES;
    const int g = lane >> 4;
    const int c16 = lane & 15;
    const int col0 = blockIdx.y * a.col_block;
    const int ncols = min(a.col_block, a.ncols - col0);   // of this workgroup, <= 16 NB
    const T* Q = (const T*)a.Q;
    T* O = (T*)a.O;

    // Part of this workgroup: tiles tile0 .. tile0 + n - 1 of (seq.b, hkv); wave w takes every fourth from tile0 + w on
    struct Part {
        Where seq;
        int hkv, tile0, n;
    };
    Lengths lengths(kv);
    Part now;
    int f = 0, f_end = 0;
    if (a.direct) {
        const int b = divide(blockIdx.x, a.by_hkv);
        const int len = __builtin_amdgcn_readfirstlane(paged_len(kv, b));
        now = {{b, len, tiles_of(len), 0}, (int)blockIdx.x - b * kv.Hkv, 0, tiles_of(len)};
        f_end = now.n;
    } else {
        const Cut cut = lengths.cut(a);
        f = blockIdx.x * cut.quota;
        f_end = min(f + cut.quota, cut.total);
        if (f >= f_end) return;
        now.seq = lengths.find(f);
        if (now.seq.tiles == 0) return;   // (where lengths change under the call)
        const int rest = f - now.seq.before * kv.Hkv;
        now.hkv = (int)((uint32_t)rest / (uint32_t)now.seq.tiles);
        now.tile0 = rest - now.hkv * now.seq.tiles;
        now.n = min(now.seq.tiles - now.tile0, f_end - f);
    }

    // The tiles in flight: of `ahead` (the part whose tiles are being requested), window of 32 of this wave's tiles. Half tile h of it is
    // lane h's: the address of its 16 keys; a half without keys or with a page outside the pool has its bit in `bad` and the pool's
    // first page to read.
    Part ahead = now;
    uint32_t adr_lo = 0, adr_hi = 0;
    uint64_t bad = 0;
    const long v_off = (long)kv.Hkv * kv.head_bytes;
    auto load_window = [&](int i) {
        const int key = ((ahead.tile0 + wave + (i + (lane >> 1)) * WAVES) * 2 + (lane & 1)) * 16;
        const int index = divide(key, kv.by_page);
        const int page = kv.table[(long)ahead.seq.b * kv.table_stride + min(index, kv.max_pages - 1)];
        const bool ok = key < ahead.seq.len && (uint32_t)page < (uint32_t)kv.n_pages;
        bad = __builtin_amdgcn_ballot_w64(!ok);
        const uint64_t adr = (uint64_t)(uintptr_t)kv.pages + (uint64_t)ahead.hkv * kv.head_bytes +
                             (ok ? (uint64_t)page * kv.page_bytes + (uint32_t)(key - index * kv.page_size) * kv.row_bytes : 0);
        adr_lo = (uint32_t)adr;
        adr_hi = (uint32_t)(adr >> 32);
    };
    // this wave's tile i of `ahead` into stage `slot`: copy c covers rows 4c + lane / 16 of a half tile, chunk lane % 16 (the rows' swizzles
    // repeat every 16); rows behind the last key repeat it (masked later)
    const int c_row = lane >> 4;
    uint32_t k_lane[4], v_lane[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const int row = 4 * c + c_row;
        k_lane[c] = (uint32_t)row * kv.row_bytes + ((uint32_t)(c16 ^ swz_k(row)) << 4);
        v_lane[c] = (uint32_t)row * kv.row_bytes + ((uint32_t)(c16 ^ swz_v(row)) << 4);
    }
    uint32_t bad_stage0 = 0, bad_stage1 = 0;   // halves (bits 0, 1) of the tile in each stage that hold no keys at all
    auto issue_tile = [&](int i, int slot) {
        if ((i & (WINDOW - 1)) == 0) load_window(i);
        MI355_LDS char* st = wbase + slot * STAGE_BYTES;
        const int w = (i & (WINDOW - 1)) * 2;
        const uint32_t none = (uint32_t)(bad >> w) & 3;
        if (slot == 0) bad_stage0 = none;
        else bad_stage1 = none;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const char* kb = (const char*)(uintptr_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)adr_lo, w + h) |
                                                      (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)adr_hi, w + h) << 32);
            const char* vb = kb + v_off;
            const int last = ahead.seq.len - 1 - ((ahead.tile0 + wave + i * WAVES) * 2 + h) * 16;
            if (last >= 15) {
#pragma unroll
                for (int c = 0; c < 4; ++c) copy16_global_to_lds(kb, k_lane[c], st + (4 * h + c) * 1024);
#pragma unroll
                for (int c = 0; c < 4; ++c) copy16_global_to_lds(vb, v_lane[c], st + TILE_BYTES + (4 * h + c) * 1024);
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int row = 4 * c + c_row;
                    copy16_global_to_lds(kb, k_lane[c] - (uint32_t)(row - min(row, max(last, 0))) * kv.row_bytes, st + (4 * h + c) * 1024);
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int row = 4 * c + c_row;
                    copy16_global_to_lds(vb, v_lane[c] - (uint32_t)(row - min(row, max(last, 0))) * kv.row_bytes, st + TILE_BYTES + (4 * h + c) * 1024);
                }
            }
        }
    };
    const auto count_of = [&](const Part& p) { return max((p.n - wave + WAVES - 1) / WAVES, 0); };
    // The part behind `now` becomes `ahead` and its first tile is requested. (Tiles are left in front of f_end, so the sequences that follow
    // have some.)
    auto begin_next = [&](int slot) {
        ahead.tile0 = 0;
        if (++ahead.hkv == kv.Hkv) {
            ahead.hkv = 0;
            ahead.seq = lengths.find(f + now.n);
        }
        ahead.n = min(ahead.seq.tiles, f_end - f - now.n);
        const bool any = count_of(ahead) > 0;
        if (any) issue_tile(0, slot);
        return any;
    };

    if (count_of(now) > 0) issue_tile(0, 0);
    int slot = 0;   // stage of the next tile
    for (;;) {      // the parts
        const int n = now.n, n_loc = count_of(now), hkv = now.hkv, b = now.seq.b, len = now.seq.len;
        const bool more = n > 0 && f + n < f_end;   // (a part of nothing ends the walk even where lengths change under the call)
        const int k_base = c16 * ROW_BYTES + ((g ^ c16) << 4);   // xor (ks << 6), + kb * 16 rows
        const int v_row = 4 * g + (c16 >> 2);
        const int v_base = TILE_BYTES + v_row * ROW_BYTES + ((((c16 & 3) >> 1) ^ swz_v(v_row)) << 4) + (c16 & 1) * 8;  // xor (db << 5)

        float4v o[NB][8];
        float m_run[NB], l_run[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            m_run[nb] = -INFINITY;
            l_run[nb] = 0.f;
#pragma unroll
            for (int db = 0; db < 8; ++db) o[nb][db] = float4v{0.f, 0.f, 0.f, 0.f};
        }
        // queries behind the first copies: column c of the kv head = (its query head c / Sq, row c % Sq)
        const int n_new = paged_new(kv, b, a.Sq);
        int lim[NB];      // last visible key of this lane's column(s); -1: none
        int qrow[NB];
        V8 qf[NB][4];     // Q[column][32 ks + 8 g .. +7]
        int lim_min = len - 1, lim_max = -1;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int col = col0 + min(16 * nb + c16, ncols - 1);
            const int head = divide(col, a.by_sq);
            const int qi = col - head * a.Sq;
            const T* qp = Q + b * a.q_batch + (long)(hkv * a.group + head) * a.q_head + qi * a.q_row + 8 * g;
            qrow[nb] = qi;
            lim[nb] = qi < n_new ? min(len - 1, qi + len - n_new) : -1;
            lim_min = min(lim_min, lim[nb]);
            lim_max = max(lim_max, lim[nb]);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) qf[nb][ks] = *(const V8*)(qp + ks * 32);
        }
        int row_min = a.Sq, row_max = -1;   // rows of the columns of this wave
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) row_min = min(row_min, qrow[nb]), row_max = max(row_max, qrow[nb]);
#pragma unroll
        for (int off = 8; off >= 1; off >>= 1) {
            lim_min = min(lim_min, __shfl_xor(lim_min, off, 64));
            lim_max = max(lim_max, __shfl_xor(lim_max, off, 64));
            row_min = min(row_min, __shfl_xor(row_min, off, 64));
            row_max = max(row_max, __shfl_xor(row_max, off, 64));
        }
        lim_min = __builtin_amdgcn_readfirstlane(lim_min);
        lim_max = __builtin_amdgcn_readfirstlane(lim_max);
        row_min = __builtin_amdgcn_readfirstlane(row_min);
        row_max = __builtin_amdgcn_readfirstlane(row_max);
        // a use of the query fragments in front of the loop: their first use inside it would make the compiler wait there, on every
        // iteration, for everything in flight
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) asm volatile("" : "+v"(qf[nb][0]), "+v"(qf[nb][1]), "+v"(qf[nb][2]), "+v"(qf[nb][3]));

        bool begun = false;   // the next part's first tile has been requested
        for (int i = 0; i < n_loc; ++i) {
            bool newer = true;
            if (i + 1 < n_loc) {
                issue_tile(i + 1, slot ^ 1);
            } else if (a.apart && more) {
                newer = begin_next(slot ^ 1);
                begun = true;
            } else {
                newer = false;
            }
            if (newer) wait_vmcnt<COPIES>();   // everything but the newest tile has landed
            else wait_vmcnt<0>();
            MI355_LDS char* st = wbase + slot * STAGE_BYTES;
            const int tile = now.tile0 + wave + i * WAVES;
            const int key0 = tile * TK;
            const uint32_t no_keys = slot == 0 ? bad_stage0 : bad_stage1;
            slot ^= 1;

            // S^T = K Q^T: lane holds keys 16 kb + 4 g + 0..3 of its column
            float4v s[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) s[nb][0] = s[nb][1] = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) {
                    V8 kf = Elem<T>::frag(lds_read_b128(st + ((k_base ^ (ks << 6)) + kb * 16 * ROW_BYTES)));
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) s[nb][kb] = Elem<T>::mfma16(kf, qf[nb][ks], s[nb][kb]);
                }
            const bool masked = key0 + TK - 1 > lim_min || no_keys != 0;
            if (masked) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        if (key0 + 16 * (e >> 2) + 4 * g + (e & 3) > lim[nb] || ((no_keys >> (e >> 2)) & 1)) s[nb][e >> 2][e & 3] = -INFINITY;
            }
            if constexpr (SCORES) {
                float* sp = a.scores + (((long)b * kv.Hkv + hkv) * a.max_tiles + tile) * (a.ncols * TK);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
                    if (16 * nb + c16 < ncols) {
                        *(float4v*)(sp + (16 * nb + c16) * TK + 4 * g) = s[nb][0];
                        *(float4v*)(sp + (16 * nb + c16) * TK + 16 + 4 * g) = s[nb][1];
                    }
            }
            // lazy rescaling: m_run is the exponent reference of the running sums and only moves (with O and l rescaled) when
            // some score exceeds it by more than 2^kLazyLog2
            float mx[NB];
            bool raise = false;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                mx[nb] = fmaxf(fmaxf(fmaxf(s[nb][0][0], s[nb][0][1]), fmaxf(s[nb][0][2], s[nb][0][3])),
                               fmaxf(fmaxf(s[nb][1][0], s[nb][1][1]), fmaxf(s[nb][1][2], s[nb][1][3])));
                raise = raise || (mx[nb] - m_run[nb]) * a.scale_log2 > kLazyLog2;  // -inf - -inf = NaN compares false
            }
            if (__builtin_amdgcn_ballot_w64(raise) != 0) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    const float m_new = fmaxf(m_run[nb], quad_max(mx[nb]));
                    const float m_use = (m_new == -INFINITY) ? 0.f : m_new;
                    const float alpha = __builtin_amdgcn_exp2f((m_run[nb] - m_use) * a.scale_log2);
                    m_run[nb] = m_new;
                    l_run[nb] *= alpha;
#pragma unroll
                    for (int db = 0; db < 8; ++db) o[nb][db] *= alpha;
                }
            }
            V8 pf[NB];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const float neg_ms = (m_run[nb] == -INFINITY) ? 0.f : -m_run[nb] * a.scale_log2;
                float psum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[nb][e >> 2][e & 3], a.scale_log2, neg_ms));
                    psum += p;
                    pf[nb][e] = (T)p;   // the second product's operand: 16 bits, at most half a step off each
                }
                l_run[nb] += psum;
            }
            // O^T += V^T P^T; the 8 keys of a lane of P are 4 g + 0..3 and 16 + 4 g + 0..3, V^T is gathered in that order
            // A product with p = 0 is not nothing where v is infinite or NaN: a masked tile that holds such values takes the way below.
            bool finite = true;
            if (masked) {
                ushort2v top = {0, 0};
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const int4v x = *(MI355_LDS const int4v*)(st + TILE_BYTES + c * 1024 + lane * 16);
#pragma unroll
                    for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(ushort2v, x[e] & 0x7fff7fff));
                }
                constexpr unsigned short kInfinity = std::is_same<T, half_t>::value ? 0x7c00 : 0x7f80;
                finite = __builtin_amdgcn_ballot_w64(top[0] >= kInfinity || top[1] >= kInfinity) == 0;
            }
            if (finite) {
#pragma unroll
                for (int db = 0; db < 8; ++db) {
                    MI355_LDS char* vp = st + (v_base ^ (db << 5));
                    V8 vf = Elem<T>::frag(concat(lds_read_tr16_b64(vp), lds_read_tr16_b64(vp + 16 * ROW_BYTES)));
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) o[nb][db] = Elem<T>::mfma16(vf, pf[nb], o[nb][db]);
                }
            } else if (key0 <= lim_max) {
                // What a row does not see is taken out of V, row by row, and the sum is taken over for that row's columns alone.
                for (int r = row_min; r <= row_max; ++r) {
                    const int last = r < n_new ? min(len - 1, r + len - n_new) : -1;
#pragma unroll
                    for (int db = 0; db < 8; ++db) {
                        MI355_LDS char* vp = st + (v_base ^ (db << 5));
                        V8 vf = Elem<T>::frag(concat(lds_read_tr16_b64(vp), lds_read_tr16_b64(vp + 16 * ROW_BYTES)));
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (key0 + 16 * (e >> 2) + 4 * g + (e & 3) > last || ((no_keys >> (e >> 2)) & 1)) vf[e] = (T)0.f;
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {   // (of the row's own columns)
                            const float4v sum = Elem<T>::mfma16(vf, pf[nb], o[nb][db]);
                            if (qrow[nb] == r) o[nb][db] = sum;
                        }
                    }
                }
            }
            wait_lgkmcnt<0>();  // the reads of this slot are complete before a later copy refills it
        }

        if (a.apart && more && !begun) begin_next(slot);   // (a wave without a tile of this part)
        // ---- the waves' results meet in LDS, behind the stages where there is room (a.apart: the next part's first tiles are on their way into
        // those), otherwise in them: per wave O~ [ncols][128] floats, then m [32], l [32] ----
        __syncthreads();
        MI355_LDS float* cmb = (MI355_LDS float*)(smem_raw + (a.apart ? LDS_BYTES : 0));
        const int wave_floats = ncols * D + 64;
        {
            MI355_LDS float* mine = cmb + wave * wave_floats;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const int col = 16 * nb + c16;
                const float l_tot = quad_sum(l_run[nb]);
                if (col < ncols) {
#pragma unroll
                    for (int db = 0; db < 8; ++db) *(MI355_LDS float4v*)(mine + col * D + db * 16 + 4 * g) = o[nb][db];
                    if (g == 0) {
                        mine[ncols * D + col] = m_run[nb];
                        mine[ncols * D + 32 + col] = l_tot;
                    }
                }
            }
        }
        __syncthreads();
        const bool whole = n == now.seq.tiles;   // this part is all of its pair
        float* part = a.part + (whole ? 0 : blockIdx.y * a.part_block + (long)(blockIdx.x + b * kv.Hkv + hkv) * (a.col_block * PART_STRIDE));
        for (int e4 = tid; e4 < ncols * (D / 4); e4 += NTHREADS) {   // output elements (column e4 / 32, d 4 (e4 % 32) .. +3)
            const int c = e4 >> 5, d = (e4 & 31) * 4;
            float mw[WAVES], lw[WAVES];
            float4v ow[WAVES];
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                mw[w] = cmb[w * wave_floats + ncols * D + c];
                lw[w] = cmb[w * wave_floats + ncols * D + 32 + c];
                ow[w] = *(MI355_LDS const float4v*)(cmb + w * wave_floats + 4 * e4);
            }
            float m = -INFINITY, l = 0.f;
            float4v acc = float4v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < WAVES; ++w) m = fmaxf(m, mw[w]);
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                // a wave without a visible key has no weight
                const float wgt = (mw[w] == -INFINITY) ? 0.f : __builtin_amdgcn_exp2f((mw[w] - m) * a.scale_log2);
                acc += wgt * ow[w];
                l += wgt * lw[w];
            }
            if (whole) {
                const float inv = l != 0.f ? 1.f / l : 0.f;
                const int head = divide(col0 + c, a.by_sq), qi = col0 + c - head * a.Sq, hq = hkv * a.group + head;
                typename Elem<T>::v4 ov;
#pragma unroll
                for (int e = 0; e < 4; ++e) ov[e] = (T)(acc[e] * inv);
                *(typename Elem<T>::v4*)(O + b * a.o_batch + (long)hq * a.o_head + qi * a.o_row + d) = ov;
                if (a.LSE != nullptr && d == 0)
                    a.LSE[((long)b * a.Hq + hq) * a.Sq + qi] = l != 0.f ? (m * a.scale_log2 + __builtin_log2f(l)) * 0.69314718055994531f : -INFINITY;
            } else {
                *(float4v*)(part + c * PART_STRIDE + d) = acc;
                if (d == 0) {
                    part[c * PART_STRIDE + D] = m;
                    part[c * PART_STRIDE + D + 1] = l;
                }
            }
        }
        if (!more) return;
        if (!a.apart) {
            __syncthreads();   // the next part's copies overwrite what was read above
            begin_next(slot);
        }
        f += n;
        now = ahead;
    }
}

// The parts of a pair: how many, and the workgroup that has the first
__device__ __forceinline__ int parts_of(const PagedKv& kv, const PagedAttn& a, int b, int hkv, int& first) {
    using namespace pdec;
    Lengths lengths(kv);
    const Cut cut = lengths.cut(a);
    const Where seq = lengths.at(b);
    const int f = seq.before * kv.Hkv + hkv * seq.tiles;
    first = (int)((uint32_t)f / (uint32_t)cut.quota);
    return seq.tiles == 0 ? 0 : (int)((uint32_t)(f + seq.tiles - 1) / (uint32_t)cut.quota) - first + 1;
}

// Joins the parts of a (pair, column): O = sum_p w_p O~_p / sum_p w_p l_p with w_p = 2^((m_p - max m) c). Pairs
// without a key get zeros, those of one part were written by its workgroup. Bound by its chain of memory round trips: the lengths, then
// up to 32 parts at once (a thread takes 4 d of every eighth part, up to four of them in flight; the eight sums meet in LDS). The last
// workgroup of a pair doing this inside the first launch, which takes loads and stores at device scope, was slower: 1 x 32/8 heads over 8191 keys 14.1
// us with this launch, 15.5 without, 4 drafted tokens of 4 x 2048 keys 15.6 and 22.5.
template <typename T>
__device__ __forceinline__ void join_parts(const PagedKv& kv, const PagedAttn& a, int pair, int col) {
    using namespace pdec;
    constexpr int ROUNDS = 4;
    __shared__ __attribute__((aligned(16))) float sums[8][PART_STRIDE];
    const int tid = threadIdx.x, part0 = tid >> 5, d = (tid & 31) * 4;
    const int b = divide(pair, a.by_hkv), hkv = pair - b * kv.Hkv;
    int first;
    const int n = parts_of(kv, a, b, hkv, first);
    if (n == 1) return;
    const int cb = (int)((uint32_t)col / (uint32_t)a.col_block), c = col - cb * a.col_block;
    const int head = divide(col, a.by_sq), qi = col - head * a.Sq, hq = hkv * a.group + head;
    const long stride = (long)a.col_block * PART_STRIDE;
    const float* base = a.part + cb * a.part_block + (long)(first + pair) * stride + c * PART_STRIDE;
    float m = -INFINITY, l = 0.f;
    float4v acc = float4v{0.f, 0.f, 0.f, 0.f};
    // of a part that saw no key: its outputs and l are 0 (or NaN, which stays)
    const auto weight = [&](float x, float ref) { return x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((x - ref) * a.scale_log2); };
    for (int p0 = part0; p0 < n; p0 += 8 * ROUNDS) {
        float4v v[ROUNDS];
        float2v ml[ROUNDS];
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r)
            if (r == 0 || p0 + 8 * r < n) {
                const float* pp = base + (long)(p0 + 8 * r) * stride;
                v[r] = *(const float4v*)(pp + d);
                ml[r] = *(const float2v*)(pp + D);
            } else {
                v[r] = float4v{0.f, 0.f, 0.f, 0.f};
                ml[r] = float2v{-INFINITY, 0.f};
            }
        float m_new = m;
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) m_new = fmaxf(m_new, ml[r][0]);
        const float keep = weight(m, m_new);
        acc *= keep;
        l *= keep;
        m = m_new;
#pragma unroll
        for (int r = 0; r < ROUNDS; ++r) {
            const float w = weight(ml[r][0], m);
            acc += w * v[r];
            l += w * ml[r][1];
        }
    }
    *(float4v*)&sums[part0][d] = acc;
    if (d == 0) sums[part0][D] = m, sums[part0][D + 1] = l;
    __syncthreads();
    if (tid >= 32) return;
    m = -INFINITY;
#pragma unroll
    for (int p = 0; p < 8; ++p) m = fmaxf(m, sums[p][D]);
    acc = float4v{0.f, 0.f, 0.f, 0.f};
    l = 0.f;
#pragma unroll
    for (int p = 0; p < 8; ++p) {
        const float w = weight(sums[p][D], m);
        acc += w * *(const float4v*)&sums[p][d];
        l += w * sums[p][D + 1];
    }
    const float inv = l != 0.f ? 1.f / l : 0.f;
    typename Elem<T>::v4 ov;
#pragma unroll
    for (int e = 0; e < 4; ++e) ov[e] = (T)(acc[e] * inv);
    *(typename Elem<T>::v4*)((T*)a.O + b * a.o_batch + (long)hq * a.o_head + qi * a.o_row + d) = ov;
    if (a.LSE != nullptr && d == 0)
        a.LSE[((long)b * a.Hq + hq) * a.Sq + qi] = l != 0.f ? (m * a.scale_log2 + __builtin_log2f(l)) * 0.69314718055994531f : -INFINITY;
}

// weights[page][kv head][slot] += sum over the pair's columns of 2^(s c - LSE) for 256 keys, one a thread. The log-sum-exp comes from the parts'
// statistics, so that this need not wait for the joining; a pair of one part has it in place.
__device__ __forceinline__ void add_weights(const PagedKv& kv, const PagedAttn& a, int pair, int chunk) {
    using namespace pdec;
    __shared__ float lse[kMostScores];
    const int tid = threadIdx.x;
    const int b = divide(pair, a.by_hkv), hkv = pair - b * kv.Hkv;
    const int len = paged_len(kv, b);
    const int key = chunk * 256 + tid;
    if (chunk * 256 >= len) return;
    // the account as it is and the first scores are fetched beside the statistics
    const int at = min(key, len - 1), i = divide(at, kv.by_page);
    const int page = kv.table[(long)b * kv.table_stride + i];
    const bool there = key < len && (uint32_t)page < (uint32_t)kv.n_pages;
    float* w = kv.weights + ((long)(there ? page : 0) * kv.Hkv + hkv) * kv.page_size + (at - i * kv.page_size);
    const float* sp = a.scores + ((long)pair * a.max_tiles + (at >> 5)) * (a.ncols * TK) + (at & 31);
    constexpr int AHEAD = 8;
    float s[AHEAD];
#pragma unroll
    for (int c = 0; c < AHEAD; ++c) s[c] = sp[min(c, a.ncols - 1) * TK];
    const float old = *w;
    int first = 0;
    const int n = a.direct ? 1 : parts_of(kv, a, b, hkv, first);
    if (n == 1) {
        if (tid < a.ncols) {
            const float x = a.LSE[((long)b * a.Hq + hkv * a.group) * a.Sq + tid];   // columns are consecutive rows
            lse[tid] = x * 1.4426950408889634f;
        }
    } else {
        // 32 lanes a column
        for (int c = tid >> 5; c < a.ncols; c += 8) {
            const float* ps = a.part + (long)(first + pair) * (a.col_block * PART_STRIDE) + c * PART_STRIDE + D;
            const long stride = (long)a.col_block * PART_STRIDE;
            float m = -INFINITY, l = 0.f;
            for (int p = tid & 31; p < n; p += 32) {
                const float2v ml = *(const float2v*)(ps + p * stride);
                const float m_new = fmaxf(m, ml[0]);
                l = m_new == -INFINITY ? l + ml[1]   // (nothing yet, or NaN)
                                       : l * __builtin_amdgcn_exp2f((m - m_new) * a.scale_log2) + ml[1] * __builtin_amdgcn_exp2f((ml[0] - m_new) * a.scale_log2);
                m = m_new;
            }
            float m_all = m;
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) m_all = fmaxf(m_all, __shfl_xor(m_all, off, 64));
            l = m_all == -INFINITY ? l : l * __builtin_amdgcn_exp2f((m - m_all) * a.scale_log2);
#pragma unroll
            for (int off = 16; off >= 1; off >>= 1) l += __shfl_xor(l, off, 64);
            if ((tid & 31) == 0) lse[c] = l != 0.f ? m_all * a.scale_log2 + __builtin_log2f(l) : -INFINITY;
        }
    }
    __syncthreads();
    if (!there) return;
    float sum = 0.f;
    // a row that does not see the key adds nothing, whatever its log-sum-exp is
    const auto add = [&](int c, float x) {
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(x, a.scale_log2, -lse[c]));
        sum += x == -INFINITY ? 0.f : p;
    };
    for (int c0 = 0;;) {
#pragma unroll
        for (int c = 0; c < AHEAD; ++c)
            if (c0 + c < a.ncols) add(c0 + c, s[c]);
        c0 += AHEAD;
        if (c0 >= a.ncols) break;
#pragma unroll
        for (int c = 0; c < AHEAD; ++c) s[c] = sp[min(c0 + c, a.ncols - 1) * TK];
    }
    *w = old + sum;
}

// What is left behind fmha_paged_kernel, side by side: a workgroup per (pair, column) joins parts (none where one workgroup walked all keys), then
// one per (pair, 256 keys) adds to the account (none without one).
template <typename T>
__global__ __launch_bounds__(pdec::NTHREADS) void paged_finish_kernel(PagedKv kv, PagedAttn a) {
    const int joins = a.direct ? 0 : kv.B * kv.Hkv * a.ncols;
    if ((int)blockIdx.x < joins) {
        const int pair = divide(blockIdx.x, a.by_ncols);
        join_parts<T>(kv, a, pair, blockIdx.x - pair * a.ncols);
    } else {
        const int i = blockIdx.x - joins, pair = divide(i, a.by_chunks);
        add_weights(kv, a, pair, i - pair * a.chunks);
    }
}

// What a call takes of its workspace
struct PagedPlan {
    int nb, col_block, blocks, workgroups, direct, max_tiles, scores, lds;
    size_t part_bytes, score_bytes, lse_bytes;
};
static PagedPlan paged_plan(int B, int Hkv, int max_len, int Hq, int Sq, bool weights, bool lse) {
    using namespace pdec;
    PagedPlan p = {};
    const int ncols = Hq / Hkv * Sq;
    const long pairs = (long)B * Hkv;
    p.nb = ncols > 16 ? 2 : 1;
    p.col_block = std::min(ncols, 32);
    p.blocks = (ncols + p.col_block - 1) / p.col_block;
    p.max_tiles = (max_len + TK - 1) / TK;
    // A workgroup per pair needs no joining, but walks the longest sequence alone. us, so / in equal shares, sequences as long as the table is wide: 8 pairs
    // over 512 keys 7.9 / 8.5, over 768 9.4 / 8.5, over 1024 11.1 / 8.6; 128 pairs over 512 9.2 / 12.3, over 1024 14.1 / 17.4 (over 2048 23.0 / 26.6, but 17.5 / 9.1 where
    // one sequence is that long and the others short).
    p.direct = max_len <= kDirectLen || (max_len <= 2 * kDirectLen && pairs >= 128);
    // one workgroup per CU over the blocks of columns (two at most where the work is cut)
    p.workgroups = p.direct ? (int)pairs : (int)std::min<long>((kWorkgroups + p.blocks - 1) / p.blocks, (pairs * p.max_tiles + kMinTiles - 1) / kMinTiles);
    if (!p.direct) p.part_bytes = sizeof(float) * (size_t)p.blocks * (p.workgroups + pairs) * p.col_block * PART_STRIDE;
    p.scores = weights && ncols <= kMostScores;
    const int meet = WAVES * (p.col_block * D + 64) * (int)sizeof(float);
    p.lds = LDS_BYTES + (meet <= kMeetBytes ? meet : 0);
    if (p.scores) p.score_bytes = sizeof(float) * (size_t)pairs * p.max_tiles * ncols * TK;
    if (weights && !lse) p.lse_bytes = (sizeof(float) * (size_t)B * Hq * Sq + 15) & ~size_t(15);
    return p;
}

// Whether the kernel of fmha_paged_rows.hip, whose waves share the keys, takes a call. This one's blocks of 32 columns walk them again and again, but cost
// less where there is little to do. us, this kernel / that one, 32/8 heads: 8191 keys, 16 rows 19.1 / 25, 48 rows 53.8 / 28, 512 rows 197 / 94; 8 sequences
// of 4096 keys, 16 rows 36.4 / 38, 24 rows 93 / 42; 32 of 2048, 16 rows 75 / 59; one of 500 keys, 64 rows 13.8 / 17.8, 300 rows 26.2 / 18.1.
bool fmha_paged_many_rows(const mi355_paged_kv& c, int Hq, int Sq) {
    const long ncols = Hq / c.Hkv * Sq, pairs = (long)c.B * c.Hkv;
    if (ncols <= pdec::kMostScores) return false;
    if (c.max_pages * c.page_size <= pdec::kDirectLen) return pairs * ((ncols + 31) / 32) > pdec::kWorkgroups;
    return ncols > 64 || pairs > 64;
}

bool fmha_paged_keeps_scores(const mi355_paged_kv& c, int Hq, int Sq) { return Hq / c.Hkv * Sq <= pdec::kMostScores; }

size_t fmha_paged_workspace(const mi355_paged_kv& c, int Hq, int Sq, bool lse) {
    const PagedPlan p = paged_plan(c.B, c.Hkv, c.max_pages * c.page_size, Hq, Sq, c.weights != nullptr, lse);
    size_t first = fmha_paged_many_rows(c, Hq, Sq) ? paged_rows_workspace(c, Hq, Sq) : p.part_bytes + p.score_bytes;
    if (c.weights != nullptr && !p.scores) first = std::max(first, key_weights_workspace(c, Hq, Sq, 0));   // (one behind the other)
    return first + p.lse_bytes;
}

template <typename T, int NB, bool SCORES>
static hipError_t launch_paged(const PagedKv& kv, const PagedAttn& a, const PagedPlan& p, hipStream_t stream) {
    using namespace pdec;
    static DynamicLdsOnce once;
    const hipError_t e = once.ensure(reinterpret_cast<const void*>(fmha_paged_kernel<T, NB, SCORES>), LDS_BYTES + kMeetBytes);
    if (e != hipSuccess) return e;
    fmha_paged_kernel<T, NB, SCORES><<<dim3(p.workgroups, p.blocks), dim3(NTHREADS), p.lds, stream>>>(kv, a);
    return hipGetLastError();
}

template <typename T>
static hipError_t fmha_paged_t(const PagedKv& kv, const PagedAttn& a, const PagedPlan& p, hipStream_t stream) {
    using namespace pdec;
    const unsigned pairs = (unsigned)(kv.B * kv.Hkv);
    hipError_t e = p.nb == 1 ? (p.scores ? launch_paged<T, 1, true>(kv, a, p, stream) : launch_paged<T, 1, false>(kv, a, p, stream))
                             : (p.scores ? launch_paged<T, 2, true>(kv, a, p, stream) : launch_paged<T, 2, false>(kv, a, p, stream));
    const unsigned rest = pairs * ((p.direct ? 0u : (unsigned)a.ncols) + (p.scores ? (unsigned)a.chunks : 0u));
    if (e == hipSuccess && rest > 0) {
        paged_finish_kernel<T><<<dim3(rest), dim3(NTHREADS), 0, stream>>>(kv, a);
        e = hipGetLastError();
    }
    return e;
}

hipError_t fmha_paged_dispatch(const mi355_paged_kv& c, const void* Q, void* O, float* LSE, int Hq, int Sq, const long* strides, float scale,
                               void* workspace, hipStream_t stream) {
    const PagedKv kv = paged_from(c);
    const PagedPlan p = paged_plan(kv.B, kv.Hkv, kv.max_len, Hq, Sq, kv.weights != nullptr, LSE != nullptr);
    char* ws = (char*)workspace;
    PagedAttn a = {};
    a.Q = Q;
    a.O = O;
    if (p.lse_bytes) {   // the account needs the log-sum-exp even where the caller does not
        a.LSE = (float*)ws;
        ws += p.lse_bytes;
    } else {
        a.LSE = LSE;
    }
    a.scores = (float*)ws;
    ws += p.score_bytes;
    a.part = (float*)ws;
    a.q_batch = strides[0], a.q_head = strides[1], a.q_row = strides[2];
    a.o_batch = strides[3], a.o_head = strides[4], a.o_row = strides[5];
    a.Hq = Hq;
    a.Sq = Sq;
    a.group = Hq / kv.Hkv;
    a.ncols = a.group * Sq;
    a.col_block = p.col_block;
    a.workgroups = p.workgroups;
    a.min_tiles = pdec::kMinTiles;
    a.direct = p.direct;
    a.apart = p.lds > pdec::LDS_BYTES;
    a.max_tiles = p.max_tiles;
    a.part_block = (long)(p.workgroups + kv.B * kv.Hkv) * p.col_block * pdec::PART_STRIDE;
    a.scale_log2 = scale * 1.4426950408889634f;
    a.by_sq = divisor_of(Sq);
    a.by_hkv = divisor_of(kv.Hkv);
    a.chunks = (kv.max_len + 255) / 256;
    a.by_ncols = divisor_of(a.ncols);
    a.by_chunks = divisor_of(a.chunks);
    hipError_t e = fmha_paged_many_rows(c, Hq, Sq) ? paged_rows_dispatch(c, Q, O, a.LSE, Hq, Sq, strides, scale, ws, stream)
                   : c.dtype == MI355_DTYPE_BF16      ? fmha_paged_t<bf16_t>(kv, a, p, stream)
                                                      : fmha_paged_t<half_t>(kv, a, p, stream);
    if (e == hipSuccess && kv.weights != nullptr && !p.scores)   // many rows: from the log-sum-exp, with the scores worked out again
        e = key_weights_dispatch(c, Q, a.LSE, Hq, Sq, strides, 0, scale, ws, stream);
    return e;
}

}  // namespace mi355
