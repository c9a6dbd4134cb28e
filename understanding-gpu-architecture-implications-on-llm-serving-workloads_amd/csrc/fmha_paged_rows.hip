// Attention of many rows (a chunk of a prompt, long drafts) of every sequence over a paged key-value cache, for gfx950 (MI355X): the formulas of
// fmha_paged.hip for more query columns a kv head than one wave holds.
//
// A column is a (row, query head) of a kv head, the heads of a row side by side, so that a block of columns sees nearly the same keys. A
// workgroup is 8 waves of 32 columns each: KG == 1: 256 columns and tiles of 64 keys that all waves read from LDS; KG == 2: 128 columns, and two halves of
// the workgroup that take tiles of 32 keys in turn and meet in LDS at the end. Per 32 keys and wave S^T = K Q^T and O^T += V^T P^T are 32 MFMA 16x16x32 with
// the queries in registers; four LDS stages, filled by direct-to-LDS copies (each wave copies 8 rows of K and of V of a tile, which lie in one page).
//
// Bound by issue: the two waves of a SIMD issue some 400 instructions per 32 keys, of which 64 are the products (2048 rows of 32/8 heads over 8191 keys: 300 us,
// 800 TFLOP/s, matrix pipes busy 40 % of the time). Their products and exponentials take turns (phases, below), which alone gave nothing before the
// maximum was taken with v_max3 and the steps without masks had a loop of their own (104 -> 94 us for 512 rows). Reading V in front of the exponentials
// and all of K in front of the products, three stages, one barrier a tile and no phases: 325 us. With masks and what infinities need inside the one
// loop the registers did not suffice (506 us).
//
// The (block of columns, sequence, kv head) triples lie one behind the other on one axis, each with the tiles that its rows see (lengths are known to the device
// only) and a head that stands for what a part costs beside them, and each of up to 256 workgroups takes an equal piece. A triple that a workgroup
// walks alone is written out at once; the parts of the others go to the workspace, two for a workgroup at most (its first part and its last), and
// paged_rows_join_kernel adds them up in order. Where triples of much the same length come out even, whole ones are dealt out in turn; short sequences,
// one sequence of many rows, and many triples get a workgroup a triple and nothing to join.
//
// Drafted tokens that are a tree (TREE): words of bits as in fmha_paged.hip, a row's in LDS, and triples cut by rules of their own (Pieces). 32 tokens of 32 sequences of up to 4097
// keys, 32/8 heads: 72 us and 6.8 for the join; the keys, each read once, come at 4.2 TB/s, a workgroup takes 1.3 us for 64 keys of 128 columns. 64 tokens over
// 8191 keys: 21.5 + 5.5, of which 10 are the steps; the rest is what comes in front of the first tile (8 us, the queries and three tiles of every workgroup on their way together), the halves'
// meeting, and 17 MB of parts on their way out and in.
#include <algorithm>
#include <type_traits>

#include "paged.h"

namespace mi355 {

namespace prow {
constexpr int D = 128, ROW_BYTES = D * 2;
constexpr int WAVES = 8, NTHREADS = WAVES * 64;
constexpr int NB = 2, WCOLS = 16 * NB;        // columns of a wave
constexpr int NSTAGE = 4;                     // one or two being worked on, three on their way at most
constexpr int STAGE_BYTES = 64 * ROW_BYTES * 2;   // K and V of 64 keys, of one tile or of the halves' two
constexpr int LDS_BYTES = NSTAGE * STAGE_BYTES;   // 128 KiB
constexpr int COPIES = 4;                     // of 4 rows, of a wave and tile
constexpr float kLazyLog2 = 8.f;              // rescale only when a column maximum grows by more than 2^8
constexpr int PART_FLOATS = NB * 8 * 64 * 4 + 2 * WCOLS;   // of a wave: its accumulators as they lie, m, l
constexpr int kWorkgroups = 256;              // one per CU
constexpr int kMinKeys = 256;                 // of a piece
constexpr int kHeadKeys = 512;                // what a part costs beside its keys, in keys (~9 us: its first tiles' way, its accumulators' way out)
constexpr int kPieceKeys = 512, kJoinKeys = 256;   // what a piece of a tree's triple costs beside its keys, and what cutting does, in keys (Pieces)
constexpr int kDirectLen = 512;               // up to this many keys, and from that many triples on, none is cut (plan_of)
constexpr long kDirectTriples = 1024;
constexpr long kWholeColumns = 256 * 256;     // from this many columns of all pairs on a workgroup is one of 256 (plan_of)

__device__ __forceinline__ float quad_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16, 64));
    return fmaxf(x, __shfl_xor(x, 32, 64));
}
// the largest of 8 in four instructions (fmaxf makes the compiler quiet possible signalling NaNs first; v_max3_f32 returns the operands that are none)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ float max8(const float4v& a, const float4v& b) {
    const float x = max3(a[0], a[1], a[2]), y = max3(a[3], b[0], b[1]);
    return max3(max3(x, y, b[2]), b[3], b[3]);
}
__device__ __forceinline__ float quad_sum(float x) {
    x += __shfl_xor(x, 16, 64);
    return x + __shfl_xor(x, 32, 64);
}
}  // namespace prow

struct RowsAttn {
    const void* Q;
    void* O;
    float* LSE;      // may be nullptr
    float* part;     // [2 workgroups][waves of columns][PART_FLOATS]
    long q_batch, q_head, q_row, o_batch, o_head, o_row;
    int Hq, Sq, group, ncols, entries, workgroups;   // entries: (block of columns, sequence)
    PagedTree tree;  // of the drafted tokens, where they are one
    float scale_log2;
    int direct;      // a workgroup a triple
    int joins, few;  // triples or borders, which of them
    int blocks;      // of columns
    int* cuts;       // (a tree's) how many triples are cut, and a CutTriple of each
    Divisor by_group, by_batch, by_hkv;
};

namespace prow {

// Entry e: block of columns e / B of sequence e % B, and the keys that it sees
template <int COLS>
struct Entries {
    const PagedKv& kv;
    const RowsAttn& a;
    int lane, first, len, n_new, keys, incl;   // of entry `first + lane`
    __device__ __forceinline__ Entries(const PagedKv& kv_, const RowsAttn& a_) : kv(kv_), a(a_), lane(threadIdx.x & 63), first(-1) {}
    static constexpr int TK = COLS / 4;           // keys of a tile: 64 or 32
    static constexpr int HEAD = kHeadKeys / TK;   // tiles that a triple counts for beside its own
    static __device__ __forceinline__ int tiles_of(int keys) { return (keys + TK - 1) / TK; }
    static __device__ __forceinline__ int units_of(int keys) { return keys > 0 ? tiles_of(keys) + HEAD : 0; }
    struct Seen {
        int len, n_new, keys;
    };
    struct Where {
        int e, len, n_new, keys, tiles, units, before;   // before: units of the entries in front, per kv head
    };
    __device__ __forceinline__ Seen keys_of(int e) const {
        const int block = divide(e, a.by_batch), b = e - block * kv.B;
        const int len = paged_len(kv, b), n_new = paged_new(kv, b, a.Sq);
        const int row0 = divide(block * COLS, a.by_group), row1 = min(divide(min(block * COLS + COLS, a.ncols) - 1, a.by_group), n_new - 1);
        return {len, n_new, row0 >= n_new ? 0 : max(min(len, len - n_new + row1 + 1), 0)};
    }
    __device__ __forceinline__ void load(int e0) {
        if (first == e0) return;
        first = e0;
        const Seen seen = keys_of(min(e0 + lane, a.entries - 1));
        len = seen.len;
        n_new = seen.n_new;
        keys = e0 + lane < a.entries ? seen.keys : 0;
        incl = wave_inclusive_sum(units_of(keys));
    }
    // block `block` of a sequence
    __device__ __forceinline__ Where block_of(int block, int b, int len, int n_new) const {
        const int row0 = divide(block * COLS, a.by_group), row1 = min(divide(min(block * COLS + COLS, a.ncols) - 1, a.by_group), n_new - 1);
        const int keys = row0 >= n_new ? 0 : max(min(len, len - n_new + row1 + 1), 0);
        return {block * kv.B + b, len, n_new, keys, tiles_of(keys), units_of(keys), 0};
    }
    // units (tiles and heads) of all, and the most of a triple
    struct Sum {
        int total, most;
    };
    __device__ __forceinline__ Sum sum() {
        int n = 0, most = 0;
        for (int e0 = 0; e0 < a.entries; e0 += 64) {
            load(e0);
            n += __builtin_amdgcn_readlane(incl, 63);
            most = max(most, wave_max(units_of(keys)));
        }
        return {n * kv.Hkv, most};
    }
    __device__ __forceinline__ int quota(const Sum& s) const {
        return max((int)((uint32_t)(s.total + a.workgroups - 1) / (uint32_t)a.workgroups), kMinKeys / TK);
    }
    // whether whole triples, dealt to the workgroups in turn, take at most a quarter longer than equal pieces, which cost their parts' way through the
    // workspace (8 x 512 rows of 32/8 heads over 2048 keys 162 us, cut 190; 8 x 128 over 1024 31 / 44)
    __device__ __forceinline__ bool in_turn(const Sum& s) const {
        const int rounds = (int)((uint32_t)(a.entries * kv.Hkv + a.workgroups - 1) / (uint32_t)a.workgroups);
        return 4L * rounds * s.most <= 5L * (s.total / a.workgroups);
    }
    __device__ __forceinline__ Where pick(int i, int before) const {
        const int n = __builtin_amdgcn_readlane(keys, i), u = units_of(n);
        return {first + i, __builtin_amdgcn_readlane(len, i), __builtin_amdgcn_readlane(n_new, i), n, tiles_of(n), u, before + __builtin_amdgcn_readlane(incl, i) - u};
    }
    // the entry that unit f of the axis belongs to
    __device__ __forceinline__ Where find(int f) {
        int before = 0;
        for (int e0 = 0;; e0 += 64) {
            load(e0);
            const uint64_t past = __builtin_amdgcn_ballot_w64(f < (before + incl) * kv.Hkv);
            if (past != 0) return pick(__builtin_ctzll(past), before);
            before += __builtin_amdgcn_readlane(incl, 63);
            if (e0 + 64 >= a.entries) return {a.entries - 1, 0, 0, 0, 0, 0, before};   // (not reached for f < total)
        }
    }
    __device__ __forceinline__ Where at(int e) {
        int before = 0;
        for (int e0 = 0;; e0 += 64) {
            load(e0);
            if (e < e0 + 64) return pick(e - e0, before);
            before += __builtin_amdgcn_readlane(incl, 63);
        }
    }
};

// How the triples of a tree's call of up to 64 sequences are cut: into `pieces` of equal length where they are longer than a piece may be, and dealt out largest
// first, in rounds that run forwards and backwards in turn. Every wave of every workgroup works the same out from the lengths: lane r has the sequence whose pieces are the r-th
// longest, and the sums up to it. The longest piece is one of the longest sequence's 1 / 1 .. 1 / 64 that is no shorter than an equal share (so that at most two pieces a
// workgroup are parts of a triple): the one whose heaviest workgroup is expected to have the least to do. Equal shares of the axis, of which most workgroups have two parts, / this, us, 32/8
// heads (both 1 .. 3 us less since): 32 tokens, 8 sequences of up to 8191 keys 51 / 46, 16 of up to 4097 55 / 54, 32 of up to 2000 59 / 52, 24 of 2000 67 / 50; 64 tokens, 16 of up to 4097
// 87 / 72, 20 of up to 1000 53 / 37; 64/8 heads, 64 tokens, 16 of up to 4097 125 / 116. More sequences get a workgroup a triple, which walks a long one alone: 32 tokens, 64 / 65 / 128 sequences of up to 4097 keys 127 / 149 / 252, one of
// 16384 keys among others of 200 69 / 259 / 277.
template <int COLS>
struct Pieces {
    static constexpr int TK = COLS / 4, HEAD = kPieceKeys / TK, JOIN = kJoinKeys / TK, kLeast = 128 / TK;   // in tiles; kLeast: of a piece
    int b, len, n_new, tiles, pieces, length;   // of this lane's sequence; tiles of a piece
    int items, parts, cut;                      // pieces, pieces of triples that are cut, such triples, up to this lane's
    int all, all_cut;
    __device__ __forceinline__ Pieces() {}
    __device__ __forceinline__ void store(int (*to)[64]) const {
        const int lane = threadIdx.x & 63, all_of[9] = {b, len, n_new, tiles, pieces, length, items, parts, cut};
#pragma unroll
        for (int i = 0; i < 9; ++i) to[i][lane] = all_of[i];
    }
    __device__ __forceinline__ void load(const int (*from)[64]) {
        const int lane = threadIdx.x & 63;
        int* const all_of[9] = {&b, &len, &n_new, &tiles, &pieces, &length, &items, &parts, &cut};
#pragma unroll
        for (int i = 0; i < 9; ++i) *all_of[i] = from[i][lane];
    }
    __device__ __forceinline__ Pieces(const PagedKv& kv, const RowsAttn& a) {
        const int lane = threadIdx.x & 63, each = a.blocks * kv.Hkv;   // triples of a sequence
        int my_len = 0, my_new = 0;
        if (lane < kv.B) my_len = paged_len(kv, lane), my_new = paged_new(kv, lane, a.Sq);
        const int my_tiles = my_new > 0 ? (my_len + TK - 1) / TK : 0;
        const int most = max(wave_max(my_tiles), 1), total = __builtin_amdgcn_readlane(wave_inclusive_sum(my_tiles), 63) * each;
        const int share = (int)((uint32_t)(total + a.workgroups - 1) / (uint32_t)a.workgroups);
        int longest = max(max((int)ceilf((float)most / (float)(lane + 1)), share), kLeast);
        const float per = 1.f / (float)longest;
        float n = 0.f, small = 0.f;   // pieces, those of less than half the length
        for (int s = 0; s < kv.B; ++s) {
            const float share_of = (float)__builtin_amdgcn_readlane(my_tiles, s) * per;
            n += ceilf(share_of);
            small += share_of < .5f ? 1.f : 0.f;
        }
        n *= (float)each;
        small *= (float)each;
        // tiles that the heaviest workgroup counts
        const float load = ((float)total + (float)HEAD * n) / (float)a.workgroups * 1.1f;
        float cost = (float)min(longest, most) + (float)HEAD + (longest < most ? (float)JOIN : 0.f);
        if (n > (float)a.workgroups) {   // (in rounds: the smallest pieces come last)
            const float rounds = n - (float)a.workgroups <= small ? (float)min(longest, most) + 2.f * (float)HEAD
                                                                  : ceilf(n / (float)a.workgroups) * (.9f * (float)total / n + (float)HEAD);
            cost = fmaxf(cost, fmaxf(load, rounds) + (longest < most ? (float)JOIN : 0.f));
        }
        const int best = -wave_max(-(int)fminf(cost * 64.f, 1e9f));
        const int choice = __builtin_ctzll(__builtin_amdgcn_ballot_w64((int)fminf(cost * 64.f, 1e9f) == best));
        longest = __builtin_amdgcn_readlane(longest, choice);
        const int my_pieces = max((int)((uint32_t)(my_tiles + longest - 1) / (uint32_t)longest), 1);
        const int my_length = (int)((uint32_t)(my_tiles + my_pieces - 1) / (uint32_t)my_pieces);
        int longer = 0;
        for (int s = 0; s < kv.B; ++s) {
            const int x = __builtin_amdgcn_readlane(my_length, s);
            longer += x > my_length || (x == my_length && s < lane);
        }
        const int to = lane < kv.B ? longer * 4 : lane * 4;
        b = __builtin_amdgcn_ds_permute(to, lane);
        len = __builtin_amdgcn_ds_permute(to, my_len);
        n_new = __builtin_amdgcn_ds_permute(to, my_new);
        tiles = __builtin_amdgcn_ds_permute(to, my_tiles);
        pieces = __builtin_amdgcn_ds_permute(to, my_pieces);
        length = __builtin_amdgcn_ds_permute(to, my_length);
        const bool there = tiles > 0;
        items = wave_inclusive_sum(there ? pieces * each : 0);
        parts = wave_inclusive_sum(there && pieces > 1 ? pieces * each : 0);
        cut = wave_inclusive_sum(there && pieces > 1 ? each : 0);
        all = __builtin_amdgcn_readlane(items, 63);
        all_cut = __builtin_amdgcn_readlane(cut, 63);
    }
    struct Piece {
        int b, triple, len, n_new, piece, pieces, length, part0, cut;   // triple: (block, kv head) of its sequence; part0: its first part; cut: which of those that are cut
    };
    // item u < all
    __device__ __forceinline__ Piece item(int u, int each) const {
        const int r = __builtin_ctzll(__builtin_amdgcn_ballot_w64(u < items)), p = __builtin_amdgcn_readlane(pieces, r);
        const int i = u - __builtin_amdgcn_readlane(items, r) + p * each, triple = __builtin_amdgcn_readfirstlane((int)((uint32_t)i / (uint32_t)p));
        return {__builtin_amdgcn_readlane(b, r), triple, __builtin_amdgcn_readlane(len, r), __builtin_amdgcn_readlane(n_new, r), i - triple * p, p, __builtin_amdgcn_readlane(length, r),
                __builtin_amdgcn_readlane(parts, r) - p * each + triple * p, __builtin_amdgcn_readlane(cut, r) - each + triple};
    }
};
// What the second kernel needs of a triple that was cut (pieces: 0 where its columns see no key)
struct CutTriple {
    int b, triple, pieces, part0;
};
constexpr int kCutBytes = 16 * (kWorkgroups + 1);   // how many there are, and which, in front of the parts

}  // namespace prow

// TREE: the rows are drafted tokens of a.tree (fmha_paged.hip)
template <typename T, int KG, bool TREE>
__global__ __launch_bounds__(prow::NTHREADS, 2) void paged_rows_kernel(PagedKv kv, RowsAttn a) {
    using namespace prow;
    using V8 = typename Elem<T>::v8;
    using V4 = typename Elem<T>::v4;
    constexpr int CW = WAVES / KG, COLS = CW * WCOLS, TK = 64 / KG;
    constexpr int NKB = TK / 16, NH = TK / 32;               // blocks of 16 keys of a tile, steps of 32
    constexpr int TILES_AHEAD = 64 / NKB;                    // whose addresses a wave holds, a 16-key block a lane
    constexpr int HALF_BYTES = TK * ROW_BYTES * 2, V_AT = TK * ROW_BYTES;
    constexpr unsigned short kInfinity = std::is_same<T, half_t>::value ? 0x7c00 : 0x7f80;
    const auto is_finite = [](T x) { return (__builtin_bit_cast(unsigned short, x) & 0x7fff) < kInfinity; };
    static_assert(HALF_BYTES * KG == STAGE_BYTES && Entries<COLS>::TK == TK, "");
    extern __shared__ __attribute__((aligned(1024))) char smem_raw[];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cw = wave % CW, kg = wave / CW;
    MI355_LDS char* lds = (MI355_LDS char*)smem_raw;
    const int g = lane >> 4, c16 = lane & 15;
    const T* Q = (const T*)a.Q;
    T* O = (T*)a.O;

    // This workgroup's piece of the axis: unit `at` of triple (seq.e, hkv) and the following ones
    Entries<COLS> entries(kv, a);
    typename Entries<COLS>::Where seq;
    int hkv, at = 0, f = 0, f_end = 0;   // (whole triples: f counts them down, the blocks with the most keys first, f_end is the step)
    bool whole = a.direct;
    // (TREE) tile `at` and the n_piece - 1 behind it, the piece's number among the parts
    int n_piece = 0, part_number = 0, round = 0, all_pieces = 0;
    __shared__ int held[TREE ? 9 : 1][64];   // `Pieces`, from one piece to the next
    const auto take_piece = [&]() {          // this workgroup's next; false: none is left
        if constexpr (TREE) {
            const int each = a.blocks * kv.Hkv;
            for (;;) {
                const int u = round * a.workgroups + (round & 1 ? a.workgroups - 1 - (int)blockIdx.x : (int)blockIdx.x);
                if (u >= all_pieces) return false;
                Pieces<COLS> p;
                p.load(held);
                const auto x = p.item(u, each);
                ++round;
                const int block = divide(x.triple, a.by_hkv);
                seq = entries.block_of(block, x.b, x.len, x.n_new);
                if (x.pieces > 1 && x.piece == 0 && tid == 0) ((CutTriple*)a.cuts)[1 + x.cut] = {x.b, x.triple, seq.keys == 0 ? 0 : x.pieces, x.part0};
                if (seq.keys == 0) continue;   // (zeros: the second kernel's)
                hkv = x.triple - block * kv.Hkv;
                at = x.piece * x.length;
                n_piece = max(min(x.length, seq.tiles - at), 0);
                whole = x.pieces == 1;
                part_number = x.part0 + x.piece;
                return true;
            }
        }
        return false;
    };
    const auto take = [&]() {
        const int e = divide(f, a.by_hkv);
        hkv = f - e * kv.Hkv;
        if (a.direct) {
            entries.load(e);
            seq = entries.pick(0, 0);
        } else {
            seq = entries.at(e);
        }
    };
    if constexpr (TREE) {
        if (whole) {   // a workgroup a triple, the blocks with the most keys first
            const int i = a.entries * kv.Hkv - 1 - blockIdx.x, e = divide(i, a.by_hkv), block = divide(e, a.by_batch), b = e - block * kv.B;
            hkv = i - e * kv.Hkv;
            seq = entries.block_of(block, b, __builtin_amdgcn_readfirstlane(paged_len(kv, b)), __builtin_amdgcn_readfirstlane(paged_new(kv, b, a.Sq)));
            n_piece = seq.tiles;
        } else {
            const Pieces<COLS> p(kv, a);
            all_pieces = p.all;
            if (blockIdx.x == 0 && tid == 0) *a.cuts = p.all_cut;
            if (wave == 0) p.store(held);
            __syncthreads();
            if (!take_piece()) return;
        }
    } else {
        if (!whole) {
            const auto sum = entries.sum();
            whole = entries.in_turn(sum);
            const int quota = entries.quota(sum);
            f = blockIdx.x * quota;
            f_end = min(f + quota, sum.total);
        }
        if (whole) {
            f = a.entries * kv.Hkv - 1 - blockIdx.x;
            f_end = a.workgroups;
            if (f < 0) return;
            take();
        } else {
            if (f >= f_end) return;
            seq = entries.find(f);
            if (seq.units == 0) return;   // (where lengths change under the call)
            hkv = (int)((uint32_t)(f - seq.before * kv.Hkv) / (uint32_t)seq.units);
            at = f - seq.before * kv.Hkv - hkv * seq.units;
        }
    }

    uint32_t k_lane[2], v_lane[2];   // of this wave's copies of a tile: rows 8 (cw & 1) + 4 c + lane / 16 of a 16-key block
    const int copy_row = 8 * (cw & 1) + (lane >> 4);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int row = copy_row + 4 * c;
        k_lane[c] = (uint32_t)row * kv.row_bytes + ((uint32_t)(c16 ^ row) << 4);
        v_lane[c] = (uint32_t)row * kv.row_bytes + ((uint32_t)(c16 ^ ((row & 7) << 1)) << 4);
    }
    const long v_off = (long)kv.Hkv * kv.head_bytes;
    const int k_base = c16 * ROW_BYTES + ((g ^ c16) << 4);   // xor (ks << 6), + kb * 16 rows
    const int v_row = 4 * g + (c16 >> 2);
    const int v_base = V_AT + v_row * ROW_BYTES + ((((c16 & 3) >> 1) ^ ((v_row & 7) << 1)) << 4) + (c16 & 1) * 8;   // xor (db << 5)
    int parts = 0;

    for (;;) {
        const int block = divide(seq.e, a.by_batch), b = seq.e - block * kv.B;
        const int units = TREE ? 0 : whole ? seq.units : min(seq.units - at, f_end - f);
        const int tile0 = TREE ? at : max(at - Entries<COLS>::HEAD, 0), n = TREE ? n_piece : at + units - Entries<COLS>::HEAD - tile0;   // (units of the head alone: nothing)
        if (!TREE && n <= 0 && seq.units > 0) return;
        const int n_loc = max((n - kg + KG - 1) / KG, 0);   // tiles kg, kg + KG, .. of the part
        const int keys = seq.keys;                          // those that some row of the block sees
        const int* table = kv.table + (long)b * kv.table_stride;
        const char* heads = kv.pages + (long)hkv * kv.head_bytes;

        // the 16-key blocks of TILES_AHEAD of this half's tiles, one a lane. A block without keys or with a page outside the pool has its bit in `bad` and
        // the pool's first page to read.
        uint32_t adr_lo = 0, adr_hi = 0;
        uint64_t bad = 0;
        const auto key_of_lane = [&](int i) { return ((tile0 + kg + (i + lane / NKB) * KG) * NKB + lane % NKB) * 16; };
        const auto page_of_lane = [&](int i) { return table[min(divide(key_of_lane(i), kv.by_page), kv.max_pages - 1)]; };
        const auto load_window = [&](int i, int page) {
            const int key = key_of_lane(i), index = divide(key, kv.by_page);
            const bool ok = key < keys && (uint32_t)page < (uint32_t)kv.n_pages;
            bad = __builtin_amdgcn_ballot_w64(!ok);
            const uint64_t adr = (uint64_t)(uintptr_t)heads + (ok ? (uint64_t)page * kv.page_bytes + (uint32_t)(key - index * kv.page_size) * kv.row_bytes : 0);
            adr_lo = (uint32_t)adr;
            adr_hi = (uint32_t)(adr >> 32);
        };
        int plain = n_loc * NH;   // the steps in front of the first that needs a mask
        uint32_t empty = 0;   // 4 bits a stage: its tile's blocks without keys
        // this half's tile i into its stage; rows behind the last key repeat it (masked later)
        const auto issue = [&](int i) {
            const int in_window = i & (TILES_AHEAD - 1);
            if (in_window == 0 && i > 0) load_window(i, page_of_lane(i));
            const int slot = i & (NSTAGE - 1);
            const uint32_t none = (uint32_t)(bad >> (in_window * NKB)) & ((1u << NKB) - 1);
            empty = (empty & ~(15u << (4 * slot))) | none << (4 * slot);
            if (none != 0) plain = min(plain, i * NH);
            const int w = in_window * NKB + (cw >> 1);
            const char* kb = (const char*)(uintptr_t)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)adr_lo, w) |
                                                      (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)adr_hi, w) << 32);
            const char* vb = kb + v_off;
            MI355_LDS char* st = lds + slot * STAGE_BYTES + kg * HALF_BYTES + cw * (8 * ROW_BYTES);
            const int last = keys - 1 - ((tile0 + kg + i * KG) * NKB + (cw >> 1)) * 16;
            if (last >= 15) {
#pragma unroll
                for (int c = 0; c < 2; ++c) copy16_global_to_lds(kb, k_lane[c], st + c * 1024);
#pragma unroll
                for (int c = 0; c < 2; ++c) copy16_global_to_lds(vb, v_lane[c], st + V_AT + c * 1024);
            } else {
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int row = copy_row + 4 * c;
                    copy16_global_to_lds(kb, k_lane[c] - (uint32_t)(row - min(row, max(last, 0))) * kv.row_bytes, st + c * 1024);
                }
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int row = copy_row + 4 * c;
                    copy16_global_to_lds(vb, v_lane[c] - (uint32_t)(row - min(row, max(last, 0))) * kv.row_bytes, st + V_AT + c * 1024);
                }
            }
        };
        const int first_page = page_of_lane(0);   // (in front of the queries: its wait is not theirs)
        const int up_mine = TREE && tid < a.Sq ? a.tree.parents[b * a.tree.batch + tid] : 0;   // (a parent a thread)
        // this wave's columns; their loads are under way together with the table's
        const int len = seq.len, n_new = seq.n_new;
        const int col0 = block * COLS + cw * WCOLS;
        V8 qf[NB][4];             // Q[column][32 ks + 8 g .. +7]
        int lim[NB], qrow[NB];    // last visible key of this lane's columns (-1: none), their rows
        int lim_min = len - 1, lim_max = -1, row_min = a.Sq, row_max = -1;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            const int col = min(col0 + 16 * nb + c16, a.ncols - 1);
            const int qi = divide(col, a.by_group), head = col - qi * a.group;
            const T* qp = Q + b * a.q_batch + (long)(hkv * a.group + head) * a.q_head + qi * a.q_row + 8 * g;
            qrow[nb] = qi;
            lim[nb] = qi < n_new ? min(len - 1, qi + len - n_new) : -1;
            if (!TREE || lim[nb] >= 0) lim_min = min(lim_min, lim[nb]);   // (TREE: what the columns of rows that are no tokens see is taken out at the end)
            lim_max = max(lim_max, lim[nb]);
            row_min = min(row_min, qi);
            row_max = max(row_max, qi);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) qf[nb][ks] = *(const V8*)(qp + ks * 32);
        }
        load_window(0, first_page);
        for (int i = 0; i < NSTAGE - 1 && i < n_loc; ++i) issue(i);

        const int base = len - n_new;        // (TREE) key of the first drafted token
        const int row0 = TREE ? divide(block * COLS, a.by_group) : 0;   // first row of the block
        __shared__ int up[TREE ? kMostDrafted : 1];
        __shared__ uint32_t words[TREE ? kMostDrafted * kTreeWords : 1];
        if constexpr (TREE) {
            if ((tile0 + n) * TK > base) {   // the words of the block's rows, where the part reaches the draft (the barrier waits for LDS alone; another one follows)
                if (tid < a.Sq) up[tid] = up_mine;
                wait_lgkmcnt<0>();
                asm volatile("s_barrier" ::: "memory");
                const int rows = divide(min(block * COLS + COLS, a.ncols) - 1, a.by_group) - row0 + 1;
                if (tid < rows) tree_words((MI355_LDS const int*)up, row0 + tid, n_new, base, (MI355_LDS uint32_t*)words + tid * kTreeWords);
            }
        }
        lim_min = -mi355::row_max(-lim_min);
        lim_max = mi355::row_max(lim_max);
        row_min = -mi355::row_max(-row_min);
        row_max = mi355::row_max(row_max);
        if (col0 >= a.ncols) lim_max = -1;   // (a wave without columns)
        if (TREE) lim_min = lim_max < 0 ? -1 : min(lim_min, base - 1);
        // the word of row r for 32 keys from key0 on, which reach the draft
        const auto seen = [&](int key0, int r) { return words[(r - row0) * kTreeWords + (key0 >> 5) - (max(base, 0) >> 5)]; };
        // a use of the query fragments in front of the loop: their first use inside it would make the compiler wait there, on every
        // iteration, for everything in flight
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) asm volatile("" : "+v"(qf[nb][0]), "+v"(qf[nb][1]), "+v"(qf[nb][2]), "+v"(qf[nb][3]));
        float4v o[NB][8];
        // exponent reference of the running sums, the score above which it moves, -reference * scale
        float m_run[NB], m_top[NB], neg_ms[NB], l_run[NB];
        const float margin = fminf(kLazyLog2 / a.scale_log2, 3.0e38f);   // (finite: minus infinity stays that)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            m_run[nb] = m_top[nb] = -INFINITY;
            neg_ms[nb] = 0.f;
            l_run[nb] = 0.f;
#pragma unroll
            for (int db = 0; db < 8; ++db) o[nb][db] = float4v{0.f, 0.f, 0.f, 0.f};
        }

        // The steps of 32 keys. A wave alternates between a matrix phase, S = K Q^T of a step and O += V P of the one before, and a softmax phase, from S
        // to P; the waves of the workgroup's second half, one of two on each SIMD, run one phase behind, so that the matrix pipe and the vector
        // unit are both busy. A tile has landed and is published at the end of the matrix phase in front of its first one; its stage is filled again in
        // the last softmax phase of the tile behind it, when nobody reads it any more.
        const auto phase_barrier = []() { asm volatile("s_barrier" ::: "memory"); };
        const auto pin_o = [&]() {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
                asm volatile("" : "+v"(o[nb][0]), "+v"(o[nb][1]), "+v"(o[nb][2]), "+v"(o[nb][3]), "+v"(o[nb][4]), "+v"(o[nb][5]), "+v"(o[nb][6]), "+v"(o[nb][7]));
        };
        const auto v_frag = [&](MI355_LDS char* st, int db) {
            MI355_LDS char* vp = st + (v_base ^ (db << 5));
            return Elem<T>::frag(concat(lds_read_tr16_b64(vp), lds_read_tr16_b64(vp + 16 * ROW_BYTES)));
        };
        const auto stage_of = [&](int h) { return lds + ((h / NH) & (NSTAGE - 1)) * STAGE_BYTES + kg * HALF_BYTES + (h % NH) * (32 * ROW_BYTES); };
        const auto key_of = [&](int h) { return (tile0 + kg + h / NH * KG) * TK + 32 * (h % NH); };
        const auto none_of = [&](int h) { return (empty >> (4 * ((h / NH) & (NSTAGE - 1)) + 2 * (h % NH))) & 3; };
        float4v s[NB][2];    // lane: keys 16 kb + 4 g + 0..3 of its columns
        V8 kf[4][2], vf[8], pf[NB];
        const auto read_k = [&](MI355_LDS char* st) {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb) kf[ks][kb] = Elem<T>::frag(lds_read_b128(st + ((k_base ^ (ks << 6)) + kb * 16 * ROW_BYTES)));
        };
        const auto read_v = [&](MI355_LDS char* st) {
#pragma unroll
            for (int db = 0; db < 8; ++db) vf[db] = v_frag(st, db);
        };
        // S^T = K Q^T
        const auto first_product = [&]() {
#pragma unroll
            for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) s[nb][kb] = Elem<T>::mfma16(kf[ks][kb], qf[nb][ks], ks == 0 ? float4v{0.f, 0.f, 0.f, 0.f} : s[nb][kb]);
        };
        // O^T += V^T P^T; the 8 keys of a lane of P are 4 g + 0..3 and 16 + 4 g + 0..3, V^T is gathered in that order
        const auto second_product = [&]() {
#pragma unroll
            for (int db = 0; db < 8; ++db)
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) o[nb][db] = Elem<T>::mfma16(vf[db], pf[nb], o[nb][db]);
        };
        const auto softmax = [&]() {
            // lazy rescaling: m_run is the exponent reference of the running sums and only moves (with O and l rescaled) when
            // some score exceeds it by more than 2^kLazyLog2
            float mx[NB];
            bool raise = false;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                mx[nb] = max8(s[nb][0], s[nb][1]);
                raise = raise || mx[nb] > m_top[nb];
            }
            if (__builtin_amdgcn_ballot_w64(raise) != 0) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    const float m_new = fmaxf(m_run[nb], quad_max(mx[nb]));
                    const float m_use = (m_new == -INFINITY) ? 0.f : m_new;
                    const float alpha = __builtin_amdgcn_exp2f((m_run[nb] - m_use) * a.scale_log2);
                    m_run[nb] = m_new;
                    m_top[nb] = m_new + margin;
                    neg_ms[nb] = -m_use * a.scale_log2;
                    l_run[nb] *= alpha;
#pragma unroll
                    for (int db = 0; db < 8; ++db) o[nb][db] *= alpha;
                }
            }
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                float psum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[nb][e >> 2][e & 3], a.scale_log2, neg_ms[nb]));
                    psum += p;
                    pf[nb][e] = (T)p;   // the second product's operand: 16 bits, at most half a step off each
                }
                l_run[nb] += psum;
            }
        };
        const auto landed = [&](int h) {   // the tile behind step h's
            if (h % NH != NH - 1) return;
            if (h / NH + 2 < n_loc) wait_vmcnt<COPIES>();
            else wait_vmcnt<0>();
        };
        const auto refill = [&](int h) {
            if (h % NH == NH - 1 && h / NH + NSTAGE - 1 < n_loc) issue(h / NH + NSTAGE - 1);
        };
        const int steps = (n + KG - 1) / KG * NH;
        if (n_loc >= 3) wait_vmcnt<2 * COPIES>();   // (the first tile)
        else if (n_loc == 2) wait_vmcnt<COPIES>();
        else wait_vmcnt<0>();
        wait_lgkmcnt<0>();
        phase_barrier();
        if (wave >= 4) phase_barrier();
        // the steps whose keys all columns of the wave see, up to the first that holds a page outside the pool
        const int room = lim_min - 31 - (tile0 + kg) * TK;
        plain = min(plain, room < 0 ? 0 : room / (64 / NH) + 1);
        int h = 0;
        // S is read by assembly (max3), in front of which the compiler puts no wait for the matrix pipe. It puts 8 wait states (s_nop 7) between a 16x16x32
        // product and an instruction of its own that reads the result; these are 11. Another instruction in the product's place needs this looked at again.
        const auto pin_s = [&]() { asm volatile("s_nop 10" : "+v"(s[0][0]), "+v"(s[0][1]), "+v"(s[1][0]), "+v"(s[1][1])); };
        const auto softmax_phase = [&]() {
            landed(h);
            phase_barrier();
            refill(h);
            softmax();
            asm volatile("" : "+v"(pf[0]), "+v"(pf[1]));
            phase_barrier();
            ++h;
        };
        if (plain > 0) {
            read_k(stage_of(0));
            first_product();
            pin_s();
            softmax_phase();
            while (h < plain) {
                read_v(stage_of(h - 1));
                __builtin_amdgcn_sched_barrier(0);
                second_product();
                read_k(stage_of(h));
                first_product();
                pin_s();
                pin_o();
                softmax_phase();
            }
            read_v(stage_of(h - 1));
            second_product();
        }
        // the others, with both products in their own step
        for (; h < steps; ++h) {
            MI355_LDS char* st = stage_of(h);
            const int key0 = key_of(h);
            const bool work = h / NH < n_loc && key0 <= lim_max;   // (the other half's last tile; keys that no column of the wave sees)
            if (work) {
                read_k(st);
                first_product();
                pin_s();
            }
            landed(h);
            phase_barrier();
            if (work) {
                const uint32_t none = none_of(h);
                const bool drafted = TREE && key0 + 32 > base;
                const uint32_t there = ~((none & 1 ? 0xffffu : 0u) | (none & 2 ? 0xffff0000u : 0u));   // (a word's)
                if (drafted) {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        const uint32_t mine = (seen(key0, qrow[nb]) & there) >> (4 * g);
#pragma unroll
                        for (int e = 0; e < 8; ++e) s[nb][e >> 2][e & 3] = mine & (1u << (16 * (e >> 2) + (e & 3))) ? s[nb][e >> 2][e & 3] : -INFINITY;
                    }
                } else {
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (key0 + 16 * (e >> 2) + 4 * g + (e & 3) > lim[nb] || ((none >> (e >> 2)) & 1)) s[nb][e >> 2][e & 3] = -INFINITY;
                }
                softmax();
                read_v(st);
                // A product with p = 0 is not nothing where v is infinite or NaN: such values are taken out and go to the rows that see them, one
                // after the other.
                bool finite;
                if constexpr (TREE) {   // (the matrix pipe asks: 0 * v is 0 but for those)
                    V8 zero;
#pragma unroll
                    for (int e = 0; e < 8; ++e) zero[e] = (T)0.f;
                    float4v sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int db = 0; db < 8; ++db) sum = Elem<T>::mfma16(vf[db], zero, sum);
                    finite = __builtin_amdgcn_ballot_w64(!(sum[0] == 0.f && sum[1] == 0.f && sum[2] == 0.f && sum[3] == 0.f)) == 0;
                } else {
                    ushort2v top = {0, 0};
#pragma unroll
                    for (int db = 0; db < 8; ++db) {
                        const int4v x = __builtin_bit_cast(int4v, vf[db]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) top = __builtin_elementwise_max(top, __builtin_bit_cast(ushort2v, x[e] & 0x7fff7fff));
                    }
                    finite = __builtin_amdgcn_ballot_w64(top[0] >= kInfinity || top[1] >= kInfinity) == 0;
                }
                if (!finite) {
#pragma unroll
                    for (int db = 0; db < 8; ++db)
#pragma unroll
                        for (int e = 0; e < 8; ++e) vf[db][e] = is_finite(vf[db][e]) ? vf[db][e] : (T)0.f;
                }
                second_product();
                if (!finite) {
#pragma unroll 1
                    for (int r = row_min; r <= row_max; ++r) {
                        const int last = r < n_new ? min(len - 1, r + len - n_new) : -1;
                        const uint32_t word = drafted ? (seen(key0, r) & there) >> (4 * g) : 0;
#pragma unroll
                        for (int db = 0; db < 8; ++db) {
                            V8 vs = v_frag(st, db);
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                const bool hidden = drafted ? !((word >> (16 * (e >> 2) + (e & 3))) & 1) : key0 + 16 * (e >> 2) + 4 * g + (e & 3) > last;
                                if (is_finite(vs[e]) || hidden || ((none >> (e >> 2)) & 1)) vs[e] = (T)0.f;
                            }
#pragma unroll
                            for (int nb = 0; nb < NB; ++nb) {
                                const float4v more = Elem<T>::mfma16(vs, pf[nb], float4v{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[nb][db][e] += qrow[nb] == r ? more[e] : 0.f;
                            }
                        }
                    }
                }
            }
            wait_lgkmcnt<0>();
            refill(h);
            phase_barrier();
        }
        if (wave < 4) phase_barrier();

        float l_tot[NB];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) l_tot[nb] = quad_sum(l_run[nb]);
        if constexpr (TREE) {
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
                if (lim[nb] < 0) {
                    m_run[nb] = -INFINITY;
                    l_tot[nb] = 0.f;
#pragma unroll
                    for (int db = 0; db < 8; ++db) o[nb][db] = float4v{0.f, 0.f, 0.f, 0.f};
                }
        }
        __syncthreads();   // the stages are free
        // The halves meet: the first one finishes the lower 16 columns of a wave, the second one the upper ones.
        constexpr int FINISHED = KG == 2 ? 1 : NB, COLUMN_FLOATS = 8 * 64 * 4 + 32;   // blocks of columns that a wave finishes; what a wave hands over
        if constexpr (KG == 2) {
            if (kg == 1) {
#pragma unroll
                for (int db = 0; db < 8; ++db) {
                    const float4v x = o[0][db];
                    o[0][db] = o[1][db];
                    o[1][db] = x;
                }
                const float m = m_run[0], l = l_tot[0];
                m_run[0] = m_run[1], l_tot[0] = l_tot[1], m_run[1] = m, l_tot[1] = l;
                qrow[0] = qrow[1];
            }
            MI355_LDS float* mine = (MI355_LDS float*)smem_raw + wave * COLUMN_FLOATS;
            MI355_LDS const float* theirs = (MI355_LDS const float*)smem_raw + (wave ^ CW) * COLUMN_FLOATS;
#pragma unroll
            for (int db = 0; db < 8; ++db) *(MI355_LDS float4v*)(mine + (db * 64 + lane) * 4) = o[1][db];
            if (g == 0) mine[8 * 256 + c16] = m_run[1], mine[8 * 256 + 16 + c16] = l_tot[1];
            __syncthreads();
            const float m1 = theirs[8 * 256 + c16], l1 = theirs[8 * 256 + 16 + c16];
            const float m = fmaxf(m_run[0], m1);
            // of a half that saw no key: its outputs and l are 0 (or NaN, which stays)
            const float w0 = m_run[0] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m_run[0] - m) * a.scale_log2);
            const float w1 = m1 == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m1 - m) * a.scale_log2);
            const auto meet = [&](float own, float other) {   // (the second half's share rounded first, on both sides)
                return kg == 0 ? __builtin_fmaf(w0, own, w1 * other) : __builtin_fmaf(w1, other, w0 * own);
            };
#pragma unroll
            for (int db = 0; db < 8; ++db) {
                const float4v x = *(MI355_LDS const float4v*)(theirs + (db * 64 + lane) * 4);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[0][db][e] = meet(o[0][db][e], x[e]);
            }
            l_tot[0] = meet(l_tot[0], l1);
            m_run[0] = m;
            __syncthreads();
        }
        if (whole || (!TREE && n == seq.tiles)) {
#pragma unroll
            for (int i = 0; i < FINISHED; ++i) {
                const int col = col0 + 16 * (KG == 2 ? kg : i) + c16;
                if (col >= a.ncols) continue;
                const int qi = qrow[i], hq = hkv * a.group + col - qi * a.group;
                const float inv = l_tot[i] != 0.f ? 1.f / l_tot[i] : 0.f;
                T* op = O + b * a.o_batch + (long)hq * a.o_head + qi * a.o_row + 4 * g;
#pragma unroll
                for (int db = 0; db < 8; ++db) {
                    V4 ov;
#pragma unroll
                    for (int e = 0; e < 4; ++e) ov[e] = (T)(o[i][db][e] * inv);
                    *(V4*)(op + 16 * db) = ov;
                }
                if (a.LSE != nullptr && g == 0)
                    a.LSE[((long)b * a.Hq + hq) * a.Sq + qi] = l_tot[i] != 0.f ? (m_run[i] * a.scale_log2 + __builtin_log2f(l_tot[i])) * 0.69314718055994531f : -INFINITY;
            }
        } else {
            float* part = a.part + ((long)(TREE ? part_number : 2 * blockIdx.x + (parts > 0)) * CW + cw) * PART_FLOATS;
#pragma unroll
            for (int i = 0; i < FINISHED; ++i) {
                const int nb = KG == 2 ? kg : i;
#pragma unroll
                for (int db = 0; db < 8; ++db) *(float4v*)(part + ((nb * 8 + db) * 64 + lane) * 4) = o[i][db];
                if (g == 0) part[NB * 8 * 256 + nb * 16 + c16] = m_run[i], part[NB * 8 * 256 + WCOLS + nb * 16 + c16] = l_tot[i];
            }
        }
        if constexpr (TREE) {
            if (a.direct || !take_piece()) return;
            continue;
        }
        if (whole) {
            f -= f_end;
            if (f < 0) return;
            take();
            continue;
        }
        f += units;
        if (units <= 0 || f >= f_end) return;   // (nothing done ends the walk even where lengths change under the call)
        ++parts;
        at = 0;
        if (++hkv == kv.Hkv) {
            hkv = 0;
            seq = entries.find(f);
        }
    }
}

// What is left behind paged_rows_kernel. Its first workgroups join the parts of the triples that were cut, O = sum_p w_p O~_p / sum_p w_p l_p with w_p =
// 2^((m_p - max m) c), a thread 4 d of a column: with few triples of many parts (a.few) four for each (triple, wave of columns), with many triples, of which only
// those between two workgroups' pieces are cut, one for each (border, wave of columns), of which that of a triple's first border does it (32 x 32 triples of
// 256 columns in 256 pieces: one workgroup or more a triple 74 us, a border 14). Then one per entry writes zeros where no key is seen.
template <typename T, int KG, bool TREE>
__global__ __launch_bounds__(256, TREE ? 3 : 1) void paged_rows_join_kernel(PagedKv kv, RowsAttn a) {
    using namespace prow;
    using V4 = typename Elem<T>::v4;
    constexpr int CW = WAVES / KG, COLS = CW * WCOLS;
    const int lane = threadIdx.x & 63, g = lane >> 4, c16 = lane & 15;
    Entries<COLS> entries(kv, a);
    const auto store = [&](int b, int hkv, int col, int d, float4v x, float lse) {
        const int qi = divide(col, a.by_group), hq = hkv * a.group + col - qi * a.group;
        V4 ov;
#pragma unroll
        for (int e = 0; e < 4; ++e) ov[e] = (T)x[e];
        *(V4*)((T*)a.O + b * a.o_batch + (long)hq * a.o_head + qi * a.o_row + d) = ov;
        if (a.LSE != nullptr && d == 0) a.LSE[((long)b * a.Hq + hq) * a.Sq + qi] = lse;
    };
    if ((int)blockIdx.x >= a.joins * CW) {
        if (blockIdx.y != 0) return;
        const int e = blockIdx.x - a.joins * CW, block = divide(e, a.by_batch), b = e - block * kv.B;
        if (entries.keys_of(e).keys != 0) return;
        const int ncols = min(COLS, a.ncols - block * COLS);
        for (int hkv = 0; hkv < kv.Hkv; ++hkv)
            for (int i = threadIdx.x; i < ncols * (D / 4); i += 256)
                store(b, hkv, block * COLS + (i >> 5), (i & 31) * 4, float4v{0.f, 0.f, 0.f, 0.f}, -INFINITY);
        return;
    }
    const int join = blockIdx.x / CW, cw = blockIdx.x % CW;
    int n, hkv, b, col0;
    const float *part0, *part1;   // its first part, and the one that stands in front of the others' places
    long stride = 2 * CW * PART_FLOATS;
    if constexpr (TREE) {
        const CutTriple cut = ((const CutTriple*)a.cuts)[1 + join];   // (requested together with how many there are)
        if (join >= *a.cuts || cut.pieces == 0) return;
        const int block = divide(cut.triple, a.by_hkv);
        n = cut.pieces, b = cut.b, hkv = cut.triple - block * kv.Hkv, col0 = block * COLS + cw * WCOLS;
        if (col0 >= a.ncols) return;
        stride = CW * PART_FLOATS;
        part0 = part1 = a.part + ((long)cut.part0 * CW + cw) * PART_FLOATS;
    } else {
        const auto sum = entries.sum();
        if (entries.in_turn(sum)) return;
        const int total = sum.total, quota = entries.quota(sum);
        typename Entries<COLS>::Where seq;
        if (a.few) {   // a triple
            const int e = divide(join, a.by_hkv);
            hkv = join - e * kv.Hkv;
            seq = entries.at(e);
            if (seq.units == 0) return;
        } else {       // a border
            if (join == 0 || join * quota >= total) return;
            seq = entries.find(join * quota);
            if (seq.units == 0) return;
            hkv = (int)((uint32_t)(join * quota - seq.before * kv.Hkv) / (uint32_t)seq.units);
        }
        const int f0 = seq.before * kv.Hkv + hkv * seq.units, first = (int)((uint32_t)(f0 + Entries<COLS>::HEAD) / (uint32_t)quota);
        n = (int)((uint32_t)(f0 + seq.units - 1) / (uint32_t)quota) - first + 1;   // (workgroups that have tiles of it)
        if (n == 1 || (!a.few && first != join - 1)) return;
        const int block = divide(seq.e, a.by_batch);
        b = seq.e - block * kv.B, col0 = block * COLS + cw * WCOLS;
        if (col0 >= a.ncols) return;
        // its part is the last of the first workgroup (unless that begins inside it) and the first of the others
        part0 = a.part + ((long)(2 * first + (first * quota < f0)) * CW + cw) * PART_FLOATS;
        part1 = a.part + ((long)(2 * first) * CW + cw) * PART_FLOATS;
    }
    const auto part_of = [&](int p) { return p == 0 ? part0 : part1 + (long)p * stride; };
    const auto weight = [&](float x, float ref) { return x == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((x - ref) * a.scale_log2); };
    for (int quarter = blockIdx.y; quarter < 4; quarter += gridDim.y) {
        const int nb = quarter >> 1, db = (quarter & 1) * 4 + (threadIdx.x >> 6);
        float m = -INFINITY, l = 0.f;
        float4v acc = float4v{0.f, 0.f, 0.f, 0.f};
        constexpr int ROUND = 8;   // parts in flight
        for (int p0 = 0; p0 < n; p0 += ROUND) {
            float4v v[ROUND];
            float mp[ROUND], lp[ROUND];
#pragma unroll
            for (int r = 0; r < ROUND; ++r) {
                mp[r] = -INFINITY;
                if (r > 1 && p0 + r >= n) continue;   // (a round has two parts at least, one of them again where the last is alone)
                const float* part = part_of(min(p0 + r, n - 1));
                v[r] = *(const float4v*)(part + ((nb * 8 + db) * 64 + lane) * 4);
                mp[r] = part[NB * 8 * 256 + nb * 16 + c16];
                lp[r] = part[NB * 8 * 256 + WCOLS + nb * 16 + c16];
            }
            float m_new = m;
#pragma unroll
            for (int r = 0; r < ROUND; ++r) m_new = fmaxf(m_new, mp[r]);
            const float keep = weight(m, m_new);
            l *= keep;
            acc *= keep;
            m = m_new;
#pragma unroll
            for (int r = 0; r < ROUND; ++r) {
                if (p0 + r >= n) break;
                const float w = weight(mp[r], m);
                l += w * lp[r];
                acc += w * v[r];
            }
        }
        const int col = col0 + 16 * nb + c16;
        if (col >= a.ncols) continue;
        const float inv = l != 0.f ? 1.f / l : 0.f;
        store(b, hkv, col, 16 * db + 4 * g, acc * inv, l != 0.f ? (m * a.scale_log2 + __builtin_log2f(l)) * 0.69314718055994531f : -INFINITY);
    }
}

namespace prow {
struct Plan {
    int kg, blocks, direct, workgroups;
    long units;    // of all triples, at most
    size_t bytes;
};
static Plan plan_of(const mi355_paged_kv& c, int Hq, int Sq, bool tree) {
    Plan p;
    const int ncols = Hq / c.Hkv * Sq, max_len = c.max_pages * c.page_size;
    const long pairs = (long)c.B * c.Hkv;
    // us, one half of 256 columns / two of 128: 2048 rows of 32/8 heads over 8191 keys 297 / 303, 8 x 512 rows over 2048 175 / 181; 512 rows over 8191 106 / 103,
    // 8 x 128 rows over 1024 58 / 54, 300 rows of 32/32 heads over 2000 49 / 44 (columns that are not there)
    p.kg = ncols > 128 && pairs * ncols >= kWholeColumns ? 1 : 2;
    const int cols = 256 / p.kg, tk = 64 / p.kg;
    p.blocks = (ncols + cols - 1) / cols;
    p.units = pairs * p.blocks * ((max_len + tk - 1) / tk + kHeadKeys / tk);
    // us, a workgroup a triple / cut: 500 rows over 500 keys 18 / 73, 8 x 1024 rows over 2048 247 / 288, one sequence (whose triples are of nearly one
    // length) of 2048 rows over 8191 300 / 320, of 1000 rows over 2000 42.7 / 58.5
    const long triples = pairs * p.blocks, rounds = (triples + kWorkgroups - 1) / kWorkgroups;
    p.direct = max_len <= kDirectLen || triples >= kDirectTriples || (c.B == 1 && 10 * triples >= 9 * rounds * kWorkgroups) || (tree && c.B > 64);   // (Pieces)
    p.workgroups = p.direct ? (int)triples : (int)std::min<long>(kWorkgroups, p.units / (kMinKeys / tk) + 1);
    p.bytes = p.direct ? 0 : sizeof(float) * 2 * (size_t)p.workgroups * (WAVES / p.kg) * PART_FLOATS;
    return p;
}
}  // namespace prow

bool paged_rows_fits(const mi355_paged_kv& c, int Hq, int Sq) { return prow::plan_of(c, Hq, Sq, false).units <= INT32_MAX - 65536; }

size_t paged_rows_workspace(const mi355_paged_kv& c, int Hq, int Sq, bool tree) {
    const size_t bytes = prow::plan_of(c, Hq, Sq, tree).bytes;
    return bytes + (bytes > 0 && tree ? prow::kCutBytes : 0);
}

template <typename T, int KG, bool TREE>
static hipError_t launch_rows(const PagedKv& kv, const RowsAttn& a, hipStream_t stream) {
    using namespace prow;
    static DynamicLdsOnce once;
    hipError_t e = once.ensure(reinterpret_cast<const void*>(paged_rows_kernel<T, KG, TREE>), LDS_BYTES);
    if (e != hipSuccess) return e;
    paged_rows_kernel<T, KG, TREE><<<dim3(a.workgroups), dim3(NTHREADS), LDS_BYTES, stream>>>(kv, a);
    e = hipGetLastError();
    if (e != hipSuccess || a.direct) return e;
    paged_rows_join_kernel<T, KG, TREE><<<dim3((unsigned)(a.joins * (WAVES / KG) + a.entries), a.few ? 4 : 1), dim3(256), 0, stream>>>(kv, a);
    return hipGetLastError();
}

hipError_t paged_rows_dispatch(const mi355_paged_kv& c, const void* Q, void* O, float* LSE, int Hq, int Sq, const long* strides, float scale,
                               const int* parents, long parents_batch, void* workspace, hipStream_t stream) {
    const PagedKv kv = paged_from(c);
    const prow::Plan p = prow::plan_of(c, Hq, Sq, parents != nullptr);
    RowsAttn a = {};
    a.Q = Q;
    a.O = O;
    a.LSE = LSE;
    a.part = (float*)workspace;
    a.q_batch = strides[0], a.q_head = strides[1], a.q_row = strides[2];
    a.o_batch = strides[3], a.o_head = strides[4], a.o_row = strides[5];
    a.Hq = Hq;
    a.Sq = Sq;
    a.group = Hq / kv.Hkv;
    a.ncols = a.group * Sq;
    a.entries = p.blocks * kv.B;
    a.workgroups = p.workgroups;
    a.direct = p.direct;
    a.blocks = p.blocks;
    if (parents != nullptr && !a.direct) {
        a.cuts = (int*)workspace;
        a.part = (float*)((char*)workspace + prow::kCutBytes);
    }
    a.few = (long)a.entries * kv.Hkv <= a.workgroups / 2;
    a.joins = a.few || parents != nullptr ? std::min(a.entries * kv.Hkv, a.workgroups) : a.workgroups;
    a.tree = {parents, parents_batch};
    a.scale_log2 = scale * 1.4426950408889634f;
    a.by_group = divisor_of(a.group);
    a.by_batch = divisor_of(kv.B);
    a.by_hkv = divisor_of(kv.Hkv);
    const auto launch = [&](auto type, auto tree) {
        using T = decltype(type);
        return p.kg == 1 ? launch_rows<T, 1, decltype(tree)::value>(kv, a, stream) : launch_rows<T, 2, decltype(tree)::value>(kv, a, stream);
    };
    if (parents != nullptr) return c.dtype == MI355_DTYPE_BF16 ? launch(bf16_t{}, std::true_type{}) : launch(half_t{}, std::true_type{});
    return c.dtype == MI355_DTYPE_BF16 ? launch(bf16_t{}, std::false_type{}) : launch(half_t{}, std::false_type{});
}

}  // namespace mi355
