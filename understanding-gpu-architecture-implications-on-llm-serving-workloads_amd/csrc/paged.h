// What the kernels of the paged key-value cache share: where a key lies, and how the lengths of a batch are read.
//
// A cache is a pool of pages, each [2 Hkv heads][page_size rows][128] with strides of its own (key heads in front of value heads).
// Key j of sequence b is row j % page_size of page block_table[b][j / page_size]. page_size is a multiple of 16, so 16 keys that
// begin at a multiple of 16 lie in one page. Entries of the block table outside [0, n_pages) hold no keys: they are masked where
// keys are read and skipped where something is written, so a wrong table gives wrong results but no access outside the pool.
// Lengths are read on the device and cut to [0, max_pages * page_size]; a launch's grid depends on what the host knows alone, so that a
// captured call serves whatever lengths its tensors hold when it is replayed.
#pragma once
#include "mi355_common.h"
#include "mi355_serving_internal.h"

namespace mi355 {

// mi355_paged_kv as the kernels take it
struct PagedKv {
    char* pages;
    long page_bytes, head_bytes;
    uint32_t row_bytes;
    const int* table;
    long table_stride;
    const int* seq_lens;
    const int* new_lens;   // nullptr: all rows are tokens
    float* weights;        // [n_pages][Hkv][page_size] or nullptr
    int* key_positions;    // likewise
    int B, Hkv, n_pages, page_size, max_pages, max_len;
    Divisor by_page;
};

inline PagedKv paged_from(const mi355_paged_kv& c) {
    PagedKv p;
    p.pages = (char*)c.pages;
    p.page_bytes = (long)c.page_stride * 2;
    p.head_bytes = (long)c.head_stride * 2;
    p.row_bytes = (uint32_t)(c.row_stride * 2);
    p.table = c.block_table;
    p.table_stride = (long)c.table_stride;
    p.seq_lens = c.seq_lens;
    p.new_lens = c.new_lens;
    p.weights = c.weights;
    p.key_positions = c.key_positions;
    p.B = c.B;
    p.Hkv = c.Hkv;
    p.n_pages = c.n_pages;
    p.page_size = c.page_size;
    p.max_pages = c.max_pages;
    p.max_len = c.max_pages * c.page_size;
    p.by_page = divisor_of(c.page_size);
    return p;
}

// keys of sequence b, those of this call's tokens among them
__device__ __forceinline__ int paged_len(const PagedKv& kv, int b) { return min(max(kv.seq_lens[b], 0), kv.max_len); }
// how many of its S rows are tokens
__device__ __forceinline__ int paged_new(const PagedKv& kv, int b, int S) {
    return kv.new_lens == nullptr ? S : min(max(kv.new_lens[b], 0), S);
}

// inclusive sum over each 16 lanes of a wave, and over all of them (row shifts inside 16 lanes, then the rows' sums are handed on: 6 additions, no LDS)
__device__ __forceinline__ int row_inclusive_sum(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);   // row_shr:1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);   // row_shr:2
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);   // row_shr:4
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);   // row_shr:8
    return x;
}
__device__ __forceinline__ int wave_inclusive_sum(int x) {
    x = row_inclusive_sum(x);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
    return x;
}
// the largest value up to this lane
__device__ __forceinline__ int wave_running_max(int x) {
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x111, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x112, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x114, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x118, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x142, 0xa, 0xf, false));
    return max(x, __builtin_amdgcn_update_dpp(x, x, 0x143, 0xc, 0xf, false));
}
// the largest of the first 16 lanes' values, and of all lanes', in every lane (likewise)
__device__ __forceinline__ int row_running_max(int x) {
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x111, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x112, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x114, 0xf, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x118, 0xf, 0xf, false));
    return x;
}
__device__ __forceinline__ int row_max(int x) { return __builtin_amdgcn_readlane(row_running_max(x), 15); }
__device__ __forceinline__ int wave_max(int x) {
    x = row_running_max(x);
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x142, 0xa, 0xf, false));
    x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x143, 0xc, 0xf, false));
    return __builtin_amdgcn_readlane(x, 63);
}

// ---- a tree of drafted tokens -----------------------------------------------------------------------------------------
//
// The last n keys of a sequence are drafted tokens, of which token i continues parents[i], 0 <= parents[i] < i, or is a root (anything else). It sees the keys
// in front of the draft, itself and the tokens on its path to a root; none of them lies behind it. What a row sees of 32 keys that begin at a multiple of 32 is
// a word of bits; the words of a row begin with the one that holds the draft's first key, whose lower bits are keys in front of the draft.
struct PagedTree {
    const int* parents;
    long batch;      // entries from one sequence's parents to the next's (0: the same for all)
};
constexpr int kTreeWords = kMostDrafted / 32 + 1;   // (odd: rows side by side in LDS lie in different banks)

// The words of drafted token `row` of n, of which the first is key `base` (negative where the sequence is shorter than its draft: the first ones are no keys).
// `parents` in LDS. Every step of the walk goes to a smaller number; the last token of a chain walks all of them. us, steps back by 1 .. 8 / a chain: 26 tokens over 300 keys 9.3 /
// 11.5, 64 over 8191 28.7 / 33.2, 256 over 8191 56 / 77, 32 of 32 sequences of up to 4097 80.8 / 81.7.
__device__ __forceinline__ void tree_words(MI355_LDS const int* parents, int row, int n, int base, MI355_LDS uint32_t* words) {
    const int skew = base >= 0 ? base & 31 : base;
#pragma unroll
    for (int w = 0; w < kTreeWords; ++w) words[w] = 0;
    if (row < 0 || row >= n) return;
    if (base > 0) words[0] = (1u << skew) - 1;
    for (int i = row; i >= 0;) {
        if (skew + i >= 0) words[(skew + i) >> 5] |= 1u << ((skew + i) & 31);
        const int up = parents[i];
        i = up < i ? up : -1;
    }
}

}  // namespace mi355
