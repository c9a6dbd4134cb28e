// The tensors of a key-value cache in pages as torch operators take them, checked and put into the C ABI's mi355_paged_kv. Host code, shared by
// the operator modules.
#pragma once
#include <torch/extension.h>

#include <optional>

#include "mi355_serving.h"

namespace mi355 {

inline void check_like(const char* name, const char* what, const at::Tensor& t, const at::Tensor& like, at::ScalarType type) {
    TORCH_CHECK(t.is_cuda() && t.device() == like.device(), name, ": ", what, " must be a GPU tensor on the device of kv_pages");
    TORCH_CHECK(t.scalar_type() == type, name, ": ", what, " must be ", type, ", got ", t.scalar_type());
}

// The pool alone: what calls that go by slots take
inline mi355_paged_kv paged_pool(const char* name, const at::Tensor& kv_pages, const std::optional<at::Tensor>& weights, const std::optional<at::Tensor>& key_positions) {
    TORCH_CHECK(kv_pages.dim() == 4 && kv_pages.size(3) == 128 && kv_pages.size(1) % 2 == 0 && kv_pages.numel() > 0, name,
                ": kv_pages must be [n_pages, 2 * Hkv, page_size, 128], got ", kv_pages.sizes());
    const bool bf16 = kv_pages.scalar_type() == at::kBFloat16;
    TORCH_CHECK(kv_pages.scalar_type() == at::kHalf || bf16, name, ": kv_pages must be float16 or bfloat16, got ", kv_pages.scalar_type());
    TORCH_CHECK(kv_pages.stride(3) == 1, name, ": the last dimension of kv_pages must be contiguous");
    TORCH_CHECK(kv_pages.is_cuda(), name, ": kv_pages must be a GPU tensor");
    const int64_t Hkv = kv_pages.size(1) / 2;
    const auto account = [&](const std::optional<at::Tensor>& t, const char* what, at::ScalarType type) -> void* {
        if (!t.has_value()) return nullptr;
        check_like(name, what, *t, kv_pages, type);
        TORCH_CHECK(t->dim() == 3 && t->size(0) == kv_pages.size(0) && t->size(1) == Hkv && t->size(2) == kv_pages.size(2) && t->is_contiguous(), name, ": ", what,
                    " must be a contiguous [", kv_pages.size(0), ", ", Hkv, ", ", kv_pages.size(2), "] tensor, got ", t->sizes());
        return t->data_ptr();
    };
    TORCH_CHECK(kv_pages.size(0) <= INT32_MAX && kv_pages.size(2) <= INT32_MAX && Hkv <= INT32_MAX, name, ": dimension exceeds int32");
    mi355_paged_kv c = {};
    c.pages = kv_pages.data_ptr();
    c.weights = static_cast<float*>(account(weights, "weights", at::kFloat));
    c.key_positions = static_cast<int32_t*>(account(key_positions, "key_positions", at::kInt));
    // (a dimension of one element may have any stride)
    c.row_stride = kv_pages.size(2) > 1 ? kv_pages.stride(2) : 128;
    c.head_stride = kv_pages.stride(1);
    c.page_stride = kv_pages.size(0) > 1 ? kv_pages.stride(0) : 128;
    c.n_pages = (int32_t)kv_pages.size(0);
    c.page_size = (int32_t)kv_pages.size(2);
    c.Hkv = (int32_t)Hkv;
    c.dtype = bf16 ? MI355_DTYPE_BF16 : MI355_DTYPE_FP16;
    return c;
}

inline mi355_paged_kv paged_kv(const char* name, const at::Tensor& kv_pages, const at::Tensor& block_table, const at::Tensor& seq_lens,
                        const std::optional<at::Tensor>& new_lens, const std::optional<at::Tensor>& weights, const std::optional<at::Tensor>& key_positions) {
    TORCH_CHECK(block_table.dim() == 2 && block_table.numel() > 0, name, ": block_table must be [B, max_pages], got ", block_table.sizes());
    mi355_paged_kv c = paged_pool(name, kv_pages, weights, key_positions);
    const int64_t B = block_table.size(0);
    check_like(name, "block_table", block_table, kv_pages, at::kInt);
    TORCH_CHECK(block_table.stride(1) == 1 || block_table.size(1) == 1, name, ": the rows of block_table must be contiguous");
    TORCH_CHECK(block_table.size(1) <= INT32_MAX && B <= INT32_MAX, name, ": dimension exceeds int32");
    const auto lengths = [&](const at::Tensor& t, const char* what) {
        check_like(name, what, t, kv_pages, at::kInt);
        TORCH_CHECK(t.dim() == 1 && t.size(0) == B && t.is_contiguous(), name, ": ", what, " must be a contiguous [", B, "] tensor, got ", t.sizes());
        return t.data_ptr<int32_t>();
    };
    c.block_table = block_table.data_ptr<int32_t>();
    c.seq_lens = lengths(seq_lens, "seq_lens");
    c.new_lens = new_lens.has_value() ? lengths(*new_lens, "new_lens") : nullptr;
    c.table_stride = block_table.stride(0);
    c.max_pages = (int32_t)block_table.size(1);
    c.B = (int32_t)B;
    return c;
}

}  // namespace mi355
