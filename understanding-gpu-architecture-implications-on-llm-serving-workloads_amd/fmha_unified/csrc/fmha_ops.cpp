// PyTorch operator layer of fmha_unified for MI355X.
//
// Same operator surface as the reference (kernels/fmha/pkg/fmha_unified/csrc/fmha_kernel.cpp:9-18): schemas
// `fmha_unified::finefmha_0 .. finefmha_7 (Tensor q, Tensor k, Tensor v, bool causal, bool is_decode,
// int decode_length) -> Tensor`, CUDA dispatch key, empty `_C` module. Every index runs the one gfx950
// attention kernel of libmi355_serving.so, for float16 or bfloat16 tensors. Host checks mirror
// semi/fmha_2_amd.cpp:322-333 (dtype, d == 128,
// is_decode implies !causal) and add the shape checks the reference omits.
//
// One operator is added without touching the reference's schemas:
//   `finefmha_fwd_lse(q, k, v, causal, is_decode, decode_length) -> (Tensor out, Tensor lse)`
// which also returns the log-sum-exp [B, Hq, Sq] in fp32 (the reference has no LSE output).
//
// decode_length is the number of valid keys (ops.py:18 passes the un-padded k.size(2)); keys at or beyond it
// are masked. The reference masks `k > decode_length` (fmha_2_amd.cpp:191), which lets the first padded key
// through; that off-by-one is not reproduced.
#include <torch/extension.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <optional>
#include <string>
#include <tuple>

#include "mi355_serving.h"
#include "../../csrc/paged_tensors.h"

namespace fmha_unified {

namespace {

using mi355::check_like;
using mi355::paged_kv;

// an uninitialised GPU tensor, without a trip through the dispatcher (0.4 us)
at::Tensor gpu_empty(at::IntArrayRef size, at::ScalarType type, const at::Tensor& like) {
    return at::Tensor(at::detail::empty_cuda(size, type, like.device(), std::nullopt));
}

// A [B, H, S, D] view the kernels can read in place: contiguous last dimension, every other stride a non-negative
// multiple of 8 elements, 16-byte aligned base. This covers `x.view(B, S, H, D).transpose(1, 2)` and slices of a fused
// QKV projection, the forms the reference's in-model caller produces (benchmarks/flashattn-cuda/modeling_llama.py:658-660)
// and which kernels/fmha/pkg/fmha_unified/ops.py:23-25 copies into contiguous tensors first.
bool readable_in_place(const at::Tensor& t) {
    if (t.stride(3) != 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0) return false;
    for (int i = 0; i < 3; ++i)
        if (t.stride(i) < 0 || t.stride(i) % 8 != 0) return false;
    return true;
}

std::tuple<at::Tensor, at::Tensor> run_fmha(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, bool causal,
                                            bool is_decode, int64_t decode_length, bool want_lse) {
    const char* name = "finefmha";
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && v.dim() == 4, name, ": q, k, v must be [B, H, S, D] tensors");
    const bool bf16 = q.scalar_type() == at::kBFloat16;  // the dtype of the reference's finefmha_5 (manual/fmha_5_nv.cu:148-150)
    TORCH_CHECK(q.scalar_type() == at::kHalf || bf16, name, ": q must be float16 or bfloat16, got ", q.scalar_type());
    TORCH_CHECK(k.scalar_type() == q.scalar_type(), name, ": k must have q's dtype ", q.scalar_type(), ", got ", k.scalar_type());
    TORCH_CHECK(v.scalar_type() == q.scalar_type(), name, ": v must have q's dtype ", q.scalar_type(), ", got ", v.scalar_type());
    const int64_t B = q.size(0), Hq = q.size(1), Sq = q.size(2), D = q.size(3);
    const int64_t Hkv = k.size(1), Sk = k.size(2);
    TORCH_CHECK(D == 128, name, ": head embedding dimension must be 128, got ", D);
    TORCH_CHECK(k.size(0) == B && k.size(3) == D, name, ": k shape does not match q");
    TORCH_CHECK(v.sizes() == k.sizes(), name, ": v shape must equal k shape");
    TORCH_CHECK(B >= 1 && Hq >= 1 && Hkv >= 1 && Sq >= 1 && Sk >= 1, name, ": empty tensors are not supported");
    TORCH_CHECK(Hq % Hkv == 0, name, ": number of q heads (", Hq, ") must be a multiple of kv heads (", Hkv, ")");
    TORCH_CHECK(!(is_decode && causal), name, ": causal is not supported in decode mode");
    TORCH_CHECK(decode_length >= 1 && decode_length <= Sk, name, ": decode_length ", decode_length,
                " outside [1, k.size(2) = ", Sk, "]");
    TORCH_CHECK(Sq <= INT32_MAX && Sk <= INT32_MAX && B <= INT32_MAX && Hq <= INT32_MAX, name, ": dimension exceeds int32");
    TORCH_CHECK(q.is_cuda() && k.is_cuda() && v.is_cuda(), name, ": q, k, v must be GPU tensors");
    TORCH_CHECK(q.device() == k.device() && q.device() == v.device(), name, ": q, k, v are on different devices");

    // torch on ROCm presents HIP devices under the "cuda" device type; these are its guard and stream for them
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
    at::Tensor qc = readable_in_place(q) ? q : q.contiguous();
    at::Tensor kc = readable_in_place(k) ? k : k.contiguous();
    at::Tensor vc = readable_in_place(v) ? v : v.contiguous();
    // The result is a freshly allocated contiguous [B, H, S, D] tensor whatever the strides of q, as in the reference
    // (`zeros_like` of a `.contiguous()` input, semi/fmha_2_amd.cpp:336; kernels/fmha/pkg/fmha_unified/ops.py:23-29), so
    // callers may `.view()` it. empty() instead of zeros(): the kernel writes every element.
    at::Tensor o = gpu_empty(qc.sizes(), qc.scalar_type(), qc);
    at::Tensor lse;
    float* lse_ptr = nullptr;
    if (want_lse) {
        lse = gpu_empty({B, Hq, Sq}, at::kFloat, qc);
        lse_ptr = lse.data_ptr<float>();
    }
    const float scale = 1.0f / std::sqrt(static_cast<float>(D));  // fmha_2_amd.cpp:320
    hipStream_t stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream();
    const int64_t strides[12] = {qc.stride(0), qc.stride(1), qc.stride(2), kc.stride(0), kc.stride(1), kc.stride(2),
                                 vc.stride(0), vc.stride(1), vc.stride(2), o.stride(0),  o.stride(1),  o.stride(2)};
    auto entry = bf16 ? &mi355_fmha_fwd_bf16 : &mi355_fmha_fwd_strided;
    int rc = entry(qc.data_ptr(), kc.data_ptr(), vc.data_ptr(), o.data_ptr(), lse_ptr, (int)B, (int)Hq, (int)Hkv, (int)Sq,
                   (int)Sk, (int)D, scale, causal ? 1 : 0, (int)decode_length, strides, stream);
    TORCH_CHECK(rc == 0, name, ": ", mi355_last_error(), " (code ", rc, ")");
    return {o, lse};
}

at::Tensor finefmha(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, bool causal, bool is_decode,
                    int64_t decode_length) {
    return std::get<0>(run_fmha(q, k, v, causal, is_decode, decode_length, false));
}

std::tuple<at::Tensor, at::Tensor> finefmha_fwd_lse(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                    bool causal, bool is_decode, int64_t decode_length) {
    return run_fmha(q, k, v, causal, is_decode, decode_length, true);
}

// ---- a key-value cache in pages (include/mi355_serving.h: mi355_paged_kv) -----------------------------------------------

// batch, head and row stride of [B, H, S, 128] queries; of a dimension of one element it may be anything and is not used
std::array<int64_t, 3> query_strides(const at::Tensor& q) {
    return {q.size(0) > 1 ? q.stride(0) : 0, q.size(1) > 1 ? q.stride(1) : 0, q.size(2) > 1 ? q.stride(2) : 128};
}

// queries [B, Hq, S, 128] of the pages' type and device
at::Tensor paged_queries(const char* name, const at::Tensor& q, const at::Tensor& kv_pages, const mi355_paged_kv& c) {
    TORCH_CHECK(q.dim() == 4 && q.size(0) == c.B && q.size(3) == 128 && q.numel() > 0, name, ": q must be [", c.B, ", Hq, S, 128], got ", q.sizes());
    check_like(name, "q", q, kv_pages, kv_pages.scalar_type());
    TORCH_CHECK(q.size(1) <= INT32_MAX && q.size(2) <= INT32_MAX, name, ": dimension exceeds int32");
    const auto st = query_strides(q);
    const bool in_place = q.stride(3) == 1 && reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0 && st[0] >= 0 && st[1] >= 0 && st[2] >= 0 &&
                          (st[0] | st[1] | st[2]) % 8 == 0 && st[2] < (1 << 24);
    return in_place ? q : q.clone(at::MemoryFormat::Contiguous);   // (contiguous() would hand back a contiguous tensor at an odd address)
}

at::Tensor workspace_of(size_t bytes, const at::Tensor& like) {
    return bytes > 0 ? gpu_empty({static_cast<int64_t>(bytes)}, at::kByte, like) : at::Tensor();
}

std::tuple<at::Tensor, at::Tensor> run_paged(const at::Tensor& q, const at::Tensor& kv_pages, const at::Tensor& block_table, const at::Tensor& seq_lens,
                                             const std::optional<at::Tensor>& new_lens, const std::optional<at::Tensor>& weights, bool want_lse) {
    const char* name = "finefmha_paged";
    const mi355_paged_kv c = paged_kv(name, kv_pages, block_table, seq_lens, new_lens, weights, std::nullopt);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(kv_pages.device());
    const at::Tensor qc = paged_queries(name, q, kv_pages, c);
    const int64_t Hq = q.size(1), S = q.size(2);
    at::Tensor o = gpu_empty(q.sizes(), q.scalar_type(), q), lse;
    if (want_lse) lse = gpu_empty({c.B, Hq, S}, at::kFloat, q);
    const size_t need = mi355_fmha_paged_workspace_bytes(&c, (int)Hq, (int)S, want_lse ? 1 : 0);
    const at::Tensor ws = workspace_of(need, q);
    const auto st = query_strides(qc);
    const int64_t strides[6] = {st[0], st[1], st[2], o.stride(0), o.stride(1), o.stride(2)};
    hipStream_t stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream();
    const int rc = mi355_fmha_paged(&c, qc.data_ptr(), o.data_ptr(), want_lse ? lse.data_ptr<float>() : nullptr, (int)Hq, (int)S, strides,
                                    1.0f / std::sqrt(128.0f), need > 0 ? ws.data_ptr() : nullptr, need, stream);
    TORCH_CHECK(rc == 0, name, ": ", mi355_last_error(), " (code ", rc, ")");
    return {o, lse};
}

at::Tensor finefmha_paged(const at::Tensor& q, const at::Tensor& kv_pages, const at::Tensor& block_table, const at::Tensor& seq_lens,
                          const std::optional<at::Tensor>& new_lens, const std::optional<at::Tensor>& weights) {
    return std::get<0>(run_paged(q, kv_pages, block_table, seq_lens, new_lens, weights, false));
}

std::tuple<at::Tensor, at::Tensor> finefmha_paged_lse(const at::Tensor& q, const at::Tensor& kv_pages, const at::Tensor& block_table,
                                                      const at::Tensor& seq_lens, const std::optional<at::Tensor>& new_lens,
                                                      const std::optional<at::Tensor>& weights) {
    return run_paged(q, kv_pages, block_table, seq_lens, new_lens, weights, true);
}

void rope_paged(const at::Tensor& qkv, const at::Tensor& kv_pages, const at::Tensor& block_table, const at::Tensor& seq_lens, const at::Tensor& cos,
                const at::Tensor& sin, const at::Tensor& positions, int64_t q_heads, const std::optional<at::Tensor>& new_lens,
                const std::optional<at::Tensor>& weights, const std::optional<at::Tensor>& key_positions, bool keep_keys) {
    const char* name = "fine_rope_paged";
    const mi355_paged_kv c = paged_kv(name, kv_pages, block_table, seq_lens, new_lens, weights, key_positions);
    TORCH_CHECK(q_heads >= 0 && qkv.dim() == 4 && qkv.size(0) == c.B && qkv.size(2) == q_heads + 2 * (int64_t)c.Hkv && qkv.size(3) == 128 && qkv.numel() > 0, name,
                ": qkv must be [", c.B, ", S, ", q_heads + 2 * (int64_t)c.Hkv, ", 128], got ", qkv.sizes());
    check_like(name, "qkv", qkv, kv_pages, kv_pages.scalar_type());
    TORCH_CHECK(qkv.stride(3) == 1 && qkv.stride(2) == 128, name, ": the heads of a token of qkv must lie side by side");
    const int64_t B = c.B, S = qkv.size(1);
    for (const at::Tensor* t : {&cos, &sin}) {
        check_like(name, "cos and sin", *t, kv_pages, at::kFloat);
        TORCH_CHECK(t->dim() == 2 && t->size(0) >= 1 && t->size(1) == 64 && t->is_contiguous() && t->sizes() == cos.sizes(), name,
                    ": cos and sin must be contiguous [n_positions, 64] tensors");
    }
    check_like(name, "positions", positions, kv_pages, at::kInt);
    TORCH_CHECK(positions.is_contiguous() && ((positions.dim() == 2 && positions.size(0) == B && positions.size(1) == S) ||
                                              (positions.dim() == 1 && positions.size(0) == S)), name, ": positions must be a contiguous [", B, ", ", S, "] or [", S,
                "] tensor, got ", positions.sizes());
    TORCH_CHECK(S <= INT32_MAX && q_heads <= INT32_MAX && cos.size(0) <= INT32_MAX, name, ": dimension exceeds int32");
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(kv_pages.device());
    hipStream_t stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream();
    const int64_t row = S > 1 ? qkv.stride(1) : (q_heads + 2 * (int64_t)c.Hkv) * 128;
    const int rc = mi355_rope_paged(&c, qkv.data_ptr(), (int)S, (int)q_heads, keep_keys ? 1 : 0, B > 1 ? qkv.stride(0) : 0, row, cos.data_ptr<float>(),
                                    sin.data_ptr<float>(), positions.data_ptr<int32_t>(), positions.dim() == 2 ? S : 0, (int)cos.size(0), stream);
    TORCH_CHECK(rc == 0, name, ": ", mi355_last_error(), " (code ", rc, ")");
}

void key_weights(const at::Tensor& q, const at::Tensor& lse, const at::Tensor& kv_pages, const at::Tensor& block_table, const at::Tensor& seq_lens,
                 const at::Tensor& weights, const std::optional<at::Tensor>& new_lens, int64_t last_rows) {
    const char* name = "fine_key_weights";
    const mi355_paged_kv c = paged_kv(name, kv_pages, block_table, seq_lens, new_lens, weights, std::nullopt);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(kv_pages.device());
    const at::Tensor qc = paged_queries(name, q, kv_pages, c);
    const int64_t Hq = q.size(1), S = q.size(2);
    check_like(name, "lse", lse, kv_pages, at::kFloat);
    TORCH_CHECK(lse.dim() == 3 && lse.size(0) == c.B && lse.size(1) == Hq && lse.size(2) == S && lse.is_contiguous(), name, ": lse must be a contiguous [", c.B, ", ",
                Hq, ", ", S, "] tensor, got ", lse.sizes());
    TORCH_CHECK(last_rows >= 0, name, ": last_rows must not be negative, got ", last_rows);
    const int last = (int)std::min<int64_t>(last_rows, INT32_MAX);
    const size_t need = mi355_fmha_key_weights_workspace_bytes(&c, (int)Hq, (int)S, last);
    const at::Tensor ws = workspace_of(need, q);
    const auto strides = query_strides(qc);
    hipStream_t stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream();
    const int rc = mi355_fmha_key_weights(&c, qc.data_ptr(), lse.data_ptr<float>(), (int)Hq, (int)S, strides.data(), last, 1.0f / std::sqrt(128.0f),
                                          need > 0 ? ws.data_ptr() : nullptr, need, stream);
    TORCH_CHECK(rc == 0, name, ": ", mi355_last_error(), " (code ", rc, ")");
}

at::Tensor evict_paged(const at::Tensor& kv_pages, const at::Tensor& block_table, const at::Tensor& seq_lens, const at::Tensor& weights,
                       const at::Tensor& key_positions, int64_t budget, int64_t recent) {
    const char* name = "fine_evict_paged";
    const mi355_paged_kv c = paged_kv(name, kv_pages, block_table, seq_lens, std::nullopt, weights, key_positions);
    TORCH_CHECK(budget >= 1 && recent >= 0, name, ": budget >= 1 and recent >= 0 required, got ", budget, " and ", recent);
    const int keep = (int)std::min<int64_t>(budget, INT32_MAX), fresh = (int)std::min<int64_t>(recent, INT32_MAX);
    const c10::hip::HIPGuardMasqueradingAsCUDA guard(kv_pages.device());
    at::Tensor lens = gpu_empty({c.B}, at::kInt, kv_pages);
    const size_t need = mi355_cache_evict_workspace_bytes(&c, keep);
    const at::Tensor ws = workspace_of(need, kv_pages);
    hipStream_t stream = c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream();
    const int rc = mi355_cache_evict(&c, keep, fresh, lens.data_ptr<int32_t>(), need > 0 ? ws.data_ptr() : nullptr, need, stream);
    TORCH_CHECK(rc == 0, name, ": ", mi355_last_error(), " (code ", rc, ")");
    return lens;
}

}  // namespace

// Defines the operators (the first eight schema strings are the reference's).
TORCH_LIBRARY(fmha_unified, m) {
    m.def("finefmha_0(Tensor q, Tensor k, Tensor v, bool causal, bool is_decode, int decode_length) -> Tensor");
    m.def("finefmha_1(Tensor q, Tensor k, Tensor v, bool causal, bool is_decode, int decode_length) -> Tensor");
    m.def("finefmha_2(Tensor q, Tensor k, Tensor v, bool causal, bool is_decode, int decode_length) -> Tensor");
    m.def("finefmha_3(Tensor q, Tensor k, Tensor v, bool causal, bool is_decode, int decode_length) -> Tensor");
    m.def("finefmha_4(Tensor q, Tensor k, Tensor v, bool causal, bool is_decode, int decode_length) -> Tensor");
    m.def("finefmha_5(Tensor q, Tensor k, Tensor v, bool causal, bool is_decode, int decode_length) -> Tensor");
    m.def("finefmha_6(Tensor q, Tensor k, Tensor v, bool causal, bool is_decode, int decode_length) -> Tensor");
    m.def("finefmha_7(Tensor q, Tensor k, Tensor v, bool causal, bool is_decode, int decode_length) -> Tensor");
    m.def("finefmha_fwd_lse(Tensor q, Tensor k, Tensor v, bool causal, bool is_decode, int decode_length) -> (Tensor, Tensor)");
    m.def("finefmha_paged(Tensor q, Tensor kv_pages, Tensor block_table, Tensor seq_lens, Tensor? new_lens, Tensor(a!)? weights) -> Tensor");
    m.def("finefmha_paged_lse(Tensor q, Tensor kv_pages, Tensor block_table, Tensor seq_lens, Tensor? new_lens, Tensor(a!)? weights) -> (Tensor, Tensor)");
    m.def("rope_paged(Tensor(a!) qkv, Tensor(b!) kv_pages, Tensor block_table, Tensor seq_lens, Tensor cos, Tensor sin, Tensor positions, int q_heads, "
          "Tensor? new_lens, Tensor(c!)? weights, Tensor(d!)? key_positions, bool keep_keys) -> ()");
    m.def("key_weights(Tensor q, Tensor lse, Tensor kv_pages, Tensor block_table, Tensor seq_lens, Tensor(a!) weights, Tensor? new_lens, int last_rows) -> ()");
    m.def("evict_paged(Tensor(a!) kv_pages, Tensor block_table, Tensor seq_lens, Tensor(b!) weights, Tensor(c!) key_positions, int budget, int recent) -> Tensor");
}

TORCH_LIBRARY_IMPL(fmha_unified, CUDA, m) {
    m.impl("finefmha_0", &finefmha);
    m.impl("finefmha_1", &finefmha);
    m.impl("finefmha_2", &finefmha);
    m.impl("finefmha_3", &finefmha);
    m.impl("finefmha_4", &finefmha);
    m.impl("finefmha_5", &finefmha);
    m.impl("finefmha_6", &finefmha);
    m.impl("finefmha_7", &finefmha);
    m.impl("finefmha_fwd_lse", &finefmha_fwd_lse);
    m.impl("finefmha_paged", &finefmha_paged);
    m.impl("finefmha_paged_lse", &finefmha_paged_lse);
    m.impl("rope_paged", &rope_paged);
    m.impl("key_weights", &key_weights);
    m.impl("evict_paged", &evict_paged);
}

// The same functions under the CPU key: CPU tensors then reach the argument validation above and are
// rejected with its message ("must be GPU tensors") instead of a dispatcher error. Nothing is computed on the CPU.
TORCH_LIBRARY_IMPL(fmha_unified, CPU, m) {
    m.impl("finefmha_0", &finefmha);
    m.impl("finefmha_1", &finefmha);
    m.impl("finefmha_2", &finefmha);
    m.impl("finefmha_3", &finefmha);
    m.impl("finefmha_4", &finefmha);
    m.impl("finefmha_5", &finefmha);
    m.impl("finefmha_6", &finefmha);
    m.impl("finefmha_7", &finefmha);
    m.impl("finefmha_fwd_lse", &finefmha_fwd_lse);
    m.impl("finefmha_paged", &finefmha_paged);
    m.impl("finefmha_paged_lse", &finefmha_paged_lse);
    m.impl("rope_paged", &rope_paged);
    m.impl("key_weights", &key_weights);
    m.impl("evict_paged", &evict_paged);
}

// _C as a Python extension module. The operators of the paged cache are functions of it as well: with eight to twelve arguments, most of them tensors, a call
// through the dispatcher takes the host 1 us longer than one of these, and a step's calls are a few us long on the GPU (64 tokens filed, calls one
// behind the other: 6.4 us each, 7.5 through the dispatcher). Where something is there that only the dispatcher shows a call to (a mode, a transform, a
// tracer, a tensor that needs a gradient, whose result says on the way back that there is none), it is asked.
namespace {

const c10::DispatchKeySet kWatchers({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot, c10::DispatchKey::PythonDispatcher, c10::DispatchKey::Functionalize,
                                     c10::DispatchKey::FuncTorchDynamicLayerFrontMode, c10::DispatchKey::FuncTorchDynamicLayerBackMode,
                                     c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::Batched, c10::DispatchKey::Tracer});

bool watched(const at::Tensor& t) { return t.defined() && (t.key_set().has_any(kWatchers) || (t.requires_grad() && at::GradMode::is_enabled())); }
bool watched(const std::optional<at::Tensor>& t) { return t.has_value() && watched(*t); }
bool watched(int64_t) { return false; }

template <typename R, typename... A>
void def(py::module_& m, const char* name, R (*kernel)(A...)) {
    const auto op = c10::Dispatcher::singleton().findSchemaOrThrow((std::string("fmha_unified::") + name).c_str(), "").typed<R(A...)>();
    m.def(name, [=](A... a) -> R {
        if (c10::impl::tls_local_dispatch_key_set().included_.has_any(kWatchers) || (watched(a) || ...)) return op.call(a...);
        return kernel(a...);
    }, py::call_guard<py::gil_scoped_release>());
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    def(m, "finefmha_paged", &finefmha_paged);
    def(m, "finefmha_paged_lse", &finefmha_paged_lse);
    def(m, "rope_paged", &rope_paged);
    def(m, "key_weights", &key_weights);
    def(m, "evict_paged", &evict_paged);
}

}  // namespace fmha_unified
