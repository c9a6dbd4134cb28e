// C ABI of libmi355_serving.so (see include/mi355_serving.h): argument validation and error reporting around
// the kernel dispatchers. Nothing here allocates device memory or synchronises (the library's workspaces, one per device and
// stream each, are those of fmha_decode.hip, fmha_fwd.hip and hgemm_dispatch.hip).
#include <cstdarg>
#include <cstdio>
#include <cstring>
#include "mi355_serving_internal.h"

namespace {
thread_local char g_err[256] = "";

int fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return code;
}
int hip_fail(hipError_t e, const char* what) {
    return fail(static_cast<int>(e), "%s: %s", what, hipGetErrorString(e));
}
mi355::FmhaStrides contiguous_strides(int Hq, int Hkv, int Sq, int Sk, int D) {
    const long q_head = (long)Sq * D, k_head = (long)Sk * D;
    return {Hq * q_head, q_head, D, Hkv * k_head, k_head, D, Hkv * k_head, k_head, D, Hq * q_head, q_head, D};
}
mi355::FmhaStrides strides_from(const int64_t* s) {
    return {(long)s[0], (long)s[1], (long)s[2], (long)s[3], (long)s[4], (long)s[5],
            (long)s[6], (long)s[7], (long)s[8], (long)s[9], (long)s[10], (long)s[11]};
}
}  // namespace

extern "C" {

// R == nullptr: the plain product; otherwise the residual operand of the *_add entry points (checked by the caller)
static int hgemm_impl(const char* fn, int dtype, const void* A, const void* B, void* C, const void* R, int M, int N, int K, int64_t lda,
                      int64_t ldb, int64_t ldc, int64_t ldr, int layout, void* stream, int variant = 0, void* workspace = nullptr,
                      size_t workspace_bytes = 0) {
    if (!A || !B || !C) return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer", fn);
    if (M < 1 || N < 1 || K < 1) return fail(MI355_ERR_BAD_ARGUMENT, "%s: M, N, K must be >= 1 (got %d, %d, %d)", fn, M, N, K);
    if (layout != MI355_GEMM_NN && layout != MI355_GEMM_NT && layout != MI355_GEMM_TN)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: unknown layout %d", fn, layout);
    const int64_t a_min = (layout == MI355_GEMM_TN) ? M : K;
    const int64_t b_min = (layout == MI355_GEMM_NT) ? K : N;
    if (lda < a_min || ldb < b_min || ldc < N)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: leading dimension too small (lda %lld >= %lld, ldb %lld >= %lld, ldc %lld >= %d required)", fn,
                    (long long)lda, (long long)a_min, (long long)ldb, (long long)b_min, (long long)ldc, N);
    if (R != nullptr && ldr < N)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: leading dimension too small (ldr %lld >= %d required)", fn, (long long)ldr, N);
    if (R != nullptr && R == C && ldr != ldc)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: R aliases C but ldr (%lld) differs from ldc (%lld)", fn, (long long)ldr, (long long)ldc);
    hipError_t e = mi355::hgemm_dispatch(A, B, C, R, M, N, K, lda, ldb, ldc, R ? ldr : 0, layout, dtype, variant, workspace, workspace_bytes,
                                     static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, fn);
    return 0;
}

int mi355_hgemm(const void* A, const void* B, void* C, int M, int N, int K, int64_t lda, int64_t ldb, int64_t ldc,
                int layout, void* stream) {
    return hgemm_impl("mi355_hgemm", MI355_DTYPE_FP16, A, B, C, nullptr, M, N, K, lda, ldb, ldc, 0, layout, stream);
}

int mi355_gemm_bf16(const void* A, const void* B, void* C, int M, int N, int K, int64_t lda, int64_t ldb, int64_t ldc,
                int layout, void* stream) {
    return hgemm_impl("mi355_gemm_bf16", MI355_DTYPE_BF16, A, B, C, nullptr, M, N, K, lda, ldb, ldc, 0, layout, stream);
}

int mi355_hgemm_add(const void* A, const void* B, const void* R, void* C, int M, int N, int K, int64_t lda, int64_t ldb, int64_t ldr,
                    int64_t ldc, int layout, void* stream) {
    if (!R) return fail(MI355_ERR_BAD_ARGUMENT, "mi355_hgemm_add: null pointer");
    return hgemm_impl("mi355_hgemm_add", MI355_DTYPE_FP16, A, B, C, R, M, N, K, lda, ldb, ldc, ldr, layout, stream);
}

int mi355_gemm_add_bf16(const void* A, const void* B, const void* R, void* C, int M, int N, int K, int64_t lda, int64_t ldb, int64_t ldr,
                        int64_t ldc, int layout, void* stream) {
    if (!R) return fail(MI355_ERR_BAD_ARGUMENT, "mi355_gemm_add_bf16: null pointer");
    return hgemm_impl("mi355_gemm_add_bf16", MI355_DTYPE_BF16, A, B, C, R, M, N, K, lda, ldb, ldc, ldr, layout, stream);
}


size_t mi355_gemm_workspace_bytes(const void* A, const void* B, int M, int N, int K, int64_t lda, int64_t ldb, int layout) {
    if (!A || !B || M < 1 || N < 1 || K < 1 || layout < MI355_GEMM_NN || layout > MI355_GEMM_TN) return 0;
    return mi355::hgemm_workspace_bytes(A, B, M, N, K, lda, ldb, layout);
}

size_t mi355_internal_gemm_copy_bytes(const void* A, const void* B, int M, int N, int K, int64_t lda, int64_t ldb, int layout) {
    if (!A || !B || M < 1 || N < 1 || K < 1 || layout < MI355_GEMM_NN || layout > MI355_GEMM_TN) return 0;
    return mi355::hgemm_copy_bytes(A, B, M, N, K, lda, ldb, layout);
}

int mi355_gemm_ws(const void* A, const void* B, const void* R, void* C, int M, int N, int K, int64_t lda, int64_t ldb, int64_t ldr,
                  int64_t ldc, int layout, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    if (dtype != MI355_DTYPE_FP16 && dtype != MI355_DTYPE_BF16) return fail(MI355_ERR_BAD_ARGUMENT, "mi355_gemm_ws: unknown dtype %d", dtype);
    if (reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
        return fail(MI355_ERR_BAD_ARGUMENT, "mi355_gemm_ws: the workspace must be 16-byte aligned (got %p)", workspace);
    return hgemm_impl("mi355_gemm_ws", dtype, A, B, C, R, M, N, K, lda, ldb, ldc, ldr, layout, stream, 0, workspace, workspace_bytes);
}

static int fmha_checked(const char* fn, const void* Q, const void* K, const void* V, void* O, float* LSE, int B, int Hq, int Hkv,
                        int Sq, int Sk, int D, float scale, int causal, int kv_valid_len, const mi355::FmhaStrides& sd,
                        int dtype, void* stream, int variant = 0, const mi355::FmhaWorkspace& ws = mi355::FmhaWorkspace()) {
    if (!Q || !K || !V || !O) return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer", fn);
    if (B < 1 || Hq < 1 || Hkv < 1 || Sq < 1 || Sk < 1)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: B, Hq, Hkv, Sq, Sk must be >= 1", fn);
    if (D != 128) return fail(MI355_ERR_UNSUPPORTED, "%s: head_dim must be 128 (got %d)", fn, D);
    if (Hq % Hkv != 0) return fail(MI355_ERR_BAD_ARGUMENT, "%s: Hq (%d) must be a multiple of Hkv (%d)", fn, Hq, Hkv);
    if (kv_valid_len < 1 || kv_valid_len > Sk)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: kv_valid_len %d outside [1, Sk=%d]", fn, kv_valid_len, Sk);
    if (!(scale > 0.f) || scale > 3.0e38f)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: scale must be positive and finite (got %g)", fn, (double)scale);
    if ((reinterpret_cast<uintptr_t>(Q) | reinterpret_cast<uintptr_t>(K) | reinterpret_cast<uintptr_t>(V) |
         reinterpret_cast<uintptr_t>(O)) % 16 != 0)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: Q, K, V, O must be 16-byte aligned", fn);
    const long all[12] = {sd.q_batch, sd.q_head, sd.q_row, sd.k_batch, sd.k_head, sd.k_row,
                          sd.v_batch, sd.v_head, sd.v_row, sd.o_batch, sd.o_head, sd.o_row};
    for (int i = 0; i < 12; ++i)
        if (all[i] < 0 || all[i] % 8 != 0)
            return fail(MI355_ERR_BAD_ARGUMENT, "%s: stride %d is %ld; strides must be non-negative multiples of 8 elements", fn, i,
                        all[i]);
    if (sd.o_row < D || (Hq > 1 && sd.o_head < D) || (B > 1 && sd.o_batch < D))
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: rows of O overlap (o strides %ld, %ld, %ld)", fn, sd.o_batch, sd.o_head, sd.o_row);
    if (ws.kind == mi355::FmhaWorkspace::kCaller) {
        const size_t need = mi355::fmha_decode_workspace_bytes(B, Hq, Hkv, Sq, Sk, kv_valid_len);
        if (need > 0 && (ws.ptr == nullptr || ws.bytes < need || reinterpret_cast<uintptr_t>(ws.ptr) % 16 != 0))
            return fail(MI355_ERR_BAD_ARGUMENT, "%s: workspace of %zu bytes at %p; this call needs %zu bytes, 16-byte aligned "
                        "(mi355_fmha_fwd_workspace_bytes)", fn, ws.bytes, ws.ptr, need);
    }
    hipError_t e = mi355::fmha_fwd_dispatch(Q, K, V, O, LSE, B, Hq, Hkv, Sq, Sk, scale, causal != 0, kv_valid_len, sd, dtype,
                                            variant, ws, static_cast<hipStream_t>(stream));
    if (e == hipErrorNotSupported)
        return fail(MI355_ERR_UNSUPPORTED, "%s: row strides of K and V must be below 2^24 elements (got %ld, %ld)", fn, sd.k_row, sd.v_row);
    if (e == hipErrorStreamCaptureUnsupported)
        return fail(static_cast<int>(e), "%s: the split-KV workspace of this stream would have to be allocated or enlarged while "
                    "the stream is capturing; run the call once before capture, or use mi355_fmha_fwd_ws", fn);
    if (e != hipSuccess) return hip_fail(e, fn);
    return 0;
}

static int hgemm_silu_mul_impl(const char* fn, int dtype, const void* A, const void* B, void* C, int M, int N, int K, int64_t lda, int64_t ldb, int64_t ldc,
                         int layout, void* stream, int variant = 0) {
    if (!A || !B || !C) return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer", fn);
    if (M < 1 || N < 1 || K < 1) return fail(MI355_ERR_BAD_ARGUMENT, "%s: M, N, K must be >= 1", fn);
    if (layout != MI355_GEMM_NN && layout != MI355_GEMM_NT)
        return fail(MI355_ERR_UNSUPPORTED, "%s: layout %d has no fused epilogue (NN and NT do)", fn, layout);
    const int64_t b_min = (layout == MI355_GEMM_NT) ? K : 2 * (int64_t)N;
    if (lda < K || ldb < b_min || ldc < N)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: leading dimension too small", fn);
    if (N > 0x3fffffff) return fail(MI355_ERR_BAD_ARGUMENT, "%s: N too large", fn);
    hipError_t e = mi355::hgemm_silu_mul_dispatch(A, B, C, M, 2 * N, K, lda, ldb, ldc, layout, dtype, variant, static_cast<hipStream_t>(stream));
    if (e == hipErrorNotSupported)
        return fail(MI355_ERR_UNSUPPORTED,
                    "%s: needs N a multiple of 32, K a multiple of 64 and 16-byte aligned operands; "
                    "run mi355_hgemm and mi355_silu_mul(interleave = 32) instead", fn);
    if (e != hipSuccess) return hip_fail(e, fn);
    return 0;
}

int mi355_hgemm_silu_mul(const void* A, const void* B, void* C, int M, int N, int K, int64_t lda, int64_t ldb, int64_t ldc,
                         int layout, void* stream) {
    return hgemm_silu_mul_impl("mi355_hgemm_silu_mul", MI355_DTYPE_FP16, A, B, C, M, N, K, lda, ldb, ldc, layout, stream);
}

int mi355_internal_hgemm_silu_mul_variant(const void* A, const void* B, void* C, int M, int N, int K, int64_t lda, int64_t ldb,
                                          int64_t ldc, int layout, int dtype, int variant, void* stream) {
    return hgemm_silu_mul_impl("mi355_internal_hgemm_silu_mul_variant", dtype, A, B, C, M, N, K, lda, ldb, ldc, layout, stream, variant);
}

int mi355_gemm_silu_mul_bf16(const void* A, const void* B, void* C, int M, int N, int K, int64_t lda, int64_t ldb, int64_t ldc,
                         int layout, void* stream) {
    return hgemm_silu_mul_impl("mi355_gemm_silu_mul_bf16", MI355_DTYPE_BF16, A, B, C, M, N, K, lda, ldb, ldc, layout, stream);
}


int mi355_fmha_fwd(const void* Q, const void* K, const void* V, void* O, float* LSE, int B, int Hq, int Hkv, int Sq,
                   int Sk, int D, float scale, int causal, int kv_valid_len, void* stream) {
    return fmha_checked("mi355_fmha_fwd", Q, K, V, O, LSE, B, Hq, Hkv, Sq, Sk, D, scale, causal, kv_valid_len,
                        contiguous_strides(Hq, Hkv, Sq, Sk, D), MI355_DTYPE_FP16, stream);
}

int mi355_fmha_fwd_strided(const void* Q, const void* K, const void* V, void* O, float* LSE, int B, int Hq, int Hkv, int Sq,
                           int Sk, int D, float scale, int causal, int kv_valid_len, const int64_t* strides, void* stream) {
    if (!strides) return fail(MI355_ERR_BAD_ARGUMENT, "mi355_fmha_fwd_strided: null strides");
    return fmha_checked("mi355_fmha_fwd_strided", Q, K, V, O, LSE, B, Hq, Hkv, Sq, Sk, D, scale, causal, kv_valid_len,
                        strides_from(strides), MI355_DTYPE_FP16, stream);
}

int mi355_fmha_fwd_bf16(const void* Q, const void* K, const void* V, void* O, float* LSE, int B, int Hq, int Hkv, int Sq,
                        int Sk, int D, float scale, int causal, int kv_valid_len, const int64_t* strides, void* stream) {
    return fmha_checked("mi355_fmha_fwd_bf16", Q, K, V, O, LSE, B, Hq, Hkv, Sq, Sk, D, scale, causal, kv_valid_len,
                        strides ? strides_from(strides) : contiguous_strides(Hq, Hkv, Sq, Sk, D), MI355_DTYPE_BF16, stream);
}

size_t mi355_fmha_fwd_workspace_bytes(int B, int Hq, int Hkv, int Sq, int Sk, int kv_valid_len) {
    if (B < 1 || Hq < 1 || Hkv < 1 || Sq < 1 || Sk < 1 || Hq % Hkv != 0 || kv_valid_len < 1 || kv_valid_len > Sk) return 0;
    return mi355::fmha_workspace_bytes(B, Hq, Hkv, Sq, Sk, kv_valid_len);
}

int mi355_fmha_fwd_ws(const void* Q, const void* K, const void* V, void* O, float* LSE, int B, int Hq, int Hkv, int Sq,
                      int Sk, int D, float scale, int causal, int kv_valid_len, const int64_t* strides, int dtype,
                      void* workspace, size_t workspace_bytes, void* stream) {
    if (dtype != MI355_DTYPE_FP16 && dtype != MI355_DTYPE_BF16)
        return fail(MI355_ERR_BAD_ARGUMENT, "mi355_fmha_fwd_ws: unknown dtype %d", dtype);
    mi355::FmhaWorkspace ws;
    ws.kind = mi355::FmhaWorkspace::kCaller;
    ws.ptr = workspace;
    ws.bytes = workspace_bytes;
    return fmha_checked("mi355_fmha_fwd_ws", Q, K, V, O, LSE, B, Hq, Hkv, Sq, Sk, D, scale, causal, kv_valid_len,
                        strides ? strides_from(strides) : contiguous_strides(Hq, Hkv, Sq, Sk, D), dtype, stream, 0, ws);
}

int mi355_fmha_fwd_noalloc(const void* Q, const void* K, const void* V, void* O, float* LSE, int B, int Hq, int Hkv, int Sq,
                           int Sk, int D, float scale, int causal, int kv_valid_len, const int64_t* strides, void* stream) {
    const char* fn = "mi355_fmha_fwd_noalloc";
    if (B >= 1 && Hq >= 1 && Hkv >= 1 && Sq >= 1 && Sk >= 1 && Hq % Hkv == 0 && kv_valid_len >= 1 && kv_valid_len <= Sk) {
        const size_t need = mi355::fmha_decode_workspace_bytes(B, Hq, Hkv, Sq, Sk, kv_valid_len);
        if (need > mi355::fmha_decode_static_scratch_bytes())
            return fail(MI355_ERR_UNSUPPORTED, "%s: the split-KV partial results of this call take %zu bytes, the static scratch "
                        "holds %zu; use mi355_fmha_fwd_ws with a workspace of your own", fn, need,
                        mi355::fmha_decode_static_scratch_bytes());
    }
    mi355::FmhaWorkspace ws;
    ws.kind = mi355::FmhaWorkspace::kStatic;
    return fmha_checked(fn, Q, K, V, O, LSE, B, Hq, Hkv, Sq, Sk, D, scale, causal, kv_valid_len,
                        strides ? strides_from(strides) : contiguous_strides(Hq, Hkv, Sq, Sk, D), MI355_DTYPE_FP16, stream, 0, ws);
}

int mi355_internal_fmha_fwd_variant(const void* Q, const void* K, const void* V, void* O, float* LSE, int B, int Hq, int Hkv,
                                    int Sq, int Sk, int D, float scale, int causal, int kv_valid_len, const int64_t* strides,
                                    int dtype, int variant, void* stream) {
    return fmha_checked("mi355_internal_fmha_fwd_variant", Q, K, V, O, LSE, B, Hq, Hkv, Sq, Sk, D, scale, causal, kv_valid_len,
                        strides ? strides_from(strides) : contiguous_strides(Hq, Hkv, Sq, Sk, D), dtype, stream, variant);
}

int mi355_internal_hgemm_choice(int M, int N, int K, int64_t ldb, int layout, float* us) {
    const mi355::KernelChoice k = mi355::choose_kernel(M, N, K, layout != MI355_GEMM_TN, layout == MI355_GEMM_NT, true, true, ldb % 64 == 0);
    if (us != nullptr) *us = k.us;
    return k.shape + (k.splits > 1 ? 16 * k.splits : 0) + (k.own_merge ? 4096 : 0);
}

int mi355_internal_hgemm_wide_ranges(int M, int N, int K, int64_t ldb, int layout) {
    const mi355::KernelChoice k = mi355::choose_kernel(M, N, K, layout != MI355_GEMM_TN, layout == MI355_GEMM_NT, true, true, ldb % 64 == 0);
    return k.shape == mi355::kSmallM && k.wide_ranges > 1 ? k.wide_ranges : 0;
}

int mi355_internal_hgemm_direct_choice(int M, int N, int K, int layout, float* us) {
    const mi355::KernelChoice k = mi355::choose_direct(M, N, K, layout, true);
    if (us != nullptr) *us = k.us;
    return k.shape + (k.splits > 1 ? 16 * k.splits : 0);
}

int mi355_internal_fmha_decode_plan(int B, int Hq, int Hkv, int Sq, int kv_valid_len, int* splits, int* waves) {
    if (B < 1 || Hkv < 1 || Hq < Hkv || Hq % Hkv != 0 || Sq < 1 || kv_valid_len < 1 || !splits || !waves)
        return fail(MI355_ERR_BAD_ARGUMENT, "mi355_internal_fmha_decode_plan: bad argument");
    mi355::fmha_decode_plan_of(B, Hq, Hkv, Sq, kv_valid_len, splits, waves);
    return 0;
}

int mi355_internal_hgemm_variant(const void* A, const void* B, void* C, int M, int N, int K, int64_t lda, int64_t ldb,
                                 int64_t ldc, int layout, int dtype, int variant, void* stream) {
    return hgemm_impl("mi355_internal_hgemm_variant", dtype, A, B, C, nullptr, M, N, K, lda, ldb, ldc, 0, layout, stream, variant);
}

int mi355_internal_hgemm_add_variant(const void* A, const void* B, const void* R, void* C, int M, int N, int K, int64_t lda, int64_t ldb,
                                     int64_t ldr, int64_t ldc, int layout, int dtype, int variant, void* stream) {
    if (!R) return fail(MI355_ERR_BAD_ARGUMENT, "mi355_internal_hgemm_add_variant: null pointer");
    return hgemm_impl("mi355_internal_hgemm_add_variant", dtype, A, B, C, R, M, N, K, lda, ldb, ldc, ldr, layout, stream, variant);
}

static bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

static int rmsnorm_impl(const char* fn, int dtype, const void* x, const void* residual, void* residual_out, const void* weight, void* out, int64_t rows,
                  int hidden, int64_t ldx, int64_t ldr, int64_t ldro, int64_t ldo, float eps, void* stream) {
    if (!x || !weight || !out) return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer", fn);
    if ((residual == nullptr) != (residual_out == nullptr))
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: residual and residual_out must both be given or both be NULL", fn);
    if (rows < 1 || hidden < 8 || hidden % 8 != 0)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: rows >= 1 and hidden a positive multiple of 8 required (got %lld, %d)", fn,
                    (long long)rows, hidden);
    if (ldx < hidden || ldo < hidden || ldx % 8 || ldo % 8 ||
        (residual && (ldr < hidden || ldro < hidden || ldr % 8 || ldro % 8)))
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: row strides must be multiples of 8 and >= hidden", fn);
    if (!aligned16(x) || !aligned16(weight) || !aligned16(out) || !aligned16(residual) || !aligned16(residual_out))
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: pointers must be 16-byte aligned", fn);
    if (!(eps >= 0.f) || eps > 1.f) return fail(MI355_ERR_BAD_ARGUMENT, "%s: eps outside [0, 1] (got %g)", fn, (double)eps);
    hipError_t e = mi355::rmsnorm_dispatch(x, residual, residual_out, weight, out, rows, hidden, ldx, ldr, ldro, ldo, eps, dtype,
                                           static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, fn);
    return 0;
}

int mi355_rmsnorm(const void* x, const void* residual, void* residual_out, const void* weight, void* out, int64_t rows,
                  int hidden, int64_t ldx, int64_t ldr, int64_t ldro, int64_t ldo, float eps, void* stream) {
    return rmsnorm_impl("mi355_rmsnorm", MI355_DTYPE_FP16, x, residual, residual_out, weight, out, rows, hidden, ldx, ldr, ldro, ldo, eps, stream);
}

int mi355_rmsnorm_bf16(const void* x, const void* residual, void* residual_out, const void* weight, void* out, int64_t rows,
                  int hidden, int64_t ldx, int64_t ldr, int64_t ldro, int64_t ldo, float eps, void* stream) {
    return rmsnorm_impl("mi355_rmsnorm_bf16", MI355_DTYPE_BF16, x, residual, residual_out, weight, out, rows, hidden, ldx, ldr, ldro, ldo, eps, stream);
}


static int rope_impl(const char* fn, int dtype, const void* x, void* out, int B, int S, int heads, int copy_heads, int D, int64_t x_batch, int64_t x_row,
               int64_t out_batch, int64_t out_row, const float* cos_table, const float* sin_table, const int32_t* positions,
               int64_t pos_batch, int n_positions, void* stream) {
    if (!x || !out || !cos_table || !sin_table || !positions) return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer", fn);
    if (D != 128) return fail(MI355_ERR_UNSUPPORTED, "%s: head_dim must be 128 (got %d)", fn, D);
    if (B < 1 || S < 1 || heads < 0 || copy_heads < 0 || heads + copy_heads < 1 || n_positions < 1 || pos_batch < 0)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: B, S, heads + copy_heads, n_positions must be >= 1, pos_batch >= 0", fn);
    const int64_t width = (int64_t)(heads + copy_heads) * D;
    if (x_row < width || out_row < width || x_row % 8 || out_row % 8 || x_batch % 8 || out_batch % 8 || x_batch < 0 || out_batch < 0)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: strides must be multiples of 8, row strides >= (heads + copy_heads) * 128", fn);
    if (!aligned16(x) || !aligned16(out) || !aligned16(cos_table) || !aligned16(sin_table))
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: pointers must be 16-byte aligned", fn);
    hipError_t e = mi355::rope_dispatch(x, out, B, S, 0, heads, copy_heads, x_batch, x_row, out_batch, out_row, D, cos_table, sin_table,
                                        positions, pos_batch, n_positions, dtype, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, fn);
    return 0;
}

static int rope_qkv_check(const char* fn, const void* qkv, const void* kv_out, int B, int S, int q_heads, int kv_heads, int D,
                          int64_t x_batch, int64_t x_row, int64_t out_batch, int64_t out_row, int64_t out_head, const float* cos_table,
                          const float* sin_table, const int32_t* positions, int64_t pos_batch, int n_positions) {
    if (!qkv || !kv_out || !cos_table || !sin_table || !positions) return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer", fn);
    if (D != 128) return fail(MI355_ERR_UNSUPPORTED, "%s: head_dim must be 128 (got %d)", fn, D);
    if (B < 1 || S < 1 || q_heads < 1 || kv_heads < 1 || n_positions < 1 || pos_batch < 0)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: B, S, q_heads, kv_heads, n_positions must be >= 1, pos_batch >= 0", fn);
    const int64_t in_width = ((int64_t)q_heads + 2 * (int64_t)kv_heads) * D;
    if (x_row < in_width || out_row < D || out_head < D || x_row % 8 || out_row % 8 || out_head % 8 || x_batch % 8 || out_batch % 8 ||
        x_batch < 0 || out_batch < 0)
        return fail(MI355_ERR_BAD_ARGUMENT,
                    "%s: strides must be multiples of 8, x_row >= (q_heads + 2 kv_heads) * 128, out_row >= 128, out_head >= 128", fn);
    // heads side by side in a token row (out_head == 128) need a row that holds them all; a head-major cache (out_head >= a
    // head's whole sequence) needs rows of 128
    if (out_head < (int64_t)S * out_row && out_row < 2 * (int64_t)kv_heads * out_head)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: out_row / out_head make the heads of a token overlap those of the next", fn);
    if (!aligned16(qkv) || !aligned16(kv_out) || !aligned16(cos_table) || !aligned16(sin_table))
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: pointers must be 16-byte aligned", fn);
    return 0;
}

static int rope_qkv_impl(const char* fn, int dtype, void* qkv, void* kv_out, int B, int S, int q_heads, int kv_heads, int D,
                         int64_t x_batch, int64_t x_row, int64_t out_batch, int64_t out_row, int64_t out_head, const float* cos_table,
                         const float* sin_table, const int32_t* positions, int64_t pos_batch, int n_positions, void* stream) {
    if (const int rc = rope_qkv_check(fn, qkv, kv_out, B, S, q_heads, kv_heads, D, x_batch, x_row, out_batch, out_row, out_head, cos_table, sin_table,
                                      positions, pos_batch, n_positions); rc != 0) return rc;
    hipError_t e = mi355::rope_dispatch(qkv, kv_out, B, S, q_heads, q_heads + kv_heads, kv_heads, x_batch, x_row, out_batch, out_row,
                                        out_head, cos_table, sin_table, positions, pos_batch, n_positions, dtype, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, fn);
    return 0;
}

int mi355_rope_qkv(void* qkv, void* kv_out, int B, int S, int q_heads, int kv_heads, int D, int64_t x_batch, int64_t x_row,
                   int64_t out_batch, int64_t out_row, int64_t out_head, const float* cos_table, const float* sin_table, const int32_t* positions,
                   int64_t pos_batch, int n_positions, void* stream) {
    return rope_qkv_impl("mi355_rope_qkv", MI355_DTYPE_FP16, qkv, kv_out, B, S, q_heads, kv_heads, D, x_batch, x_row, out_batch, out_row, out_head, cos_table, sin_table, positions, pos_batch, n_positions, stream);
}

int mi355_rope_qkv_bf16(void* qkv, void* kv_out, int B, int S, int q_heads, int kv_heads, int D, int64_t x_batch, int64_t x_row,
                        int64_t out_batch, int64_t out_row, int64_t out_head, const float* cos_table, const float* sin_table, const int32_t* positions,
                        int64_t pos_batch, int n_positions, void* stream) {
    return rope_qkv_impl("mi355_rope_qkv_bf16", MI355_DTYPE_BF16, qkv, kv_out, B, S, q_heads, kv_heads, D, x_batch, x_row, out_batch, out_row, out_head, cos_table, sin_table, positions, pos_batch, n_positions, stream);
}

int mi355_rope(const void* x, void* out, int B, int S, int heads, int copy_heads, int D, int64_t x_batch, int64_t x_row,
               int64_t out_batch, int64_t out_row, const float* cos_table, const float* sin_table, const int32_t* positions,
               int64_t pos_batch, int n_positions, void* stream) {
    return rope_impl("mi355_rope", MI355_DTYPE_FP16, x, out, B, S, heads, copy_heads, D, x_batch, x_row, out_batch, out_row, cos_table, sin_table, positions, pos_batch, n_positions, stream);
}

int mi355_rope_bf16(const void* x, void* out, int B, int S, int heads, int copy_heads, int D, int64_t x_batch, int64_t x_row,
               int64_t out_batch, int64_t out_row, const float* cos_table, const float* sin_table, const int32_t* positions,
               int64_t pos_batch, int n_positions, void* stream) {
    return rope_impl("mi355_rope_bf16", MI355_DTYPE_BF16, x, out, B, S, heads, copy_heads, D, x_batch, x_row, out_batch, out_row, cos_table, sin_table, positions, pos_batch, n_positions, stream);
}


static int silu_mul_impl(const char* fn, int dtype, const void* gate_up, void* out, int64_t rows, int inter, int interleave, int64_t ld_in, int64_t ld_out,
                   void* stream) {
    if (!gate_up || !out) return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer", fn);
    if (rows < 1 || inter < 8 || inter % 8 != 0)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: rows >= 1 and inter a positive multiple of 8 required", fn);
    if (interleave < 0 || interleave % 8 != 0 || (interleave > 0 && inter % interleave != 0))
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: interleave must be 0 or a multiple of 8 that divides inter (got %d)", fn,
                    interleave);
    if (ld_in < 2 * (int64_t)inter || ld_out < inter || ld_in % 8 || ld_out % 8)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: ld_in >= 2 * inter, ld_out >= inter, both multiples of 8 required", fn);
    if (!aligned16(gate_up) || !aligned16(out)) return fail(MI355_ERR_BAD_ARGUMENT, "%s: pointers must be 16-byte aligned", fn);
    hipError_t e = mi355::silu_mul_dispatch(gate_up, out, rows, inter, interleave, ld_in, ld_out, dtype, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return hip_fail(e, fn);
    return 0;
}

int mi355_silu_mul(const void* gate_up, void* out, int64_t rows, int inter, int interleave, int64_t ld_in, int64_t ld_out,
                   void* stream) {
    return silu_mul_impl("mi355_silu_mul", MI355_DTYPE_FP16, gate_up, out, rows, inter, interleave, ld_in, ld_out, stream);
}

int mi355_silu_mul_bf16(const void* gate_up, void* out, int64_t rows, int inter, int interleave, int64_t ld_in, int64_t ld_out,
                   void* stream) {
    return silu_mul_impl("mi355_silu_mul_bf16", MI355_DTYPE_BF16, gate_up, out, rows, inter, interleave, ld_in, ld_out, stream);
}


// Used by the decoder layer only (declared in mi355_serving_internal.h). A refusal (MI355_ERR_UNSUPPORTED) is no failure, its caller goes
// on with the single calls: it writes no text.
int mi355_internal_step_qkv(const void* x, const void* norm_weight, float eps, const void* w_qkv, void* qkv, void* kv_out, int B, int S, int q_heads,
                            int kv_heads, int hidden, int64_t out_batch, int64_t out_row, int64_t out_head, const float* cos_table,
                            const float* sin_table, const int32_t* positions, int64_t pos_batch, int n_positions, int dtype, void* stream) {
    const char* fn = "mi355_internal_step_qkv";
    if (!x || !w_qkv || hidden < 1) return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer or no columns", fn);
    if (B < 1 || S < 1) return fail(MI355_ERR_BAD_ARGUMENT, "%s: no rows", fn);
    if ((int64_t)B * S > 64) return MI355_ERR_UNSUPPORTED;
    if (q_heads < 1 || kv_heads < 1 || q_heads > (1 << 20) || kv_heads > (1 << 20))
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: q_heads and kv_heads must be >= 1", fn);
    const int64_t width = ((int64_t)q_heads + 2 * (int64_t)kv_heads) * 128;
    if (const int rc = rope_qkv_check(fn, qkv, kv_out, B, S, q_heads, kv_heads, 128, S * width, width, out_batch, out_row, out_head, cos_table,
                                      sin_table, positions, pos_batch, n_positions); rc != 0) return rc;
    const mi355::RopeEpilogue rope = {kv_out, (long)out_batch, (long)out_row, (long)out_head, cos_table, sin_table, positions, (long)pos_batch,
                                      n_positions, S, q_heads, kv_heads};
    const hipError_t e = mi355::gemm_step_qkv_dispatch(x, {norm_weight, eps}, w_qkv, qkv, B * S, (int)width, hidden, rope, dtype,
                                                       static_cast<hipStream_t>(stream));
    if (e == hipErrorNotSupported) return MI355_ERR_UNSUPPORTED;
    return e == hipSuccess ? 0 : hip_fail(e, fn);
}

int mi355_internal_step_gate_up(const void* x, const void* norm_weight, float eps, const void* w_gu, void* out, int rows, int inter, int hidden,
                                int dtype, void* stream) {
    const char* fn = "mi355_internal_step_gate_up";
    if (!x || !norm_weight || !w_gu || !out || rows < 1 || inter < 1 || inter > 0x3fffffff || hidden < 1)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer or empty operand", fn);
    const hipError_t e = mi355::gemm_step_gate_up_dispatch(x, {norm_weight, eps}, w_gu, out, rows, 2 * inter, hidden, dtype,
                                                           static_cast<hipStream_t>(stream));
    if (e == hipErrorNotSupported) return MI355_ERR_UNSUPPORTED;
    return e == hipSuccess ? 0 : hip_fail(e, fn);
}


// ---- the paged key-value cache ----
// Whether the counts (keys, tiles of keys, rows) of a cache and a call stay within what the kernels and their plans count in ints
static bool paged_sizes(const mi355_paged_kv* c) {
    if (!c || c->B < 1 || c->Hkv < 1 || c->max_pages < 1 || c->page_size < 16 || c->page_size % 16 != 0) return false;
    const int64_t pairs = (int64_t)c->B * c->Hkv, max_len = (int64_t)c->max_pages * c->page_size;
    return pairs <= 65535 && max_len <= (1 << 28) && pairs * (max_len / 32 + 1) <= INT32_MAX - 65536;
}
constexpr int64_t kMostWorkgroups = (1 << 24) - 1;   // of 256 threads in one launch
// Likewise of the query columns of a kv head that a call works on: S rows, or the last `last_rows` of them, for each of its query heads. A sequence has no
// more tokens than it has room for keys; a padded batch may be longer, up to 65535 columns
static bool paged_rows(const mi355_paged_kv* c, int Hq, int S, int last_rows) {
    if (Hq < c->Hkv || S < 1 || S > (1 << 28) || last_rows < 0) return false;
    const int64_t rows = last_rows > 0 && last_rows < S ? last_rows : S, max_len = (int64_t)c->max_pages * c->page_size;
    return Hq / c->Hkv * rows <= (rows <= max_len ? kMostWorkgroups : 65535);
}

// What a call needs of the pool itself
static int pool_checked(const char* fn, const mi355_paged_kv* c) {
    if (c->row_stride < 128 || c->row_stride % 8 != 0 || c->head_stride < 128 || c->head_stride % 8 != 0 || c->page_stride < 128 || c->page_stride % 8 != 0)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: strides of the pages must be multiples of 8 elements, 128 or more (got %lld, %lld, %lld)", fn,
                    (long long)c->page_stride, (long long)c->head_stride, (long long)c->row_stride);
    if (c->row_stride >= (1 << 24) || c->row_stride * 2 * c->page_size > INT32_MAX)
        return fail(MI355_ERR_UNSUPPORTED, "%s: row stride %lld of the pages is too large", fn, (long long)c->row_stride);
    if (!aligned16(c->pages) || !aligned16(c->weights) || !aligned16(c->key_positions))
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: pages, weights and key_positions must be 16-byte aligned", fn);
    return 0;
}

static int paged_checked(const char* fn, const mi355_paged_kv* c) {
    if (!c || !c->pages || !c->block_table || !c->seq_lens) return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer", fn);
    if (c->dtype != MI355_DTYPE_FP16 && c->dtype != MI355_DTYPE_BF16) return fail(MI355_ERR_BAD_ARGUMENT, "%s: unknown dtype %d", fn, c->dtype);
    if (c->B < 1 || c->Hkv < 1 || c->n_pages < 1 || c->max_pages < 1)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: B, Hkv, n_pages and max_pages must be >= 1 (got %d, %d, %d, %d)", fn, c->B, c->Hkv, c->n_pages, c->max_pages);
    if (c->page_size < 16 || c->page_size % 16 != 0)
        return fail(MI355_ERR_UNSUPPORTED, "%s: page_size must be a positive multiple of 16 (got %d)", fn, c->page_size);
    const int64_t max_len = (int64_t)c->max_pages * c->page_size;
    if ((int64_t)c->B * c->Hkv > 65535) return fail(MI355_ERR_UNSUPPORTED, "%s: B * Hkv must be at most 65535 (got %d * %d)", fn, c->B, c->Hkv);
    if (!paged_sizes(c))
        return fail(MI355_ERR_UNSUPPORTED, "%s: %d sequences of up to %lld keys of %d heads are more than a call takes", fn, c->B, (long long)max_len, c->Hkv);
    if (c->B > 1 && c->table_stride < c->max_pages)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: rows of the block table overlap (stride %lld, %d entries)", fn, (long long)c->table_stride, c->max_pages);
    return pool_checked(fn, c);
}

static int paged_queries_checked(const char* fn, const mi355_paged_kv* c, const void* Q, int Hq, int S, int last_rows, const int64_t* strides, int n,
                                 float scale) {
    if (!Q) return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer", fn);
    if (Hq < 1 || S < 1) return fail(MI355_ERR_BAD_ARGUMENT, "%s: Hq and S must be >= 1", fn);
    if (Hq % c->Hkv != 0) return fail(MI355_ERR_BAD_ARGUMENT, "%s: Hq (%d) must be a multiple of Hkv (%d)", fn, Hq, c->Hkv);
    if (!paged_rows(c, Hq, S, last_rows))
        return fail(MI355_ERR_UNSUPPORTED, "%s: Hq / Hkv * S must be below 2^24, and below 2^16 for more rows than a sequence may have keys (got %d / %d * %d, %lld keys)", fn,
                    Hq, c->Hkv, S, (long long)c->max_pages * c->page_size);
    // (times log2 e it must be finite too)
    if (!(scale > 0.f) || scale > 2.3e38f) return fail(MI355_ERR_BAD_ARGUMENT, "%s: scale must be positive and at most 2.3e38 (got %g)", fn, (double)scale);
    if (!aligned16(Q)) return fail(MI355_ERR_BAD_ARGUMENT, "%s: Q must be 16-byte aligned", fn);
    for (int i = 0; i < n; ++i)
        if (strides[i] < 0 || strides[i] % 8 != 0)
            return fail(MI355_ERR_BAD_ARGUMENT, "%s: stride %d is %lld; strides must be non-negative multiples of 8 elements", fn, i, (long long)strides[i]);
    if (strides[2] >= (1 << 24)) return fail(MI355_ERR_UNSUPPORTED, "%s: the row stride of Q must be below 2^24 elements (got %lld)", fn, (long long)strides[2]);
    return 0;
}

static int workspace_checked(const char* fn, size_t need, const void* workspace, size_t bytes) {
    if (need > 0 && (workspace == nullptr || bytes < need || !aligned16(workspace)))
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: workspace of %zu bytes at %p; this call needs %zu bytes, 16-byte aligned (%s_workspace_bytes)", fn, bytes,
                    workspace, need, fn);
    return 0;
}

size_t mi355_fmha_paged_workspace_bytes(const mi355_paged_kv* cache, int Hq, int S, int want_lse) {
    if (!paged_sizes(cache) || !paged_rows(cache, Hq, S, 0)) return 0;   // (the call is refused)
    return mi355::fmha_paged_workspace(*cache, Hq, S, want_lse != 0, false);
}

// `parents`: the rows are a tree of drafted tokens (null otherwise)
static int fmha_paged_impl(const char* fn, const mi355_paged_kv* cache, const void* Q, void* O, float* LSE, int Hq, int S, const int64_t* strides,
                           const int32_t* parents, int64_t parents_batch, float scale, void* workspace, size_t workspace_bytes, void* stream) {
    if (int rc = paged_checked(fn, cache)) return rc;
    if (!O) return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer", fn);
    const int64_t dense[6] = {(int64_t)Hq * S * 128, (int64_t)S * 128, 128, (int64_t)Hq * S * 128, (int64_t)S * 128, 128};
    const int64_t* st = strides ? strides : dense;
    if (int rc = paged_queries_checked(fn, cache, Q, Hq, S, 0, st, 6, scale)) return rc;
    if (!aligned16(O)) return fail(MI355_ERR_BAD_ARGUMENT, "%s: O must be 16-byte aligned", fn);
    // (the account of many rows is made by mi355_fmha_key_weights' kernel)
    if ((int64_t)cache->B * cache->Hkv * ((int64_t)(Hq / cache->Hkv) * S + (int64_t)cache->max_pages * cache->page_size / 256 + 1) > kMostWorkgroups ||
        (mi355::fmha_paged_many_rows(*cache, Hq, S) && !mi355::paged_rows_fits(*cache, Hq, S)) ||
        (cache->weights && !mi355::fmha_paged_keeps_scores(*cache, Hq, S) && mi355::key_weights_workgroups(*cache, Hq, S, 0) > kMostWorkgroups / 2))
        return fail(MI355_ERR_UNSUPPORTED, "%s: %d sequences of %d rows over up to %lld keys are more than a call takes", fn, cache->B, S,
                    (long long)cache->max_pages * cache->page_size);
    if ((S > 1 && st[5] < 128) || (Hq > 1 && st[4] < 128) || (cache->B > 1 && st[3] < 128))
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: rows of O overlap (o strides %lld, %lld, %lld)", fn, (long long)st[3], (long long)st[4], (long long)st[5]);
    if (int rc = workspace_checked(fn, mi355::fmha_paged_workspace(*cache, Hq, S, LSE != nullptr, parents != nullptr), workspace, workspace_bytes)) return rc;
    const long l[6] = {(long)st[0], (long)st[1], (long)st[2], (long)st[3], (long)st[4], (long)st[5]};
    const hipError_t e = mi355::fmha_paged_dispatch(*cache, Q, O, LSE, Hq, S, l, scale, parents, (long)parents_batch, workspace, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : hip_fail(e, fn);
}

int mi355_fmha_paged(const mi355_paged_kv* cache, const void* Q, void* O, float* LSE, int Hq, int S, const int64_t* strides, float scale,
                     void* workspace, size_t workspace_bytes, void* stream) {
    return fmha_paged_impl("mi355_fmha_paged", cache, Q, O, LSE, Hq, S, strides, nullptr, 0, scale, workspace, workspace_bytes, stream);
}

size_t mi355_fmha_paged_tree_workspace_bytes(const mi355_paged_kv* cache, int Hq, int S) {
    if (!paged_sizes(cache) || !paged_rows(cache, Hq, S, 0)) return 0;   // (the call is refused)
    mi355_paged_kv c = *cache;
    c.weights = nullptr;
    return mi355::fmha_paged_workspace(c, Hq, S, true, true);
}

int mi355_fmha_paged_tree(const mi355_paged_kv* cache, const void* Q, void* O, float* LSE, int Hq, int S, const int64_t* strides, const int32_t* parents,
                          int64_t parents_batch, float scale, void* workspace, size_t workspace_bytes, void* stream) {
    const char* fn = "mi355_fmha_paged_tree";
    if (!cache || !parents) return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer", fn);
    if (S > mi355::kMostDrafted) return fail(MI355_ERR_UNSUPPORTED, "%s: a tree has at most %d tokens (got %d)", fn, mi355::kMostDrafted, S);
    if (parents_batch != 0 && parents_batch < S) return fail(MI355_ERR_BAD_ARGUMENT, "%s: parents_batch must be 0 or >= S (got %lld)", fn, (long long)parents_batch);
    mi355_paged_kv c = *cache;
    c.weights = nullptr;   // (no account is kept of drafted tokens)
    return fmha_paged_impl(fn, &c, Q, O, LSE, Hq, S, strides, parents, parents_batch, scale, workspace, workspace_bytes, stream);
}

int mi355_rope_paged(const mi355_paged_kv* cache, void* qkv, int S, int q_heads, int keep_keys, int64_t x_batch, int64_t x_row,
                     const float* cos_table, const float* sin_table, const int32_t* positions, int64_t pos_batch, int n_positions, void* stream) {
    const char* fn = "mi355_rope_paged";
    if (int rc = paged_checked(fn, cache)) return rc;
    if (!qkv || !cos_table || !sin_table || !positions) return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer", fn);
    if (S < 1 || q_heads < 0 || n_positions < 1) return fail(MI355_ERR_BAD_ARGUMENT, "%s: S, n_positions >= 1 and q_heads >= 0 required", fn);
    const int64_t heads = (int64_t)q_heads + 2 * (int64_t)cache->Hkv;
    if ((int64_t)cache->B * S > kMostWorkgroups || heads > 65535 * 32) return fail(MI355_ERR_UNSUPPORTED, "%s: too many tokens or heads", fn);
    if (x_row < heads * 128 || x_row % 8 || x_batch < 0 || x_batch % 8 || (cache->B > 1 && x_batch < heads * 128))
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: rows of qkv overlap or strides are no multiples of 8 (batch %lld, row %lld, %lld heads)", fn,
                    (long long)x_batch, (long long)x_row, (long long)heads);
    if (pos_batch != 0 && pos_batch < S) return fail(MI355_ERR_BAD_ARGUMENT, "%s: pos_batch must be 0 or >= S (got %lld)", fn, (long long)pos_batch);
    if (!aligned16(qkv) || !aligned16(cos_table) || !aligned16(sin_table))
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: pointers must be 16-byte aligned", fn);
    const hipError_t e = mi355::rope_paged_dispatch(*cache, qkv, S, q_heads, keep_keys, (long)x_batch, (long)x_row, cos_table, sin_table, positions,
                                                    (long)pos_batch, n_positions, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : hip_fail(e, fn);
}

size_t mi355_fmha_key_weights_workspace_bytes(const mi355_paged_kv* cache, int Hq, int S, int last_rows) {
    if (!paged_sizes(cache) || !paged_rows(cache, Hq, S, last_rows)) return 0;   // (the call is refused)
    return mi355::key_weights_workspace(*cache, Hq, S, last_rows);
}

int mi355_fmha_key_weights(const mi355_paged_kv* cache, const void* Q, const float* LSE, int Hq, int S, const int64_t* q_strides,
                           int last_rows, float scale, void* workspace, size_t workspace_bytes, void* stream) {
    const char* fn = "mi355_fmha_key_weights";
    if (int rc = paged_checked(fn, cache)) return rc;
    if (!LSE || !cache->weights) return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer", fn);
    if (last_rows < 0) return fail(MI355_ERR_BAD_ARGUMENT, "%s: last_rows must be >= 0 (got %d)", fn, last_rows);
    const int64_t dense[3] = {(int64_t)Hq * S * 128, (int64_t)S * 128, 128};
    const int64_t* st = q_strides ? q_strides : dense;
    if (int rc = paged_queries_checked(fn, cache, Q, Hq, S, last_rows, st, 3, scale)) return rc;
    if (mi355::key_weights_workgroups(*cache, Hq, S, last_rows) > kMostWorkgroups / 2)
        return fail(MI355_ERR_UNSUPPORTED, "%s: %d sequences of %d rows over up to %lld keys are more than a call takes", fn, cache->B, S,
                    (long long)cache->max_pages * cache->page_size);
    if (int rc = workspace_checked(fn, mi355::key_weights_workspace(*cache, Hq, S, last_rows), workspace, workspace_bytes)) return rc;
    const long l[3] = {(long)st[0], (long)st[1], (long)st[2]};
    const hipError_t e = mi355::key_weights_dispatch(*cache, Q, LSE, Hq, S, l, last_rows, scale, workspace, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : hip_fail(e, fn);
}

size_t mi355_cache_evict_workspace_bytes(const mi355_paged_kv* cache, int budget) {
    if (!paged_sizes(cache) || budget < 1) return 0;   // (the call is refused)
    return mi355::evict_workspace(*cache, budget);
}

int mi355_cache_evict(const mi355_paged_kv* cache, int budget, int recent, int32_t* lens_out, void* workspace, size_t workspace_bytes,
                      void* stream) {
    const char* fn = "mi355_cache_evict";
    if (int rc = paged_checked(fn, cache)) return rc;
    if (!cache->weights || !cache->key_positions || !lens_out) return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer", fn);
    if (budget < 1 || recent < 0) return fail(MI355_ERR_BAD_ARGUMENT, "%s: budget >= 1 and recent >= 0 required (got %d, %d)", fn, budget, recent);
    if (lens_out < cache->seq_lens + cache->B && cache->seq_lens < lens_out + cache->B)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: lens_out overlaps seq_lens", fn);
    if (int rc = workspace_checked(fn, mi355::evict_workspace(*cache, budget), workspace, workspace_bytes)) return rc;
    const hipError_t e = mi355::evict_dispatch(*cache, budget, recent, lens_out, workspace, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : hip_fail(e, fn);
}

int mi355_cache_keep_path(const mi355_paged_kv* cache, const int32_t* path, int length, int64_t path_batch, int32_t* lens_out, void* stream) {
    const char* fn = "mi355_cache_keep_path";
    if (int rc = paged_checked(fn, cache)) return rc;
    if (!cache->new_lens || !path || !lens_out) return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer", fn);
    if (length < 1 || length > (1 << 28)) return fail(MI355_ERR_BAD_ARGUMENT, "%s: length of a path must be in 1 .. 2^28 (got %d)", fn, length);
    if (path_batch < 0 || (cache->B > 1 && path_batch < length))
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: paths overlap (stride %lld, %d entries)", fn, (long long)path_batch, length);
    for (const int32_t* lens : {cache->seq_lens, cache->new_lens})
        if (lens_out < lens + cache->B && lens < lens_out + cache->B) return fail(MI355_ERR_BAD_ARGUMENT, "%s: lens_out overlaps seq_lens or new_lens", fn);
    const hipError_t e = mi355::keep_path_dispatch(*cache, path, length, (long)path_batch, lens_out, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : hip_fail(e, fn);
}

// ---- packed batches ----
size_t mi355_packed_plan_workspace_bytes(int B) { return B < 1 || B > 65535 ? 0 : mi355::packed_plan_workspace(B); }

int mi355_packed_plan(int32_t* block_table, int64_t table_stride, int32_t* seq_lens, const int32_t* new_lens, int32_t* next_positions, int32_t* free_pages,
                      int32_t* free_span, int B, int max_pages, int n_pages, int page_size, int rows, int32_t* offsets, int32_t* positions, int32_t* slots,
                      int32_t* taken, void* workspace, size_t workspace_bytes, void* stream) {
    const char* fn = "mi355_packed_plan";
    if (!block_table || !seq_lens || !new_lens || !free_pages || !free_span || !offsets || !taken || (rows > 0 && (!positions || !slots)))
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer", fn);
    if (B < 1 || max_pages < 1 || n_pages < 1 || rows < 0)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: B, max_pages, n_pages >= 1 and rows >= 0 required (got %d, %d, %d, %d)", fn, B, max_pages, n_pages, rows);
    if (page_size < 16 || page_size % 16 != 0)
        return fail(MI355_ERR_UNSUPPORTED, "%s: page_size must be a positive multiple of 16 (got %d)", fn, page_size);
    if (B > 65535 || rows > (1 << 28) || (int64_t)max_pages * page_size > (1 << 28) || (int64_t)n_pages * page_size > INT32_MAX || n_pages > (1 << 30) ||
        (int64_t)B * max_pages > INT32_MAX)
        return fail(MI355_ERR_UNSUPPORTED, "%s: %d sequences of up to %lld keys, %lld slots and %d rows are more than a call takes", fn, B,
                    (long long)max_pages * page_size, (long long)n_pages * page_size, rows);
    if (B > 1 && table_stride < max_pages)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: rows of the block table overlap (stride %lld, %d entries)", fn, (long long)table_stride, max_pages);
    if (next_positions && next_positions < seq_lens + B && seq_lens < next_positions + B)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: next_positions overlaps seq_lens (null: a token's position is the number of its key)", fn);
    if (int rc = workspace_checked(fn, mi355::packed_plan_workspace(B), workspace, workspace_bytes)) return rc;
    const hipError_t e = mi355::packed_plan_dispatch(block_table, (long)table_stride, seq_lens, new_lens, next_positions, free_pages, free_span, B, max_pages, n_pages,
                                                     page_size, rows, offsets, positions, slots, taken, workspace, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : hip_fail(e, fn);
}

int mi355_rope_packed(const mi355_paged_kv* pool, void* qkv, int rows, int q_heads, int keep_keys, int64_t x_row, const float* cos_table, const float* sin_table,
                      const int32_t* positions, const int32_t* slots, int n_positions, void* stream) {
    const char* fn = "mi355_rope_packed";
    if (!pool || !pool->pages || !qkv || !cos_table || !sin_table || !positions || !slots) return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer", fn);
    if (pool->dtype != MI355_DTYPE_FP16 && pool->dtype != MI355_DTYPE_BF16) return fail(MI355_ERR_BAD_ARGUMENT, "%s: unknown dtype %d", fn, pool->dtype);
    if (rows < 1 || q_heads < 0 || n_positions < 1 || pool->Hkv < 1 || pool->n_pages < 1)
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: rows, n_positions, Hkv, n_pages >= 1 and q_heads >= 0 required", fn);
    if (pool->page_size < 16 || pool->page_size % 16 != 0)
        return fail(MI355_ERR_UNSUPPORTED, "%s: page_size must be a positive multiple of 16 (got %d)", fn, pool->page_size);
    if (int rc = pool_checked(fn, pool)) return rc;
    const int64_t heads = (int64_t)q_heads + 2 * (int64_t)pool->Hkv;
    if (rows > kMostWorkgroups || heads > 65535 * 32 || (int64_t)pool->n_pages * pool->page_size > INT32_MAX)
        return fail(MI355_ERR_UNSUPPORTED, "%s: too many tokens, heads or slots", fn);
    if (x_row % 8 || (rows > 1 && x_row < heads * 128))
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: rows of qkv overlap or their stride is no multiple of 8 (%lld, %lld heads)", fn, (long long)x_row, (long long)heads);
    if (!aligned16(qkv) || !aligned16(cos_table) || !aligned16(sin_table))
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: pointers must be 16-byte aligned", fn);
    const hipError_t e = mi355::rope_packed_dispatch(*pool, qkv, rows, q_heads, keep_keys, (long)x_row, cos_table, sin_table, positions, slots, n_positions,
                                                     static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : hip_fail(e, fn);
}

static bool packed_sizes(int rows, int B, int Hq, int Hkv) {
    return rows >= 1 && B >= 1 && Hkv >= 1 && Hq >= Hkv && rows <= (1 << 28) && B <= (1 << 28) && Hq <= 65535 && mi355::packed_fits(rows, B, Hq, Hkv);
}

size_t mi355_fmha_packed_workspace_bytes(int rows, int B, int Hq, int Hkv) { return packed_sizes(rows, B, Hq, Hkv) ? mi355::packed_workspace(rows, B, Hq, Hkv) : 0; }

static int fmha_packed_impl(const char* fn, const void* Q, const void* K, const void* V, void* O, float* LSE, const int32_t* offsets, int rows, int B, int Hq, int Hkv,
                            const int64_t* strides, float scale, int causal, int dtype, void* workspace, size_t workspace_bytes, int variant, void* stream) {
    if (!Q || !K || !V || !O || !offsets) return fail(MI355_ERR_BAD_ARGUMENT, "%s: null pointer", fn);
    if (dtype != MI355_DTYPE_FP16 && dtype != MI355_DTYPE_BF16) return fail(MI355_ERR_BAD_ARGUMENT, "%s: unknown dtype %d", fn, dtype);
    if (rows < 1 || B < 1 || Hq < 1 || Hkv < 1) return fail(MI355_ERR_BAD_ARGUMENT, "%s: rows, B, Hq, Hkv must be >= 1 (got %d, %d, %d, %d)", fn, rows, B, Hq, Hkv);
    if (Hq % Hkv != 0) return fail(MI355_ERR_BAD_ARGUMENT, "%s: Hq (%d) must be a multiple of Hkv (%d)", fn, Hq, Hkv);
    if (!packed_sizes(rows, B, Hq, Hkv)) return fail(MI355_ERR_UNSUPPORTED, "%s: %d rows of %d sequences and %d heads are more than a call takes", fn, rows, B, Hq);
    if (!(scale > 0.f) || scale > 2.3e38f) return fail(MI355_ERR_BAD_ARGUMENT, "%s: scale must be positive and at most 2.3e38 (got %g)", fn, (double)scale);
    const int64_t dense[8] = {(int64_t)Hq * 128, 128, (int64_t)Hkv * 128, 128, (int64_t)Hkv * 128, 128, (int64_t)Hq * 128, 128};
    const int64_t* st = strides ? strides : dense;
    for (int i = 0; i < 8; ++i)
        if (st[i] < 0 || st[i] % 8 != 0)
            return fail(MI355_ERR_BAD_ARGUMENT, "%s: stride %d is %lld; strides must be non-negative multiples of 8 elements", fn, i, (long long)st[i]);
    for (int i = 0; i < 8; i += 2)
        if (st[i] >= (1 << 24)) return fail(MI355_ERR_UNSUPPORTED, "%s: row strides must be below 2^24 elements (got %lld)", fn, (long long)st[i]);
    if ((rows > 1 && st[6] < 128) || (Hq > 1 && st[7] < 128))
        return fail(MI355_ERR_BAD_ARGUMENT, "%s: rows of O overlap (o strides %lld, %lld)", fn, (long long)st[6], (long long)st[7]);
    if (!aligned16(Q) || !aligned16(K) || !aligned16(V) || !aligned16(O)) return fail(MI355_ERR_BAD_ARGUMENT, "%s: pointers must be 16-byte aligned", fn);
    if (int rc = workspace_checked(fn, mi355::packed_workspace(rows, B, Hq, Hkv), workspace, workspace_bytes)) return rc;
    const mi355::FmhaStrides sd = {0, (long)st[1], (long)st[0], 0, (long)st[3], (long)st[2], 0, (long)st[5], (long)st[4], 0, (long)st[7], (long)st[6]};
    const hipError_t e = mi355::packed_dispatch(Q, K, V, O, LSE, offsets, rows, B, Hq, Hkv, sd, scale, causal, dtype, workspace, variant, static_cast<hipStream_t>(stream));
    return e == hipSuccess ? 0 : hip_fail(e, fn);
}

int mi355_fmha_packed(const void* Q, const void* K, const void* V, void* O, float* LSE, const int32_t* offsets, int rows, int B, int Hq, int Hkv,
                      const int64_t* strides, float scale, int causal, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
    return fmha_packed_impl("mi355_fmha_packed", Q, K, V, O, LSE, offsets, rows, B, Hq, Hkv, strides, scale, causal, dtype, workspace, workspace_bytes, 0, stream);
}

int mi355_internal_fmha_packed_variant(const void* Q, const void* K, const void* V, void* O, float* LSE, const int32_t* offsets, int rows, int B, int Hq, int Hkv,
                                       const int64_t* strides, float scale, int causal, int dtype, void* workspace, size_t workspace_bytes, int variant,
                                       void* stream) {
    const char* fn = "mi355_internal_fmha_packed_variant";
    if (variant < 0 || variant > 2) return fail(MI355_ERR_BAD_ARGUMENT, "%s: unknown variant %d", fn, variant);
    return fmha_packed_impl(fn, Q, K, V, O, LSE, offsets, rows, B, Hq, Hkv, strides, scale, causal, dtype, workspace, workspace_bytes, variant, stream);
}

const char* mi355_last_error(void) { return g_err; }

int mi355_serving_version(void) { return MI355_SERVING_VERSION; }

}  // extern "C"
