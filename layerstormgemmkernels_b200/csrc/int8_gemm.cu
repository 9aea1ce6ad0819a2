// Products of 8-bit integers with a scale per token and per output channel:
//
//   D[m, n] = scale_A[m] * scale_B[n] * sum_k A[m, k] B[n, k]        A, B int8, the sum in int32
//
// dense, and for rows grouped by expert.  The sum is exact (128 * 128 * K stays below 2^31 for the K
// accepted here), so results do not depend on how K is cut; it is converted to fp32, multiplied by
// the two scales in fp32 and rounded once to the output type.
#include "common.cuh"
#include "host.h"
#include "int8.cuh"

namespace lsg {

namespace {

int check(const char* op, int K, const void* A, long long lda, const void* B, long long ldb, const void* D, int dt,
          const float* sa, const float* sb) {
    if (dt != LSG_DTYPE_BF16 && dt != LSG_DTYPE_F16 && dt != LSG_DTYPE_F32)
        return fail(LSG_ERR_UNSUPPORTED, "%s: output dtype must be bf16, fp16 or f32", op);
    if (K < 1 || K > kInt8MaxK)
        return fail(LSG_ERR_INVALID, "%s: need 1 <= K <= %d, where the int32 sums cannot overflow (K=%d)", op, kInt8MaxK, K);
    if (lda < K || ldb < K) return fail(LSG_ERR_INVALID, "%s: a row stride is smaller than K", op);
    if (!A || !B || !D) return fail(LSG_ERR_INVALID, "%s: null pointer", op);
    if (((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(B)) & 15) || lda % 16 || ldb % 16)
        return fail(LSG_ERR_ALIGNMENT, "%s: operand rows must start on 16-byte boundaries", op);
    if ((reinterpret_cast<uintptr_t>(D) & (dt == LSG_DTYPE_F32 ? 3 : 1)) ||
        ((reinterpret_cast<uintptr_t>(sa) | reinterpret_cast<uintptr_t>(sb)) & 3))
        return fail(LSG_ERR_ALIGNMENT, "%s: the output or the scales are not aligned to their type", op);
    return LSG_OK;
}

}  // namespace

// Rows grouped by expert go to the tensor cores however few they are: one token, 8 of 128 experts of 1536 x 2048
// 9.1 us (2.8 TB/s), 2 of 8 of 4096 x 4096 10.0 (3.3).
int int8_gemm(const Int8Gemm& a, bool early, cudaStream_t s) {
    if (!a.expert_offsets && int8_gemv_takes(a.M, a.N, a.K)) return int8_gemv(a, -1, s);
    return int8_mma(a, false, early, s);
}

}  // namespace lsg

using namespace lsg;

namespace {
size_t a256(size_t v) { return (v + 255) & ~size_t(255); }
long long pad16(long long v) { return (v + 15) & ~15ll; }
}  // namespace

extern "C" int lsg_int8_gemm(const lsg_int8_gemm_params* p, void* stream) {
    if (!p) return fail(LSG_ERR_INVALID, "int8_gemm: null params");
    if (p->M < 0 || p->N < 0) return fail(LSG_ERR_INVALID, "int8_gemm: negative shape");
    if (p->M == 0 || p->N == 0) return LSG_OK;
    const int rc = check("int8_gemm", p->K, p->A, p->lda, p->B, p->ldb, p->D, p->output_dtype, p->scale_A, p->scale_B);
    if (rc != LSG_OK) return rc;
    if (!p->scale_A || !p->scale_B) return fail(LSG_ERR_INVALID, "int8_gemm: null pointer");
    Int8Gemm a = {};
    a.A = static_cast<const int8_t*>(p->A); a.lda = p->lda;
    a.B = static_cast<const int8_t*>(p->B); a.ldb = p->ldb;
    a.D = p->D; a.out_dtype = p->output_dtype;
    a.scale_A = p->scale_A; a.scale_B = p->scale_B;
    a.M = p->M; a.N = p->N; a.K = p->K; a.E = 1;
    return int8_gemm(a, false, static_cast<cudaStream_t>(stream));
}

extern "C" size_t lsg_int8_gemm_from_bf16_workspace_bytes(int M, int K) {
    if (M <= 0 || K <= 0 || (M == 1 && int8_gemv_takes(1, 1, K))) return 0;   // quantized inside the mat-vec
    return a256(static_cast<size_t>(M) * pad16(K)) + a256(static_cast<size_t>(M) * 4);
}

extern "C" int lsg_int8_gemm_from_bf16(const lsg_int8_gemm_params* p, int input_dtype, void* workspace,
                                       size_t workspace_bytes, void* stream) {
    if (!p) return fail(LSG_ERR_INVALID, "int8_gemm_from_bf16: null params");
    if (p->M < 0 || p->N < 0) return fail(LSG_ERR_INVALID, "int8_gemm_from_bf16: negative shape");
    if (input_dtype != LSG_DTYPE_BF16 && input_dtype != LSG_DTYPE_F16)
        return fail(LSG_ERR_UNSUPPORTED, "int8_gemm_from_bf16: input must be bf16 or fp16");
    if (p->M == 0 || p->N == 0) return LSG_OK;
    if (p->lda < p->K) return fail(LSG_ERR_INVALID, "int8_gemm_from_bf16: a row stride is smaller than K");
    // the activations may lie anywhere: the product reads their codes
    const long long ldq = pad16(p->K > 0 ? p->K : 0);
    int rc = check("int8_gemm_from_bf16", p->K, p->B, ldq, p->B, p->ldb, p->D, p->output_dtype, nullptr, p->scale_B);
    if (rc != LSG_OK) return rc;
    if (!p->A || !p->scale_B) return fail(LSG_ERR_INVALID, "int8_gemm_from_bf16: null pointer");
    if (reinterpret_cast<uintptr_t>(p->A) & 1) return fail(LSG_ERR_ALIGNMENT, "int8_gemm_from_bf16: the input is not aligned to its type");
    const size_t need = lsg_int8_gemm_from_bf16_workspace_bytes(p->M, p->K);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(LSG_ERR_WORKSPACE, "int8_gemm_from_bf16: workspace too small (have %zu, need %zu)",
                    workspace ? workspace_bytes : size_t(0), need);
    if (need > 0 && (reinterpret_cast<uintptr_t>(workspace) & 255))
        return fail(LSG_ERR_ALIGNMENT, "int8_gemm_from_bf16: workspace must be 256-byte aligned");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    Int8Gemm a = {};
    a.B = static_cast<const int8_t*>(p->B); a.ldb = p->ldb;
    a.D = p->D; a.out_dtype = p->output_dtype; a.scale_B = p->scale_B;
    a.M = p->M; a.N = p->N; a.K = p->K; a.E = 1;
    if (int8_gemv_takes(p->M, p->N, p->K)) {
        a.A = static_cast<const int8_t*>(p->A); a.lda = p->lda;
        return int8_gemv(a, input_dtype, s);
    }
    int8_t* codes = static_cast<int8_t*>(workspace);
    float* scales = reinterpret_cast<float*>(codes + a256(static_cast<size_t>(p->M) * ldq));
    a.A = codes; a.lda = ldq; a.scale_A = scales;
    rc = int8_quant_rows(p->A, p->lda, input_dtype, codes, ldq, scales, p->M, p->K, nullptr, 1, 0, s);
    if (rc != LSG_OK) return rc;
    return int8_gemm(a, true, s);
}

extern "C" int lsg_int8_grouped_gemm(const lsg_int8_grouped_gemm_params* p, int total_tokens, void* stream) {
    if (!p) return fail(LSG_ERR_INVALID, "int8_grouped_gemm: null params");
    if (p->num_experts < 0 || total_tokens < 0 || p->N < 0) return fail(LSG_ERR_INVALID, "int8_grouped_gemm: negative shape");
    if (p->num_experts > 1024) return fail(LSG_ERR_INVALID, "int8_grouped_gemm: at most 1024 experts (E=%d)", p->num_experts);
    if (p->num_experts == 0 || total_tokens == 0 || p->N == 0) return LSG_OK;
    const int rc = check("int8_grouped_gemm", p->K, p->A_base, p->lda, p->B_base, p->ldb, p->D_base, p->output_dtype,
                         p->scale_A_base, p->scale_B_base);
    if (rc != LSG_OK) return rc;
    if (!p->scale_A_base || !p->scale_B_base || !p->expert_offsets)
        return fail(LSG_ERR_INVALID, "int8_grouped_gemm: null pointer");
    if (static_cast<long long>(p->num_experts) * p->N > 0x7fffffffll)
        return fail(LSG_ERR_INVALID, "int8_grouped_gemm: more than 2^31 - 1 weight rows");
    Int8Gemm a = {};
    a.A = static_cast<const int8_t*>(p->A_base); a.lda = p->lda;
    a.B = static_cast<const int8_t*>(p->B_base); a.ldb = p->ldb;
    a.D = p->D_base; a.out_dtype = p->output_dtype;
    a.scale_A = p->scale_A_base; a.scale_B = p->scale_B_base;
    a.M = total_tokens; a.N = p->N; a.K = p->K; a.E = p->num_experts;
    a.expert_offsets = p->expert_offsets;
    return int8_gemm(a, false, static_cast<cudaStream_t>(stream));
}

namespace {
struct FfnPlan {
    size_t codes, scales, h, act, act_scales, total;
    long long ldh, ldi;
};
FfnPlan ffn_plan(long long rows, int H, int I) {
    FfnPlan f;
    f.ldh = pad16(H);
    f.ldi = pad16(I);
    f.codes = 0;
    f.scales = f.codes + a256(static_cast<size_t>(rows) * f.ldh);
    f.h = f.scales + a256(static_cast<size_t>(rows) * 4);
    f.act = f.h + a256(static_cast<size_t>(rows) * I * 4);
    f.act_scales = f.act + a256(static_cast<size_t>(rows) * f.ldi);
    f.total = f.act_scales + a256(static_cast<size_t>(rows) * 4);
    return f;
}
}  // namespace

extern "C" size_t lsg_int8_moe_ffn_workspace_bytes(int num_tokens, int top_k, int H, int I) {
    if (num_tokens <= 0 || top_k <= 0 || H <= 0 || I <= 0) return 0;
    return ffn_plan(static_cast<long long>(num_tokens) * top_k, H, I).total;
}

extern "C" int lsg_int8_moe_ffn(const lsg_int8_moe_ffn_params* p, void* workspace, size_t workspace_bytes, void* stream) {
    if (!p) return fail(LSG_ERR_INVALID, "int8_moe_ffn: null params");
    if (p->num_tokens < 0 || p->num_experts < 0 || p->H < 0 || p->I < 0) return fail(LSG_ERR_INVALID, "int8_moe_ffn: negative shape");
    if (p->num_experts > 1024) return fail(LSG_ERR_INVALID, "int8_moe_ffn: at most 1024 experts (E=%d)", p->num_experts);
    if (p->top_k < 1 || static_cast<long long>(p->num_tokens) * p->top_k > 0x7fffffffll)
        return fail(LSG_ERR_INVALID, "int8_moe_ffn: need top_k >= 1 and at most 2^31 - 1 pairs");
    if (p->input_dtype != LSG_DTYPE_BF16 && p->input_dtype != LSG_DTYPE_F16)
        return fail(LSG_ERR_UNSUPPORTED, "int8_moe_ffn: hidden must be bf16 or fp16");
    if (p->num_tokens == 0 || p->num_experts == 0) return LSG_OK;
    if (p->H < 1 || p->I < 1 || p->H % 16 != 0 || p->I % 16 != 0 || p->H > kInt8MaxK || p->I > kInt8MaxK)
        return fail(LSG_ERR_INVALID, "int8_moe_ffn: H and I must be positive multiples of 16 up to %d (H=%d, I=%d)", kInt8MaxK, p->H, p->I);
    if (static_cast<long long>(p->num_experts) * 2 * p->I > 0x7fffffffll || static_cast<long long>(p->num_experts) * p->H > 0x7fffffffll)
        return fail(LSG_ERR_INVALID, "int8_moe_ffn: more than 2^31 - 1 weight rows");
    if (!p->hidden || !p->inv_perm || !p->expert_offsets || !p->gate_up_scales || !p->down_scales)
        return fail(LSG_ERR_INVALID, "int8_moe_ffn: null pointer");
    if (p->ld_hidden < p->H) return fail(LSG_ERR_INVALID, "int8_moe_ffn: a row stride is smaller than the row");
    const int rows = p->num_tokens * p->top_k, H = p->H, I = p->I;
    const FfnPlan f = ffn_plan(rows, H, I);
    if (!workspace || workspace_bytes < f.total)
        return fail(LSG_ERR_WORKSPACE, "int8_moe_ffn: workspace too small (have %zu, need %zu)",
                    workspace ? workspace_bytes : size_t(0), f.total);
    if (reinterpret_cast<uintptr_t>(workspace) & 255)
        return fail(LSG_ERR_ALIGNMENT, "int8_moe_ffn: workspace must be 256-byte aligned");
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    int rc = check("int8_moe_ffn", H, ws, f.ldh, p->gate_up, H, ws, LSG_DTYPE_F32, p->gate_up_scales, nullptr);
    if (rc == LSG_OK) rc = check("int8_moe_ffn", I, ws, f.ldi, p->down, I, p->D, p->output_dtype, p->down_scales, nullptr);
    if (rc == LSG_OK && (reinterpret_cast<uintptr_t>(p->hidden) & 1))
        rc = fail(LSG_ERR_ALIGNMENT, "int8_moe_ffn: hidden is not aligned to its type");
    if (rc != LSG_OK) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    int8_t* codes = reinterpret_cast<int8_t*>(ws + f.codes);
    float* scales = reinterpret_cast<float*>(ws + f.scales);
    float* h = reinterpret_cast<float*>(ws + f.h);
    int8_t* act = reinterpret_cast<int8_t*>(ws + f.act);
    float* act_scales = reinterpret_cast<float*>(ws + f.act_scales);
    Int8Gemm a = {};
    a.A = codes; a.lda = f.ldh; a.B = static_cast<const int8_t*>(p->gate_up); a.ldb = H;
    a.D = h; a.out_dtype = LSG_DTYPE_F32; a.scale_A = scales; a.scale_B = p->gate_up_scales;
    a.M = rows; a.N = I; a.K = H; a.E = p->num_experts; a.expert_offsets = p->expert_offsets;
    Int8Gemm b = a;
    b.A = act; b.lda = f.ldi; b.B = static_cast<const int8_t*>(p->down); b.ldb = I;
    b.D = p->D; b.out_dtype = p->output_dtype; b.scale_A = act_scales; b.scale_B = p->down_scales;
    b.N = H; b.K = I;
    if (int8_moe_gemv_takes(p->num_tokens, p->top_k, p->num_experts, H, I)) {
        a.A = static_cast<const int8_t*>(p->hidden); a.lda = p->ld_hidden;
        b.A = reinterpret_cast<const int8_t*>(h); b.lda = I;
        return int8_moe_gemv(a, p->input_dtype, p->inv_perm, p->top_k, b, s);
    }
    rc = int8_quant_rows(p->hidden, p->ld_hidden, p->input_dtype, codes, f.ldh, scales, p->num_tokens, H, p->inv_perm, p->top_k, rows, s);
    if (rc != LSG_OK) return rc;
    rc = int8_mma(a, true, true, s);
    if (rc != LSG_OK) return rc;
    rc = int8_quant_rows(h, I, LSG_DTYPE_F32, act, f.ldi, act_scales, rows, I, nullptr, 1, 0, s);
    if (rc != LSG_OK) return rc;
    return int8_gemm(b, true, s);
}
