// PyTorch extension module `lsg_torch_ops`: the host side of the eager operators of the 8-bit integer
// family, of the rows' ways to the experts and back, and of the MoE gradients (layerstormgemmkernels_b200/ops.py documents them) over the C ABI of
// liblsg_b200.so.  Calls of these operators at decode sizes cost their host work; argument checks,
// allocation and the call through ctypes take about 9 us, here they take about half.
// torch supplies tensors, the caching allocator and the current stream of the inputs' device.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <cstdint>
#include <stdexcept>
#include <string>
#include <tuple>

#include "lsg.h"

namespace {

using torch::Tensor;

[[noreturn]] void refuse(const char* op, const std::string& why) { throw std::runtime_error(std::string(op) + ": " + why); }

// The exceptions of layerstormgemmkernels_b200.capi for a status of the C ABI.
void check(int status) {
    if (status != LSG_OK) pybind11::module_::import("layerstormgemmkernels_b200.capi").attr("check")(status);
}

int code_of(at::ScalarType t) {
    return t == at::kBFloat16 ? LSG_DTYPE_BF16 : (t == at::kHalf ? LSG_DTYPE_F16 : LSG_DTYPE_F32);
}
bool is_half(const Tensor& t) { return t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf; }
bool is_float(const Tensor& t) { return is_half(t) || t.scalar_type() == at::kFloat; }

at::ScalarType out_type(const std::string& s) {
    if (s == "bf16" || s == "bfloat16") return at::kBFloat16;
    if (s == "fp16" || s == "float16") return at::kHalf;
    if (s == "fp32" || s == "float32") return at::kFloat;
    throw std::runtime_error("Unknown output dtype: " + s + ". Expected 'bf16', 'fp16' or 'fp32'.");
}

// What a call runs under: the device of `like` and the current stream there.
struct On {
    c10::cuda::CUDAGuard guard;
    void* stream;
    explicit On(const Tensor& like)
        : guard(like.device()), stream(at::cuda::getCurrentCUDAStream(like.get_device()).stream()) {}
};

// A CUDA matrix of one of the types whose rows are contiguous and do not overlap.
void need_rows(const char* op, const char* name, const Tensor& t, bool type_ok, const char* kinds) {
    if (!type_ok || !t.is_cuda()) refuse(op, std::string(name) + " must be " + kinds + " on CUDA");
    if (t.dim() != 2 || !(t.is_contiguous() || ((t.stride(1) == 1 || t.size(1) <= 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1)))))
        refuse(op, std::string(name) + " must be [rows, columns] with contiguous rows that do not overlap");
}
void need(const char* op, const char* name, const Tensor& t, at::ScalarType type, at::IntArrayRef shape, const Tensor& like) {
    if (t.scalar_type() != type || t.device() != like.device() || !t.is_contiguous() || t.sizes() != shape) {
        std::string dims;
        for (int64_t d : shape) dims += (dims.empty() ? "" : ", ") + std::to_string(d);
        refuse(op, std::string(name) + " must be contiguous " + c10::toString(type) + " [" + dims + "] on the inputs' device");
    }
}
void need_dense(const char* op, const char* name, const Tensor& t) {
    if (!is_float(t) || !t.is_cuda() || t.dim() != 2 || !t.is_contiguous())
        refuse(op, std::string(name) + " must be contiguous BF16, FP16 or FP32 [rows, H] on CUDA");
}
// int32 indices or fp32 weights of `n` pairs, in any shape
void need_pairs(const char* op, const char* name, const Tensor& t, at::ScalarType type, int64_t n, const Tensor& like) {
    if (t.scalar_type() != type || t.device() != like.device() || !t.is_contiguous() || t.numel() != n)
        refuse(op, std::string(name) + " must be " + std::to_string(n) + " contiguous values of " + c10::toString(type) + " on the rows' device");
}
// Sizes that the C ABI takes as int.
int as_int(const char* op, int64_t v) {
    if (v < 0 || v > 0x7fffffff) refuse(op, "a size is outside 0 .. 2^31 - 1");
    return static_cast<int>(v);
}

int64_t pad16(int64_t v) { return (v + 15) / 16 * 16; }
int64_t ld(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : std::max<int64_t>(t.size(1), 1); }
// of int8 codes; a single row has no next one, so its stride is what alignment asks for
int64_t ld_codes(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : pad16(t.size(1)); }

Tensor empty(at::IntArrayRef shape, at::ScalarType type, const Tensor& like) {
    return at::empty(shape, like.options().dtype(type));
}
// int8 [rows, K], rows 16 bytes apart or a multiple of it
Tensor code_rows(int64_t rows, int64_t K, const Tensor& like) {
    Tensor t = empty({rows, pad16(K)}, at::kChar, like);
    return K == pad16(K) ? t : t.narrow(1, 0, K);
}

}  // namespace

std::tuple<Tensor, Tensor> dynamic_int8_quant(const Tensor& input) {
    const char* op = "dynamic_int8_quant";
    need_rows(op, "input", input, is_half(input), "BF16 or FP16");
    const int64_t M = input.size(0), K = input.size(1);
    On on(input);
    Tensor codes = code_rows(M, K, input), scales = empty({M}, at::kFloat, input);
    check(lsg_dynamic_int8_quant(input.data_ptr(), ld(input), code_of(input.scalar_type()), codes.data_ptr(), pad16(K),
                                 static_cast<float*>(scales.data_ptr()), M, as_int(op, K), on.stream));
    return {codes, scales};
}

std::tuple<Tensor, Tensor> silu_mul_int8_quant(const Tensor& gate, const Tensor& up) {
    const char* op = "silu_mul_int8_quant";
    need_rows(op, "gate", gate, is_float(gate), "BF16, FP16 or FP32");
    need_rows(op, "up", up, is_float(up), "BF16, FP16 or FP32");
    if (gate.sizes() != up.sizes() || gate.scalar_type() != up.scalar_type() || gate.device() != up.device())
        refuse(op, "gate and up must have the same shape, dtype and device");
    const int64_t M = gate.size(0), K = gate.size(1);
    On on(gate);
    Tensor codes = code_rows(M, K, gate), scales = empty({M}, at::kFloat, gate);
    check(lsg_silu_mul_int8_quant(gate.data_ptr(), ld(gate), up.data_ptr(), ld(up), code_of(gate.scalar_type()), codes.data_ptr(),
                                  pad16(K), static_cast<float*>(scales.data_ptr()), M, as_int(op, K), on.stream));
    return {codes, scales};
}

Tensor int8_gemm(const Tensor& A, const Tensor& B, const Tensor& scale_A, const Tensor& scale_B, int64_t M, int64_t N, int64_t K,
                 const std::string& output_dtype) {
    const char* op = "int8_gemm";
    const at::ScalarType type = out_type(output_dtype);
    need_rows(op, "A", A, A.scalar_type() == at::kChar, "INT8");
    need_rows(op, "B", B, B.scalar_type() == at::kChar, "INT8");
    if (A.size(0) != M || A.size(1) != K) refuse(op, "A shape mismatch");
    if (B.size(0) != N || B.size(1) != K) refuse(op, "B shape mismatch");
    if (A.device() != B.device()) refuse(op, "A and B must be on one device");
    need(op, "scale_A", scale_A, at::kFloat, {M}, A);
    need(op, "scale_B", scale_B, at::kFloat, {N}, A);
    On on(A);
    Tensor D = empty({M, N}, type, A);
    lsg_int8_gemm_params p = {};
    p.M = as_int(op, M); p.N = as_int(op, N); p.K = as_int(op, K);
    p.A = A.data_ptr(); p.lda = ld_codes(A);
    p.B = B.data_ptr(); p.ldb = ld_codes(B);
    p.D = D.data_ptr();
    p.scale_A = static_cast<const float*>(scale_A.data_ptr());
    p.scale_B = static_cast<const float*>(scale_B.data_ptr());
    p.output_dtype = code_of(type);
    check(lsg_int8_gemm(&p, on.stream));
    return D;
}

Tensor int8_gemm_from_bf16(const Tensor& x, const Tensor& weight, const Tensor& weight_scales, const std::string& output_dtype) {
    const char* op = "int8_gemm_from_bf16";
    const at::ScalarType type = out_type(output_dtype);
    need_rows(op, "x", x, is_half(x), "BF16 or FP16");
    need_rows(op, "weight", weight, weight.scalar_type() == at::kChar, "INT8");
    const int64_t M = x.size(0), K = x.size(1), N = weight.size(0);
    if (weight.size(1) != K || weight.device() != x.device()) refuse(op, "weight must be [N, K] on x's device");
    need(op, "weight_scales", weight_scales, at::kFloat, {N}, x);
    On on(x);
    Tensor D = empty({M, N}, type, x), ws;
    lsg_int8_gemm_params p = {};
    p.M = as_int(op, M); p.N = as_int(op, N); p.K = as_int(op, K);
    p.A = x.data_ptr(); p.lda = ld(x);
    p.B = weight.data_ptr(); p.ldb = ld_codes(weight);
    p.D = D.data_ptr();
    p.scale_B = static_cast<const float*>(weight_scales.data_ptr());
    p.output_dtype = code_of(type);
    const size_t bytes = lsg_int8_gemm_from_bf16_workspace_bytes(p.M, p.K);
    if (bytes > 0) ws = empty({static_cast<int64_t>(bytes)}, at::kByte, x);
    check(lsg_int8_gemm_from_bf16(&p, code_of(x.scalar_type()), bytes > 0 ? ws.data_ptr() : nullptr, bytes, on.stream));
    return D;
}

Tensor int8_grouped_gemm(const Tensor& A_base, const Tensor& B_base, const Tensor& D_base, const Tensor& scale_A_base,
                         const Tensor& scale_B_base, const Tensor& expert_offsets, int64_t N, int64_t K,
                         const std::string& output_dtype) {
    const char* op = "int8_grouped_gemm";
    const at::ScalarType type = out_type(output_dtype);
    need_rows(op, "A_base", A_base, A_base.scalar_type() == at::kChar, "INT8");
    const int64_t T = A_base.size(0), E = B_base.dim() > 0 ? B_base.size(0) : 0;
    if (A_base.size(1) != K) refuse(op, "A_base.size(1) != K");
    need(op, "B_base", B_base, at::kChar, {E, N, K}, A_base);
    need(op, "D_base", D_base, type, {T, N}, A_base);
    need(op, "scale_A_base", scale_A_base, at::kFloat, {T}, A_base);
    need(op, "scale_B_base", scale_B_base, at::kFloat, {E, N}, A_base);
    need(op, "expert_offsets", expert_offsets, at::kInt, {E + 1}, A_base);
    On on(A_base);
    lsg_int8_grouped_gemm_params p = {};
    p.num_experts = as_int(op, E); p.N = as_int(op, N); p.K = as_int(op, K);
    p.A_base = A_base.data_ptr(); p.lda = ld_codes(A_base);
    p.B_base = B_base.data_ptr(); p.ldb = K;
    p.D_base = D_base.data_ptr();
    p.scale_A_base = static_cast<const float*>(scale_A_base.data_ptr());
    p.scale_B_base = static_cast<const float*>(scale_B_base.data_ptr());
    p.expert_offsets = static_cast<const int32_t*>(expert_offsets.data_ptr());
    p.output_dtype = code_of(type);
    check(lsg_int8_grouped_gemm(&p, as_int(op, T), on.stream));
    return D_base;
}

std::tuple<Tensor, Tensor> moe_permute_int8(const Tensor& hidden, const Tensor& inv_perm, int64_t top_k) {
    const char* op = "moe_permute_int8";
    need_rows(op, "hidden", hidden, is_half(hidden), "BF16 or FP16");
    if (top_k < 1) refuse(op, "top_k must be positive");
    const int64_t T = hidden.size(0), H = hidden.size(1), rows = T * top_k;
    need(op, "inv_perm", inv_perm, at::kInt, {rows}, hidden);
    On on(hidden);
    Tensor codes = code_rows(rows, H, hidden), scales = empty({rows}, at::kFloat, hidden);
    check(lsg_moe_permute_int8(hidden.data_ptr(), ld(hidden), code_of(hidden.scalar_type()),
                               static_cast<const int32_t*>(inv_perm.data_ptr()), as_int(op, T), as_int(op, top_k), as_int(op, H),
                               codes.data_ptr(), pad16(H), static_cast<float*>(scales.data_ptr()), on.stream));
    return {codes, scales};
}

Tensor int8_moe_ffn(const Tensor& hidden, const Tensor& expert_offsets, const Tensor& inv_perm, int64_t top_k, const Tensor& gate_up,
                    const Tensor& gate_up_scales, const Tensor& down, const Tensor& down_scales, const std::string& output_dtype) {
    const char* op = "int8_moe_ffn";
    const at::ScalarType type = out_type(output_dtype);
    need_rows(op, "hidden", hidden, is_half(hidden), "BF16 or FP16");
    if (top_k < 1) refuse(op, "top_k must be positive");
    if (gate_up.dim() != 3 || down.dim() != 3) refuse(op, "gate_up must be [E, 2I, H] and down [E, H, I]");
    const int64_t T = hidden.size(0), H = hidden.size(1), E = gate_up.size(0), I = down.size(2), rows = T * top_k;
    need(op, "gate_up", gate_up, at::kChar, {E, 2 * I, H}, hidden);
    need(op, "down", down, at::kChar, {E, H, I}, hidden);
    need(op, "gate_up_scales", gate_up_scales, at::kFloat, {E, 2 * I}, hidden);
    need(op, "down_scales", down_scales, at::kFloat, {E, H}, hidden);
    need(op, "expert_offsets", expert_offsets, at::kInt, {E + 1}, hidden);
    need(op, "inv_perm", inv_perm, at::kInt, {rows}, hidden);
    On on(hidden);
    Tensor D = empty({rows, H}, type, hidden), ws;
    lsg_int8_moe_ffn_params p = {};
    p.num_tokens = as_int(op, T); p.top_k = as_int(op, top_k); p.num_experts = as_int(op, E);
    p.H = as_int(op, H); p.I = as_int(op, I);
    p.hidden = hidden.data_ptr(); p.ld_hidden = ld(hidden); p.input_dtype = code_of(hidden.scalar_type());
    p.expert_offsets = static_cast<const int32_t*>(expert_offsets.data_ptr());
    p.inv_perm = static_cast<const int32_t*>(inv_perm.data_ptr());
    p.gate_up = gate_up.data_ptr();
    p.gate_up_scales = static_cast<const float*>(gate_up_scales.data_ptr());
    p.down = down.data_ptr();
    p.down_scales = static_cast<const float*>(down_scales.data_ptr());
    p.D = D.data_ptr();
    p.output_dtype = code_of(type);
    const size_t bytes = lsg_int8_moe_ffn_workspace_bytes(p.num_tokens, p.top_k, p.H, p.I);
    if (bytes > 0) ws = empty({static_cast<int64_t>(bytes)}, at::kByte, hidden);
    check(lsg_int8_moe_ffn(&p, bytes > 0 ? ws.data_ptr() : nullptr, bytes, on.stream));
    return D;
}

Tensor moe_permute(const Tensor& hidden, const Tensor& perm, int64_t top_k) {
    const char* op = "moe_permute";
    need_dense(op, "rows", hidden);
    const int64_t rows = perm.numel(), T = hidden.size(0), H = hidden.size(1);
    need_pairs(op, "perm", perm, at::kInt, rows, hidden);
    if (top_k < 1) refuse(op, "top_k must be positive");
    On on(hidden);
    Tensor out = empty({rows, H}, hidden.scalar_type(), hidden);
    check(lsg_moe_permute_dtype(hidden.data_ptr(), code_of(hidden.scalar_type()), static_cast<const int32_t*>(perm.data_ptr()),
                                as_int(op, rows), as_int(op, T), as_int(op, top_k), as_int(op, H), out.data_ptr(), on.stream));
    return out;
}

Tensor moe_unpermute(const Tensor& y, const Tensor& inv_perm, const Tensor& topk_weights, const c10::optional<std::string>& output_dtype) {
    const char* op = "moe_unpermute";
    need_dense(op, "rows", y);
    if (topk_weights.dim() != 2) refuse(op, "topk_weights must be [T, k]");
    const int64_t T = topk_weights.size(0), k = topk_weights.size(1), rows = y.size(0), H = y.size(1);
    need_pairs(op, "topk_weights", topk_weights, at::kFloat, T * k, y);
    need_pairs(op, "inv_perm", inv_perm, at::kInt, T * k, y);
    const at::ScalarType from = y.scalar_type(), to = output_dtype.has_value() ? out_type(*output_dtype) : from;
    On on(y);
    Tensor out = empty({T, H}, to, y);
    check(lsg_moe_unpermute_to(y.data_ptr(), code_of(from), static_cast<const int32_t*>(inv_perm.data_ptr()),
                               static_cast<const float*>(topk_weights.data_ptr()), as_int(op, rows), as_int(op, T), as_int(op, k),
                               as_int(op, H), out.data_ptr(), code_of(to), on.stream));
    return out;
}

Tensor moe_permute_backward(const Tensor& grad_rows, const Tensor& inv_perm, int64_t top_k) {
    const char* op = "moe_permute_backward";
    need_dense(op, "grad_rows", grad_rows);
    const int64_t pairs = inv_perm.numel(), H = grad_rows.size(1);
    if (top_k < 1 || pairs % top_k != 0) refuse(op, "inv_perm must hold top_k entries per token");
    need(op, "inv_perm", inv_perm, at::kInt, {pairs}, grad_rows);
    On on(grad_rows);
    Tensor out = empty({pairs / top_k, H}, grad_rows.scalar_type(), grad_rows);
    check(lsg_moe_permute_backward(grad_rows.data_ptr(), code_of(grad_rows.scalar_type()),
                                   static_cast<const int32_t*>(inv_perm.data_ptr()), as_int(op, grad_rows.size(0)),
                                   as_int(op, pairs / top_k), as_int(op, top_k), as_int(op, H), out.data_ptr(), on.stream));
    return out;
}

std::tuple<Tensor, Tensor> moe_unpermute_backward(const Tensor& grad_out, const Tensor& y, const Tensor& inv_perm,
                                                  const Tensor& topk_weights, const c10::optional<Tensor>& expert_offsets) {
    const char* op = "moe_unpermute_backward";
    need_dense(op, "grad_out", grad_out);
    need_dense(op, "y", y);
    if (y.scalar_type() != grad_out.scalar_type() || y.device() != grad_out.device() || y.size(1) != grad_out.size(1))
        refuse(op, "grad_out and y must have the same dtype, device and H");
    if (topk_weights.dim() != 2) refuse(op, "topk_weights must be [T, k]");
    const int64_t T = grad_out.size(0), H = grad_out.size(1), rows = y.size(0), k = topk_weights.size(1);
    need(op, "topk_weights", topk_weights, at::kFloat, {T, k}, y);
    need(op, "inv_perm", inv_perm, at::kInt, {T * k}, y);
    const int32_t* offsets = nullptr;
    int64_t experts = 0;
    if (expert_offsets.has_value()) {
        if (expert_offsets->dim() != 1 || expert_offsets->numel() < 2) refuse(op, "expert_offsets must be [E + 1]");
        need(op, "expert_offsets", *expert_offsets, at::kInt, expert_offsets->sizes(), y);
        offsets = static_cast<const int32_t*>(expert_offsets->data_ptr());
        experts = expert_offsets->numel() - 1;
    }
    On on(y);
    Tensor grad_y = empty({rows, H}, y.scalar_type(), y), grad_w = empty({T, k}, at::kFloat, y);
    check(lsg_moe_unpermute_backward(grad_out.data_ptr(), y.data_ptr(), code_of(y.scalar_type()),
                                     static_cast<const int32_t*>(inv_perm.data_ptr()),
                                     static_cast<const float*>(topk_weights.data_ptr()), offsets, as_int(op, experts),
                                     as_int(op, rows), as_int(op, T), as_int(op, k), as_int(op, H), grad_y.data_ptr(),
                                     static_cast<float*>(grad_w.data_ptr()), on.stream));
    return {grad_y, grad_w};
}

Tensor moe_route_backward(const Tensor& topk_idx, const Tensor& topk_weights, const Tensor& grad_weights, int64_t num_experts) {
    const char* op = "moe_route_backward";
    if (topk_idx.scalar_type() != at::kInt || !topk_idx.is_cuda() || topk_idx.dim() != 2 || !topk_idx.is_contiguous())
        refuse(op, "topk_idx must be contiguous int32 [T, k] on CUDA");
    const int64_t T = topk_idx.size(0), k = topk_idx.size(1);
    need(op, "topk_weights", topk_weights, at::kFloat, {T, k}, topk_idx);
    need(op, "grad_weights", grad_weights, at::kFloat, {T, k}, topk_idx);
    if (num_experts < 0) refuse(op, "num_experts must be positive");
    On on(topk_idx);
    Tensor out = empty({T, num_experts}, at::kFloat, topk_idx);
    check(lsg_moe_route_backward(static_cast<const int32_t*>(topk_idx.data_ptr()), static_cast<const float*>(topk_weights.data_ptr()),
                                 static_cast<const float*>(grad_weights.data_ptr()), as_int(op, T), as_int(op, num_experts),
                                 as_int(op, k), static_cast<float*>(out.data_ptr()), on.stream));
    return out;
}

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
    m.doc() = "Host side of the eager 8-bit integer, MoE row and MoE gradient operators; documented in layerstormgemmkernels_b200.ops.";
    m.def("dynamic_int8_quant", &dynamic_int8_quant);
    m.def("silu_mul_int8_quant", &silu_mul_int8_quant);
    m.def("int8_gemm", &int8_gemm);
    m.def("int8_gemm_from_bf16", &int8_gemm_from_bf16);
    m.def("int8_grouped_gemm", &int8_grouped_gemm);
    m.def("moe_permute_int8", &moe_permute_int8);
    m.def("int8_moe_ffn", &int8_moe_ffn);
    m.def("moe_permute", &moe_permute);
    m.def("moe_unpermute", &moe_unpermute);
    m.def("moe_permute_backward", &moe_permute_backward);
    m.def("moe_unpermute_backward", &moe_unpermute_backward);
    m.def("moe_route_backward", &moe_route_backward);
}
