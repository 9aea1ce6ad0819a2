// What the kernels of the 8-bit integer products share.
#pragma once

#include "common.cuh"

namespace lsg {

// |sum| <= 128 * 128 * K < 2^31, and K rounded up to 16 stays in the range
constexpr int kInt8MaxK = 131056;

struct Int8Gemm {
    const int8_t* A;            // [M, K] codes, row stride lda bytes (a multiple of 16)
    long long lda;
    const int8_t* B;            // [N, K], or E of them one behind the other; row stride ldb
    long long ldb;
    const float* scale_A;       // [M]
    const float* scale_B;       // [E * N]
    void* D;                    // [M, N]
    int out_dtype;
    int M, N, K, E;
    const int32_t* expert_offsets;   // null: dense
};

int int8_gemm(const Int8Gemm& a, cudaStream_t s);
// On the tensor cores (int8_mma.cu).  swiglu: B is [E, 2 N, K], gate rows in front of up rows, and D
// fp32 silu(gate) * up.
int int8_mma(const Int8Gemm& g, bool swiglu, cudaStream_t s);
int int8_quant_rows(const void* x, long long ldx, int dtype, int8_t* codes, long long ldq, float* scales, long long rows,
                    int K, const int32_t* inv, int top_k, int out_rows, cudaStream_t s);
int int8_quant_silu_mul(const void* gate, long long ldg, const void* up, long long ldu, int dtype, int8_t* codes,
                        long long ldq, float* scales, long long rows, int K, cudaStream_t s);

#if defined(__CUDACC__)

// The first n (1..15) bytes of sixteen; the others 0.  Only one operand of a product needs it.
__device__ __forceinline__ int4 keep_bytes(int4 v, int n) {
    auto part = [](int w, int left) { return left >= 4 ? w : (left <= 0 ? 0 : w & ((1 << (8 * left)) - 1)); };
    return make_int4(part(v.x, n), part(v.y, n - 4), part(v.z, n - 8), part(v.w, n - 12));
}

__device__ __forceinline__ void store_out(void* D, int dtype, size_t at, float v) {
    if (dtype == LSG_DTYPE_F32) static_cast<float*>(D)[at] = v;
    else if (dtype == LSG_DTYPE_F16) static_cast<__half*>(D)[at] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(D)[at] = __float2bfloat16_rn(v);
}

#endif  // __CUDACC__

}  // namespace lsg
