// What the kernels of the 8-bit integer products share.
#pragma once

#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

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
// A few rows on a streaming mat-vec (int8_gemv.cu): whether a call of these sizes goes there, and the
// call, with A as codes (x_dtype < 0) or as bf16 / fp16 activations that it quantizes on the way (lda in
// values, scale_A unused).
bool int8_gemv_takes(int M, int K);
int int8_gemv(const Int8Gemm& a, int x_dtype, cudaStream_t s);
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

// Values of the quantizers' input types, eight at a time from 16-byte loads.
template <typename T> struct Int8In;
template <> struct Int8In<__nv_bfloat16> {
    static constexpr int kVecs = 1;   // 16-byte loads for eight values
    static __device__ __forceinline__ float get(const void* p, size_t i) {
        return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
    }
    static __device__ __forceinline__ void unpack(const uint4* v, float (&f)[8]) {
        const uint32_t w[4] = {v->x, v->y, v->z, v->w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
};
template <> struct Int8In<__half> {
    static constexpr int kVecs = 1;
    static __device__ __forceinline__ float get(const void* p, size_t i) {
        return __half2float(static_cast<const __half*>(p)[i]);
    }
    static __device__ __forceinline__ void unpack(const uint4* v, float (&f)[8]) {
        const uint32_t w[4] = {v->x, v->y, v->z, v->w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = h.x;
            f[2 * i + 1] = h.y;
        }
    }
};
template <> struct Int8In<float> {
    static constexpr int kVecs = 2;
    static __device__ __forceinline__ float get(const void* p, size_t i) { return static_cast<const float*>(p)[i]; }
    static __device__ __forceinline__ void unpack(const uint4* v, float (&f)[8]) {
        const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
    }
};

constexpr float kMagic = 12582912.0f;   // 1.5 * 2^23: adding it rounds to an integer, in the low byte

// The row's constants: y = x * mul is 127 x, moved by a power of two where 127 a or 1 / a would leave
// the range of fp32; den = a moved alike.
struct RowScale {
    float scale, mul, den, rcp;
    bool dead;   // all zero, or not finite: codes are 0
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
    RowScale r;
    const float a = __uint_as_float(amax_bits);
    const bool finite = amax_bits < 0x7F800000u;
    r.dead = !finite || amax_bits == 0;
    r.scale = finite ? a / 127.0f : __uint_as_float(0x7FC00000u);
    const float s = a > 0x1p100f ? 0x1p-64f : (a < 0x1p-100f ? 0x1p64f : 1.0f);
    r.mul = 127.0f * s;
    r.den = a * s;
    r.rcp = r.dead ? 0.0f : 1.0f / r.den;
    return r;
}
__device__ __forceinline__ uint32_t code_bits(float x, const RowScale& r) {
    const float y = x * r.mul;
    const float t = y * r.rcp;
    return __float_as_uint(fmaf(fmaf(-t, r.den, y), r.rcp, t) + kMagic);
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

#endif  // __CUDACC__

}  // namespace lsg
