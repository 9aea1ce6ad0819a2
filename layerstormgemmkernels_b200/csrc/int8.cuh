// What the kernels of the 8-bit integer products share.
#pragma once

#include "common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

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

int int8_gemm(const Int8Gemm& a, bool early, cudaStream_t s);
// A few rows on a streaming mat-vec (int8_gemv.cu): whether a call of these sizes goes there, and the
// call, with A as codes (x_dtype < 0) or as bf16 / fp16 activations that it quantizes on the way (lda in
// values, scale_A unused).
bool int8_gemv_takes(int M, int N, int K);
int int8_gemv(const Int8Gemm& a, int x_dtype, cudaStream_t s);
// The expert block for a few rows on streaming mat-vecs (int8_moe_gemv.cu): whether these sizes go there, and both
// products.  first: A the hidden rows (lda in values), B [E, 2 N, K], D fp32 h [M, N]; second: A is h.
bool int8_moe_gemv_takes(int tokens, int top_k, int E, int H, int I);
int int8_moe_gemv(const Int8Gemm& first, int x_dtype, const int32_t* inv, int top_k, const Int8Gemm& second, cudaStream_t s);
// On the tensor cores (int8_mma.cu).  swiglu: B is [E, 2 N, K], gate rows in front of up rows, and D
// fp32 silu(gate) * up.  early: the launch in front on the stream is int8_quant_rows, which writes A.
int int8_mma(const Int8Gemm& g, bool swiglu, bool early, cudaStream_t s);
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

template <typename T> __device__ __forceinline__ T out_of(float v);
template <> __device__ __forceinline__ float out_of(float v) { return v; }
template <> __device__ __forceinline__ __half out_of(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 out_of(float v) { return __float2bfloat16_rn(v); }

// silu(g) * u in fp32.  With h = e^(-|g| / 2): g / (1 + h h) and, for negative g, (g h) h / (1 + h h): nothing
// overflows, and no step falls below the normal range before the result does (g / (1 + e^-g) is 0 from g = -88.8 on,
// silu -2.6e-37 there).  Off by 14 * 2^-24 at most: h by two ulp, which count twice over 1 + h h, six roundings.
// The quotient by the approximate division instruction (two ulp; 0 for denominators above 2^126, that is from
// g = -87.4 on) took 126 us for 8192 x 14336 bf16 pairs where this takes 143, by an exact division 209; the expert
// block shows nothing of it (4096 tokens of 8 experts of 4096 / 14336 1.1 ms, one token 13.0 us, all three).
__device__ __forceinline__ float silu_mul(float g, float u) {
    const float h = expf(-0.5f * fabsf(g)), d = fmaf(h, h, 1.0f);
    float r;                                        // d is in [1, 2]
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    r = fmaf(fmaf(-d, r, 1.0f), r, r);              // a step of Newton's method for 1 / d
    return (g < 0.0f ? g * h * h : g) * r * u;
}

// Four neighbouring values, aligned to themselves.
__device__ __forceinline__ void store_out4(void* D, int dtype, size_t at, const float (&v)[4]) {
    if (dtype == LSG_DTYPE_F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(D) + at) = make_float4(v[0], v[1], v[2], v[3]);
        return;
    }
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (dtype == LSG_DTYPE_F16) {
            const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
    *reinterpret_cast<uint2*>(static_cast<uint16_t*>(D) + at) = make_uint2(w[0], w[1]);
}

// Magnitudes order like their bit patterns, infinity and NaN on top.
__device__ __forceinline__ uint32_t max_halves(uint32_t m, const uint4* v) {
    const uint32_t w[4] = {v->x, v->y, v->z, v->w};
#pragma unroll
    for (int i = 0; i < 4; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
    return m;
}

// Values of the quantizers' input types, eight at a time from 16-byte loads.
template <typename T> struct Int8In;
template <> struct Int8In<__nv_bfloat16> {
    static constexpr int kVecs = 1;   // 16-byte loads for eight values
    static constexpr bool kOneFma = true;
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
    // running maximum of the magnitudes' bit patterns, two at a time, and its fp32 form
    static __device__ __forceinline__ uint32_t top(uint32_t m, const uint4* v) { return max_halves(m, v); }
    static __device__ __forceinline__ uint32_t top_bits(uint32_t m) { return max(m & 0xFFFFu, m >> 16) << 16; }
};
template <> struct Int8In<__half> {
    static constexpr int kVecs = 1;
    static constexpr bool kOneFma = false;
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
    static __device__ __forceinline__ uint32_t top(uint32_t m, const uint4* v) { return max_halves(m, v); }
    static __device__ __forceinline__ uint32_t top_bits(uint32_t m) {
        const __half_raw h = {static_cast<unsigned short>(max(m & 0xFFFFu, m >> 16))};
        return __float_as_uint(__half2float(h));
    }
};
template <> struct Int8In<float> {
    static constexpr int kVecs = 2;
    static constexpr bool kOneFma = true;    // and a look at whether it fell next to half-way
    static __device__ __forceinline__ float get(const void* p, size_t i) { return static_cast<const float*>(p)[i]; }
    static __device__ __forceinline__ void unpack(const uint4* v, float (&f)[8]) {
        const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(w[i]);
    }
    static __device__ __forceinline__ uint32_t top(uint32_t m, const uint4* v) {
        const uint32_t w[8] = {v[0].x, v[0].y, v[0].z, v[0].w, v[1].x, v[1].y, v[1].z, v[1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, w[i] & 0x7FFFFFFFu);
        return m;
    }
    static __device__ __forceinline__ uint32_t top_bits(uint32_t m) { return m; }
};

constexpr float kMagic = 12582912.0f;   // 1.5 * 2^23: adding it rounds to an integer, in the low byte

// The row's constants.  c is 127 / a rounded up: one fma(x, c, kMagic) rounds the exact x c to the
// nearest integer, and for bf16 that is the integer of 127 x / a: a quotient that is not half-way lies
// at least 2^-(9 + d) from half-way (d: by how many powers of two a exceeds x) and x c at most
// 2^-(15 + d) from the quotient; a quotient can be half-way only when a is 127 times a power of two,
// where c is exact, or when it is 63.5 (127 is prime), where c on the upper side takes it to 64, the
// even neighbour.  fp16 has other half-way cases (a = 381, x = 1.5): it forms the correctly rounded
// quotient from the exact 127 x instead.  fp32 values (of silu(g) u) have quotients as near half-way as 2^-33: where
// x c comes within 2^-16 above half-way (one value in 65536) two products and their rounding errors decide (settle).
// Rows below 2^-100 are moved up so that c stays finite.
struct RowScale {
    float scale, c, den, rcp;
    bool dead;   // all zero, or not finite: codes are 0
    bool tiny;
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
    RowScale r;
    const float a = __uint_as_float(amax_bits);
    const bool finite = amax_bits < 0x7F800000u;
    r.dead = !finite || amax_bits == 0;
    r.tiny = a < 0x1p-100f;
    r.scale = finite ? a / 127.0f : __uint_as_float(0x7FC00000u);
    r.den = r.dead ? 1.0f : (r.tiny ? a * 0x1p64f : a);
    r.c = __fdiv_ru(127.0f, r.den);
    r.rcp = 1.0f / r.den;
    return r;
}
template <typename T>
__device__ __forceinline__ uint32_t code_bits(float x, const RowScale& r) {
    if constexpr (!Int8In<T>::kOneFma) {
        const float y = x * 127.0f;
        const float t = y * r.rcp;
        return __float_as_uint(fmaf(fmaf(-t, r.den, y), r.rcp, t) + kMagic);
    } else {
        return __float_as_uint(fmaf(x, r.c, kMagic));
    }
}
// fp32: |x| c less the code's magnitude n.  Only from -1/2 to 2^-16 above it can n be one too large (c is 127 / a
// rounded up, so |x| c is never below the quotient).
constexpr float kDoubt = -0.5f + 0x1.1p-16f;
__device__ __forceinline__ float above_code(float x, uint32_t bits, const RowScale& r) {
    const float f = fmaf(x, r.c, kMagic - __uint_as_float(bits));
    return __uint_as_float(__float_as_uint(f) ^ (__float_as_uint(x) & 0x80000000u));
}
// The code in doubt: n, or n - 1 where 127 |x| / a is below n - 1/2 (or at it, and n is odd), that is by the sign of
// 254 |x| - (2 n - 1) a.  In units of 1 / 256 the products stay in range; their difference is exact, since they lie
// within a factor of two, and so are both products' rounding errors and the difference of these (at most 17 bits).
__device__ __forceinline__ uint32_t settle(float x, uint32_t bits, const RowScale& r) {
    if (above_code(x, bits, r) >= kDoubt) return bits;
    const float n = fabsf(__uint_as_float(bits) - kMagic), m = fabsf(x);
    const float w = 254.0f / 256.0f, h = fmaf(n, 2.0f / 256.0f, -1.0f / 256.0f);
    const float p = w * m, q = h * r.den;
    const float s = (p - q) + (fmaf(w, m, -p) - fmaf(h, r.den, -q));
    if (s > 0.0f || (s == 0.0f && (bits & 1) == 0)) return bits;
    return x < 0.0f ? bits + 1 : bits - 1;
}
template <typename T>
__device__ __forceinline__ uint8_t code1(float x, const RowScale& r) {
    if (r.dead) return 0;
    if (r.tiny) x *= 0x1p64f;
    uint32_t q = code_bits<T>(x, r);
    if constexpr (std::is_same<T, float>::value) q = settle(x, q, r);
    return static_cast<uint8_t>(q & 0xFFu);
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// Four fp32 values: few registers are held over the look at what is in doubt.
__device__ __forceinline__ uint32_t code4(const float (&f)[8], int at, const RowScale& r) {
    uint32_t q[4];
    float least = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        q[j] = code_bits<float>(f[at + j], r);
        least = fminf(least, above_code(f[at + j], q[j], r));
    }
    if (least < kDoubt) {
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = settle(f[at + j], q[j], r);
    }
    return pack4(q[0], q[1], q[2], q[3]);
}
template <typename T>
__device__ __forceinline__ uint2 code8(float (&f)[8], const RowScale& r) {
    if (r.dead) return make_uint2(0, 0);
    if (r.tiny) {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] *= 0x1p64f;
    }
    if constexpr (std::is_same<T, float>::value) {
        const uint32_t low = code4(f, 0, r);
        return make_uint2(low, code4(f, 4, r));
    }
    uint32_t q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = code_bits<T>(f[j], r);
    return make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
}

#endif  // __CUDACC__

}  // namespace lsg
