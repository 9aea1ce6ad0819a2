// Quantizers of the 8-bit integer family: one scale per row (per token of an activation, per output
// channel of a weight).
//
//   a = max_k |x[k]|      scale = fl(a / 127)      q[k] = rne(127 x[k] / a)
//
// An all-zero row gets scale 0 and codes 0; a row with an infinity or a NaN gets scale NaN and
// codes 0, so that whatever it is multiplied with is NaN and not a number that looks right.
//
// The codes are those of the exact quotient (row_scale says how).  fl(x / scale) would not do: the
// scale is rounded, so quotients next to a half-way point fall on either side of it.
//
// The activation silu(g) * u of silu_mul stays in fp32 up to its code (rounding it to bf16 first
// moves one code in eighty).
//
// Memory bound: one CTA per row, the row held in registers between the maximum and the codes, so
// that every input byte is read once (4096 x 4096 bf16 6.5 us).  Rows that are not whole 16-byte
// pieces, or longer than 16384 values, are read twice, value by value, and bound by the instructions
// of that: 4096 x 4100 35 us, 2048 x 20000 90.  silu(g) * u is bound by its arithmetic: 8192 x 14336
// bf16 161 us and f32 218, for 587 MB and 1.06 GB.
#include "common.cuh"
#include "host.h"
#include "int8.cuh"

namespace lsg {

namespace {

struct RowQuantArgs {
    const void* x;        // [rows, K], row stride ldx values (gate of silu_mul)
    const void* up;
    long long ldx, ldu;
    int8_t* codes;        // row stride ldq bytes
    long long ldq;
    float* scales;
    int K;
    const int32_t* inv;   // scatter: [rows * top_k] destination rows; null = row to row
    int top_k;
    int out_rows;
};

// Bits of the largest magnitude of the CTA's values; magnitudes order like their bit patterns, with
// infinity and NaN on top, so nothing that is not finite is lost.
__device__ __forceinline__ uint32_t block_max_bits(uint32_t m) {
    __shared__ uint32_t part[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, n = (blockDim.x + 31) >> 5;
    m = __reduce_max_sync(0xffffffffu, m);
    if (n == 1) return m;
    if (lane == 0) part[warp] = m;
    __syncthreads();
    return __reduce_max_sync(0xffffffffu, lane < n ? part[lane] : 0u);
}

// A warp per row, V pieces of eight values per lane: short rows, no barrier.
template <typename T, int V>
__global__ void __launch_bounds__(256)
quant_short_rows_kernel(const RowQuantArgs a, long long rows) {
    pdl_wait_prior();
    pdl_launch_dependents();
    using In = Int8In<T>;
    constexpr int L = In::kVecs;
    const int lane = threadIdx.x & 31;
    const long long row = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int nvec = a.K >> 3;
    const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + row * a.ldx);
    uint4 raw[V][L];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int v = lane + i * 32;
#pragma unroll
        for (int l = 0; l < L; ++l) raw[i][l] = v < nvec ? __ldg(x + v * L + l) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) m = In::top(m, raw[i]);
    const RowScale r = row_scale(__reduce_max_sync(0xffffffffu, In::top_bits(m)));
    uint2 out[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float f[8];
        In::unpack(raw[i], f);
        out[i] = code8<T>(f, r);
    }
    const int copies = a.inv ? a.top_k : 1;
    for (int s = 0; s < copies; ++s) {
        const long long dst = a.inv ? __ldg(a.inv + row * a.top_k + s) : row;
        if (a.inv && (dst < 0 || dst >= a.out_rows)) continue;
        uint2* q = reinterpret_cast<uint2*>(a.codes + dst * a.ldq);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int v = lane + i * 32;
            if (v < nvec) q[v] = out[i];
        }
        if (lane == 0) a.scales[dst] = r.scale;
    }
}

// V pieces of eight values per thread.
template <typename T, bool SILU, int V>
__global__ void __launch_bounds__(V <= 2 ? 1024 : 512, SILU ? 2 : 0)
quant_rows_kernel(const RowQuantArgs a) {
    // in this order: what starts after this kernel may rely on everything in front of it having ended
    pdl_wait_prior();
    pdl_launch_dependents();
    using In = Int8In<T>;
    constexpr int L = In::kVecs;
    const long long row = blockIdx.x;
    const int nvec = a.K >> 3;
    const uint4* x = reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + row * a.ldx);
    uint4 raw[V][L];
    float h[SILU ? V : 1][8];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int v = threadIdx.x + i * blockDim.x;
#pragma unroll
        for (int l = 0; l < L; ++l) raw[i][l] = v < nvec ? __ldg(x + v * L + l) : make_uint4(0, 0, 0, 0);
    }
    if constexpr (SILU) {
        const uint4* up = reinterpret_cast<const uint4*>(static_cast<const T*>(a.up) + row * a.ldu);
        uint4 ur[V][L];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int v = threadIdx.x + i * blockDim.x;
#pragma unroll
            for (int l = 0; l < L; ++l) ur[i][l] = v < nvec ? __ldg(up + v * L + l) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float g[8], u[8];
            In::unpack(raw[i], g);
            In::unpack(ur[i], u);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                h[i][j] = silu_mul(g[j], u[j]);
                m = max(m, __float_as_uint(fabsf(h[i][j])));
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) m = In::top(m, raw[i]);
        m = In::top_bits(m);
    }
    const RowScale r = row_scale(block_max_bits(m));
    uint2 out[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        if constexpr (SILU) {
            out[i] = code8<float>(h[i], r);
        } else {
            float f[8];
            In::unpack(raw[i], f);
            out[i] = code8<T>(f, r);
        }
    }
    const int copies = a.inv ? a.top_k : 1;
    for (int s = 0; s < copies; ++s) {
        const long long dst = a.inv ? __ldg(a.inv + row * a.top_k + s) : row;
        if (a.inv && (dst < 0 || dst >= a.out_rows)) continue;
        uint2* q = reinterpret_cast<uint2*>(a.codes + dst * a.ldq);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int v = threadIdx.x + i * blockDim.x;
            if (v < nvec) q[v] = out[i];
        }
        if (threadIdx.x == 0) a.scales[dst] = r.scale;
    }
}

template <typename T, bool SILU>
__global__ void __launch_bounds__(256)
quant_rows_any_kernel(const RowQuantArgs a) {
    pdl_wait_prior();
    pdl_launch_dependents();
    const long long row = blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + row * a.ldx;
    const T* up = SILU ? static_cast<const T*>(a.up) + row * a.ldu : nullptr;
    auto value = [&](int k) {
        const float g = Int8In<T>::get(x, k);
        return SILU ? silu_mul(g, Int8In<T>::get(up, k)) : g;
    };
    uint32_t m = 0;
    for (int k = threadIdx.x; k < a.K; k += 256) m = max(m, __float_as_uint(fabsf(value(k))));
    const RowScale r = row_scale(block_max_bits(m));
    const int copies = a.inv ? a.top_k : 1;
    for (int k = threadIdx.x; k < a.K; k += 256) {
        const int8_t q = static_cast<int8_t>(SILU ? code1<float>(value(k), r) : code1<T>(value(k), r));
        for (int s = 0; s < copies; ++s) {
            const long long dst = a.inv ? __ldg(a.inv + row * a.top_k + s) : row;
            if (a.inv && (dst < 0 || dst >= a.out_rows)) continue;
            a.codes[dst * a.ldq + k] = q;
        }
    }
    if (threadIdx.x == 0)
        for (int s = 0; s < copies; ++s) {
            const long long dst = a.inv ? __ldg(a.inv + row * a.top_k + s) : row;
            if (a.inv && (dst < 0 || dst >= a.out_rows)) continue;
            a.scales[dst] = r.scale;
        }
}

template <typename T, bool SILU>
int launch_rows(const RowQuantArgs& a, long long rows, cudaStream_t s) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(a.x) | (SILU ? reinterpret_cast<uintptr_t>(a.up) : 0) |
                         static_cast<uintptr_t>(a.ldx * static_cast<long long>(sizeof(T))) |
                         (SILU ? static_cast<uintptr_t>(a.ldu * static_cast<long long>(sizeof(T))) : 0);
    const int nvec = a.K / 8;
    const dim3 grid(static_cast<unsigned>(rows));
    if ((at & 15) != 0 || a.K % 8 != 0 || nvec == 0 || nvec > 2048) {
        LSG_CUDA_TRY(launch_kernel(quant_rows_any_kernel<T, SILU>, grid, dim3(256), 0, s, true, a));
        return LSG_OK;
    }
    if constexpr (!SILU) {
        // Many short rows, a warp each: 32000 x 768 f32 36.6 -> 20 us, 16384 x 2048 bf16 17.8 -> 14.9.  Tokens
        // that go to several rows stay with the CTA form (4096 x 8 rows of 2048: 13.8 us against 16.2).
        if (rows >= 1024 && nvec <= 128) {
            LSG_CUDA_TRY(launch_kernel(quant_short_rows_kernel<T, 4>, dim3(static_cast<unsigned>((rows + 7) / 8)), dim3(256), 0, s, true, a, rows));
            return LSG_OK;
        }
        if (rows >= 1024 && nvec <= 256 && !a.inv) {
            LSG_CUDA_TRY(launch_kernel(quant_short_rows_kernel<T, 8>, dim3(static_cast<unsigned>((rows + 7) / 8)), dim3(256), 0, s, true, a, rows));
            return LSG_OK;
        }
    }
    // Four pieces a thread make small CTAs, so that loads of one row cover the arithmetic of others:
    // 4096 x 4096 bf16 7.6 us (10.0 with two pieces), 4096 x 14336 27.1 (38.9).  SiLU holds twice the
    // inputs and its results in registers: two pieces, and few enough of them that two rows are resident
    // (8192 x 14336 bf16 160 us, 188 with one row at a time).
    const int v = nvec <= 128 ? 1 : (SILU ? 2 : 4);
    const dim3 block(static_cast<unsigned>(((nvec + v - 1) / v + 31) / 32 * 32));
    if (v == 1) LSG_CUDA_TRY(launch_kernel(quant_rows_kernel<T, SILU, 1>, grid, block, 0, s, true, a));
    else if constexpr (SILU) LSG_CUDA_TRY(launch_kernel(quant_rows_kernel<T, SILU, 2>, grid, block, 0, s, true, a));
    else LSG_CUDA_TRY(launch_kernel(quant_rows_kernel<T, SILU, 4>, grid, block, 0, s, true, a));
    return LSG_OK;
}

// Shape and pointer checks shared by the entries; `ld` in values, ldq in bytes.
int check_rows(const char* op, int dtype, bool f32_ok, long long rows, int K, uintptr_t x, long long ld, const void* codes,
               long long ldq, const float* scales) {
    if (dtype != LSG_DTYPE_BF16 && dtype != LSG_DTYPE_F16 && !(f32_ok && dtype == LSG_DTYPE_F32))
        return fail(LSG_ERR_UNSUPPORTED, "%s: input must be bf16 or fp16%s", op, f32_ok ? " or f32" : "");
    if (rows < 0 || K < 0) return fail(LSG_ERR_INVALID, "%s: negative shape", op);
    if (rows > 0x7fffffffll) return fail(LSG_ERR_INVALID, "%s: more than 2^31 - 1 rows", op);
    if (ld < K || ldq < K) return fail(LSG_ERR_INVALID, "%s: a row stride is smaller than the row", op);
    if (ldq % 16 != 0 || (reinterpret_cast<uintptr_t>(codes) & 15))
        return fail(LSG_ERR_ALIGNMENT, "%s: code rows must start on 16-byte boundaries", op);
    if ((x & (dtype == LSG_DTYPE_F32 ? 3 : 1)) || (reinterpret_cast<uintptr_t>(scales) & 3))
        return fail(LSG_ERR_ALIGNMENT, "%s: a buffer is not aligned to its type", op);
    return LSG_OK;
}

}  // namespace

int int8_quant_rows(const void* x, long long ldx, int dtype, int8_t* codes, long long ldq, float* scales, long long rows,
                    int K, const int32_t* inv, int top_k, int out_rows, cudaStream_t s) {
    RowQuantArgs a = {};
    a.x = x; a.ldx = ldx; a.codes = codes; a.ldq = ldq; a.scales = scales; a.K = K;
    a.inv = inv; a.top_k = top_k; a.out_rows = out_rows;
    if (dtype == LSG_DTYPE_F32) return launch_rows<float, false>(a, rows, s);
    return dtype == LSG_DTYPE_F16 ? launch_rows<__half, false>(a, rows, s) : launch_rows<__nv_bfloat16, false>(a, rows, s);
}

int int8_quant_silu_mul(const void* gate, long long ldg, const void* up, long long ldu, int dtype, int8_t* codes,
                        long long ldq, float* scales, long long rows, int K, cudaStream_t s) {
    RowQuantArgs a = {};
    a.x = gate; a.ldx = ldg; a.up = up; a.ldu = ldu; a.codes = codes; a.ldq = ldq; a.scales = scales; a.K = K;
    if (dtype == LSG_DTYPE_F32) return launch_rows<float, true>(a, rows, s);
    return dtype == LSG_DTYPE_F16 ? launch_rows<__half, true>(a, rows, s) : launch_rows<__nv_bfloat16, true>(a, rows, s);
}

}  // namespace lsg

using namespace lsg;

extern "C" int lsg_dynamic_int8_quant(const void* x, long long ldx, int dtype, void* codes, long long ldq, float* scales,
                                      long long rows, int K, void* stream) {
    const int rc = check_rows("dynamic_int8_quant", dtype, false, rows, K, reinterpret_cast<uintptr_t>(x), ldx, codes, ldq, scales);
    if (rc != LSG_OK) return rc;
    if (rows == 0) return LSG_OK;
    if (!scales || (K > 0 && (!x || !codes))) return fail(LSG_ERR_INVALID, "dynamic_int8_quant: null pointer");
    return int8_quant_rows(x, ldx, dtype, static_cast<int8_t*>(codes), ldq, scales, rows, K, nullptr, 1, 0,
                           static_cast<cudaStream_t>(stream));
}

extern "C" int lsg_silu_mul_int8_quant(const void* gate, long long ldg, const void* up, long long ldu, int dtype,
                                       void* codes, long long ldq, float* scales, long long rows, int K, void* stream) {
    int rc = check_rows("silu_mul_int8_quant", dtype, true, rows, K, reinterpret_cast<uintptr_t>(gate) | reinterpret_cast<uintptr_t>(up),
                        ldg < ldu ? ldg : ldu, codes, ldq, scales);
    if (rc != LSG_OK) return rc;
    if (rows == 0) return LSG_OK;
    if (!scales || (K > 0 && (!gate || !up || !codes))) return fail(LSG_ERR_INVALID, "silu_mul_int8_quant: null pointer");
    return int8_quant_silu_mul(gate, ldg, up, ldu, dtype, static_cast<int8_t*>(codes), ldq, scales, rows, K,
                               static_cast<cudaStream_t>(stream));
}

extern "C" int lsg_moe_permute_int8(const void* hidden, long long ld, int dtype, const int32_t* inv_perm, int num_tokens,
                                    int top_k, int H, void* codes, long long ldq, float* scales, void* stream) {
    int rc = check_rows("moe_permute_int8", dtype, false, num_tokens, H, reinterpret_cast<uintptr_t>(hidden), ld, codes, ldq, scales);
    if (rc != LSG_OK) return rc;
    if (top_k < 1 || static_cast<long long>(num_tokens) * top_k > 0x7fffffffll)
        return fail(LSG_ERR_INVALID, "moe_permute_int8: need top_k >= 1 and at most 2^31 - 1 pairs");
    if (num_tokens == 0) return LSG_OK;
    if (!scales || !inv_perm || (H > 0 && (!hidden || !codes)))
        return fail(LSG_ERR_INVALID, "moe_permute_int8: null pointer");
    return int8_quant_rows(hidden, ld, dtype, static_cast<int8_t*>(codes), ldq, scales, num_tokens, H, inv_perm, top_k,
                           num_tokens * top_k, static_cast<cudaStream_t>(stream));
}
