// The 8-bit integer product for up to four token rows: a streaming mat-vec.
//
// Bound by the weight bytes, N * K once.  One CTA per SM; a warp takes one weight row at a time (two
// from two token rows on, so that a piece of the activation read from shared memory serves two), its
// lanes 16 bytes a step, eight steps under way; the activation codes lie in shared memory, and dp4a forms
// the exact int32 sums.  Activations that come as bf16 or fp16 are quantized by every CTA for itself
// while its first weights arrive (the arithmetic of the row quantizer, the same codes and scales): one
// launch instead of two.  The warps of a CTA are as many as divide the SM's share of the rows best.
#include "common.cuh"
#include "host.h"
#include "int8.cuh"

#include <atomic>

namespace lsg {

namespace {

constexpr int kGemvRows = 2;               // token rows
constexpr int kGemvSmem = 128 * 1024;      // of activation codes
constexpr int kSteps = 8;                  // 16-byte loads of a lane under way

template <typename T, int MR>
__device__ __forceinline__ void quantize_rows(const Int8Gemm& a, int8_t* codes, int ldq, float (&scale)[MR]) {
    __shared__ uint32_t part[32][MR];
    const int threads = blockDim.x, warps = threads >> 5;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const T* x = reinterpret_cast<const T*>(a.A);
    const bool whole = a.K % 8 == 0 && ((reinterpret_cast<uintptr_t>(x) | static_cast<uintptr_t>(a.lda * 2)) & 15) == 0;
#pragma unroll
    for (int m = 0; m < MR; ++m) {
        uint32_t top = 0;
        if (m < a.M) {
            const T* row = x + m * a.lda;
            if (whole) {
                for (int v = threadIdx.x; v < a.K / 8; v += threads) {
                    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(row) + v);
                    top = Int8In<T>::top(top, &raw);
                }
                top = Int8In<T>::top_bits(top);
            } else {
                for (int k = threadIdx.x; k < a.K; k += threads) top = max(top, __float_as_uint(fabsf(Int8In<T>::get(row, k))));
            }
        }
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) part[warp][m] = top;
    }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MR; ++m) {
        const RowScale r = row_scale(__reduce_max_sync(0xffffffffu, lane < warps ? part[lane][m] : 0u));
        scale[m] = r.scale;
        if (m >= a.M) continue;
        const T* row = x + m * a.lda;
        int8_t* q = codes + m * ldq;
        if (whole) {
            for (int v = threadIdx.x; v < a.K / 8; v += threads) {
                const uint4 raw = __ldg(reinterpret_cast<const uint4*>(row) + v);
                float f[8];
                Int8In<T>::unpack(&raw, f);
                reinterpret_cast<uint2*>(q)[v] = code8<T>(f, r);
            }
            if (threadIdx.x == 0 && (a.K & 8)) reinterpret_cast<uint2*>(q)[a.K / 8] = make_uint2(0, 0);
        } else {
            for (int k = threadIdx.x; k < ldq; k += threads)
                q[k] = k < a.K ? static_cast<int8_t>(code1<T>(Int8In<T>::get(row, k), r)) : int8_t(0);
        }
    }
}

// X: the activations' type, int8_t for codes.  MR: rows held (a.M <= MR).  RW: weight rows of a warp.
template <typename X, int MR, int RW>
__global__ void __launch_bounds__(RW == 1 ? 896 : 512, 1)
int8_gemv_kernel(const Int8Gemm a, int ldq) {
    extern __shared__ __align__(16) int8_t codes[];   // [a.M][ldq], zero behind K
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int threads = blockDim.x;
    const int stride = gridDim.x * warps * RW;
    int n0 = (blockIdx.x * warps + warp) * RW;
    pdl_launch_dependents();
    const int8_t* w[RW];
    auto rows_at = [&](int n) {
#pragma unroll
        for (int r = 0; r < RW; ++r) w[r] = a.B + static_cast<long long>(min(n + r, a.N - 1)) * a.ldb;
    };
    rows_at(n0);
    // the weights may be what the kernel in front writes, so only a hint goes out before the wait
    if (n0 < a.N)
#pragma unroll
        for (int r = 0; r < RW; ++r)
            for (int k = lane * 128; k < min(a.K, 4096); k += 4096) asm volatile("prefetch.global.L2 [%0];" ::"l"(w[r] + k));
    pdl_wait_prior();

    int4 wv[RW][kSteps];
    auto fetch = [&](int k0) {
#pragma unroll
        for (int r = 0; r < RW; ++r)
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int k = k0 + (i * 32 + lane) * 16;
                wv[r][i] = k < a.K ? __ldg(reinterpret_cast<const int4*>(w[r] + k)) : make_int4(0, 0, 0, 0);
            }
    };
    if (n0 < a.N) fetch(0);

    float scale[MR];
    if constexpr (sizeof(X) == 2) {
        quantize_rows<X, MR>(a, codes, ldq, scale);
    } else {
#pragma unroll
        for (int m = 0; m < MR; ++m) {
            scale[m] = m < a.M ? __ldg(a.scale_A + m) : 0.0f;
            if (m < a.M)
                for (int k = threadIdx.x * 16; k < ldq; k += threads * 16) {
                    int4 v = __ldg(reinterpret_cast<const int4*>(a.A + m * a.lda + k));
                    if (k + 16 > a.K) v = keep_bytes(v, a.K - k);
                    *reinterpret_cast<int4*>(codes + m * ldq + k) = v;
                }
        }
    }
    __syncthreads();

    constexpr int kSpan = kSteps * 512;
    for (; n0 < a.N; n0 += stride) {
        int acc[MR][RW];
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
            for (int r = 0; r < RW; ++r) acc[m][r] = 0;
        for (int k0 = 0;;) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int k = k0 + (i * 32 + lane) * 16;
                if (k < a.K) {
#pragma unroll
                    for (int m = 0; m < MR; ++m) {
                        if (m < a.M) {
                            const int4 xv = *reinterpret_cast<const int4*>(codes + m * ldq + k);
#pragma unroll
                            for (int r = 0; r < RW; ++r)
                                acc[m][r] = dp4a_ss(wv[r][i].x, xv.x, dp4a_ss(wv[r][i].y, xv.y,
                                            dp4a_ss(wv[r][i].z, xv.z, dp4a_ss(wv[r][i].w, xv.w, acc[m][r]))));
                        }
                    }
                }
            }
            k0 += kSpan;
            if (k0 >= a.K) break;
            fetch(k0);
        }
        const int n_out = n0;
        if (n0 + stride < a.N) {   // the next row is under way while this one is summed and written
            rows_at(n0 + stride);
            fetch(0);
        }
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
            for (int r = 0; r < RW; ++r) acc[m][r] = __reduce_add_sync(0xffffffffu, acc[m][r]);
        // lane m * RW + r writes row m of channel n0 + r
        int v = acc[0][0];
        float sa = scale[0];
#pragma unroll
        for (int m = 0; m < MR; ++m)
#pragma unroll
            for (int r = 0; r < RW; ++r)
                if (lane == m * RW + r) {
                    v = acc[m][r];
                    sa = scale[m];
                }
        const int m = lane / RW, n = n_out + lane % RW;
        if (m < a.M && n < a.N && lane < MR * RW)
            store_out(a.D, a.out_dtype, static_cast<size_t>(m) * a.N + n,
                      __fmul_rn(__fmul_rn(static_cast<float>(v), sa), __ldg(a.scale_B + n)));
    }
}

template <typename X, int MR, int RW>
int launch(const Int8Gemm& a, cudaStream_t s) {
    static std::atomic<bool> configured[64];
    int dev = 0;
    LSG_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_relaxed)) {
        LSG_CUDA_TRY(cudaFuncSetAttribute(int8_gemv_kernel<X, MR, RW>, cudaFuncAttributeMaxDynamicSharedMemorySize, kGemvSmem));
        if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_relaxed);
    }
    const int ldq = (a.K + 15) & ~15;
    const int sms = sm_count(), most = RW == 1 ? 28 : 16;
    const int share = static_cast<int>((static_cast<long long>(a.N) + static_cast<long long>(sms) * RW - 1) / (static_cast<long long>(sms) * RW));
    int warps = most;
    if (share <= most) {
        warps = share < 4 ? 4 : share;   // every row at once; four warps at least to quantize with
    } else {
        long long best = -1;
        for (int w = most; w >= most / 2; --w) {
            const long long idle = static_cast<long long>((share + w - 1) / w) * w - share;   // row slots left empty
            if (best < 0 || idle < best) {
                best = idle;
                warps = w;
            }
        }
    }
    const long long ctas = (static_cast<long long>(a.N) + warps * RW - 1) / (warps * RW);
    LSG_CUDA_TRY(launch_kernel(int8_gemv_kernel<X, MR, RW>, dim3(static_cast<unsigned>(ctas < sms ? ctas : sms)), dim3(warps * 32),
                               static_cast<size_t>(a.M) * ldq, s, true, a, ldq));
    return LSG_OK;
}

template <typename X>
int by_rows(const Int8Gemm& a, cudaStream_t s) {
    if (a.M == 1) return launch<X, 1, 1>(a, s);
    return launch<X, 2, 2>(a, s);
}

}  // namespace

bool int8_gemv_takes(int M, int K) {
    return M >= 1 && M <= kGemvRows && static_cast<long long>(M) * ((K + 15) & ~15) <= kGemvSmem;
}

int int8_gemv(const Int8Gemm& a, int x_dtype, cudaStream_t s) {
    if (x_dtype == LSG_DTYPE_BF16) return by_rows<__nv_bfloat16>(a, s);
    if (x_dtype == LSG_DTYPE_F16) return by_rows<__half>(a, s);
    return by_rows<int8_t>(a, s);
}

}  // namespace lsg
