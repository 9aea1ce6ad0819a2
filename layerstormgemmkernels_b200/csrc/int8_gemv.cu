// The 8-bit integer product for one or two token rows: a streaming mat-vec.
//
// Bound by the weight bytes, N * K once.  One CTA of 16 warps per SM; every warp streams its own weight
// rows, in pieces of up to 4 KB by bulk copies into a private ring of up to three slots (192 KB under way
// per SM from the first microsecond on), and forms the exact int32 sums with dp4a against the activation
// codes in shared memory.  Activations that come as bf16 or fp16 are quantized by every CTA for itself
// while its first weights arrive (the arithmetic of the row quantizer, the same codes and scales): one
// launch instead of two.  1 x 4096 x 4096 takes 5.0 us (two launches 6.7), 14336 x 4096 12.4 (4.8 TB/s with
// launch and tail), 16384 x 16384 45 (5.9 TB/s).  Loads into registers instead of the ring: 14.2 for the second.
#include "common.cuh"
#include "host.h"
#include "int8.cuh"

#include <algorithm>
#include <atomic>

namespace lsg {

namespace {

constexpr int kGemvRows = 2;               // token rows
constexpr int kGemvWarps = 16;
constexpr int kGemvThreads = kGemvWarps * 32;
constexpr int kPiece = 4096;               // bytes of a weight row in a slot
constexpr int kSlots = 3;
constexpr int kSlotBytes = kGemvWarps * kPiece;              // one slot of every warp
constexpr int kGemvSmem = 227 * 1024 - 1024;                 // slots and codes; the barriers are static
constexpr int kGemvCodes = kGemvSmem - kSlotBytes;           // codes leave one slot at least

template <typename T, int MR>
__device__ __forceinline__ void quantize_rows(const Int8Gemm& a, int8_t* codes, int ldq, float (&scale)[MR]) {
    __shared__ uint32_t part[kGemvWarps][MR];
    constexpr int threads = kGemvThreads, warps = kGemvWarps;
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

// X: the activations' type, int8_t for codes.  MR: rows held (a.M <= MR).
template <typename X, int MR>
__global__ void __launch_bounds__(kGemvThreads, 1)
int8_gemv_kernel(const Int8Gemm a, int ldq, int slots, unsigned int* status, long long limit) {
    extern __shared__ __align__(128) uint8_t smem[];   // [slots][kGemvWarps][kPiece], then codes [a.M][ldq], zero behind K
    __shared__ uint64_t full[kSlots][kGemvWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int8_t* codes = reinterpret_cast<int8_t*>(smem + slots * kSlotBytes);
    pdl_launch_dependents();
    const int first = blockIdx.x * kGemvWarps + warp, stride = gridDim.x * kGemvWarps;
    const int per_row = (ldq + kPiece - 1) / kPiece;
    const int pieces = first < a.N ? ((a.N - 1 - first) / stride + 1) * per_row : 0;
    // piece i of this warp: its bytes and where they lie
    auto piece_at = [&](int i, int& bytes) {
        const int row = i / per_row, c = i - row * per_row;
        bytes = min(kPiece, ldq - c * kPiece);
        return a.B + static_cast<long long>(first + row * stride) * a.ldb + c * kPiece;
    };
    auto copy = [&](int i, int slot) {
        int bytes;
        const int8_t* src = piece_at(i, bytes);
        mbar_arrive_expect_tx(&full[slot][warp], bytes);
        bulk_g2s(smem + slot * kSlotBytes + warp * kPiece, src, bytes, &full[slot][warp]);
    };
    if (lane == 0) {
        for (int s = 0; s < slots; ++s) mbar_init(&full[s][warp], 1);
        mbar_fence_init();
        // the weights may be what the kernel in front writes, so only a hint goes out before the wait
        for (int i = 0; i < min(slots, pieces); ++i) {
            int bytes;
            const int8_t* src = piece_at(i, bytes);
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src), "r"(bytes) : "memory");
        }
    }
    pdl_wait_prior();
    if (lane == 0)
        for (int i = 0; i < min(slots, pieces); ++i) copy(i, i);
    __syncwarp();

    float scale[MR];
    if constexpr (sizeof(X) == 2) {
        quantize_rows<X, MR>(a, codes, ldq, scale);
    } else {
#pragma unroll
        for (int m = 0; m < MR; ++m) {
            scale[m] = m < a.M ? __ldg(a.scale_A + m) : 0.0f;
            if (m < a.M)
                for (int k = threadIdx.x * 16; k < ldq; k += kGemvThreads * 16) {
                    int4 v = __ldg(reinterpret_cast<const int4*>(a.A + m * a.lda + k));
                    if (k + 16 > a.K) v = keep_bytes(v, a.K - k);
                    *reinterpret_cast<int4*>(codes + m * ldq + k) = v;
                }
        }
    }
    // lane i: the scale of this warp's row i (of 32; a load per row would stop the stream for its latency)
    auto channel_scales = [&](int row) {
        const long long at = first + static_cast<long long>(row + lane) * stride;
        return at < a.N ? __ldg(a.scale_B + at) : 0.0f;
    };
    float sb = channel_scales(0);
    __syncthreads();

    int acc[MR], slot = 0, c = 0, n = first, r = 0;
    uint32_t lap = 0;
#pragma unroll
    for (int m = 0; m < MR; ++m) acc[m] = 0;
    for (int i = 0; i < pieces; ++i) {
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full[slot][warp], lap & 1, status, kDevWaitFull, 2000u, limit))) {
            // give up, but not before this copy and the ones behind it have landed
            for (int j = 0; j < slots && i + j < pieces; ++j) {
                const int other = (slot + j) % slots;
                mbar_wait_bounded(&full[other][warp], (lap + (slot + j >= slots ? 1 : 0)) & 1, status, kDevWaitFull);
            }
            return;
        }
        const uint8_t* w = smem + slot * kSlotBytes + warp * kPiece;
        const int8_t* x = codes + c * kPiece;
        const int bytes = min(kPiece, ldq - c * kPiece);
        if (bytes == kPiece) {
#pragma unroll
            for (int k = lane * 16; k < kPiece; k += 512) {
                const int4 wv = *reinterpret_cast<const int4*>(w + k);
#pragma unroll
                for (int m = 0; m < MR; ++m)
                    if (m < a.M) {
                        const int4 xv = *reinterpret_cast<const int4*>(x + m * ldq + k);
                        acc[m] = dp4a_ss(wv.x, xv.x, dp4a_ss(wv.y, xv.y, dp4a_ss(wv.z, xv.z, dp4a_ss(wv.w, xv.w, acc[m]))));
                    }
            }
        } else {
            for (int k = lane * 16; k < bytes; k += 512) {
                const int4 wv = *reinterpret_cast<const int4*>(w + k);
#pragma unroll
                for (int m = 0; m < MR; ++m)
                    if (m < a.M) {
                        const int4 xv = *reinterpret_cast<const int4*>(x + m * ldq + k);
                        acc[m] = dp4a_ss(wv.x, xv.x, dp4a_ss(wv.y, xv.y, dp4a_ss(wv.z, xv.z, dp4a_ss(wv.w, xv.w, acc[m]))));
                    }
            }
        }
        __syncwarp();
        if (lane == 0 && i + slots < pieces) copy(i + slots, slot);
        if (++slot == slots) {
            slot = 0;
            ++lap;
        }
        if (++c == per_row) {
            // lane m writes token row m
            int v = 0;
            float sa = 0.0f;
#pragma unroll
            for (int m = 0; m < MR; ++m) {
                const int sum = __reduce_add_sync(0xffffffffu, acc[m]);
                if (lane == m) {
                    v = sum;
                    sa = scale[m];
                }
                acc[m] = 0;
            }
            const float sb_row = __shfl_sync(0xffffffffu, sb, r & 31);
            if (lane < a.M)
                store_out(a.D, a.out_dtype, static_cast<size_t>(lane) * a.N + n,
                          __fmul_rn(__fmul_rn(static_cast<float>(v), sa), sb_row));
            c = 0;
            n += stride;
            if ((++r & 31) == 0) sb = channel_scales(r);
        }
    }
}

template <typename X, int MR>
int launch(const Int8Gemm& a, cudaStream_t s) {
    static std::atomic<bool> configured[64];
    int dev = 0;
    LSG_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_relaxed)) {
        LSG_CUDA_TRY(cudaFuncSetAttribute(int8_gemv_kernel<X, MR>, cudaFuncAttributeMaxDynamicSharedMemorySize, kGemvSmem));
        if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_relaxed);
    }
    const int ldq = (a.K + 15) & ~15, sms = sm_count();
    const int codes = a.M * ldq;
    const int ctas = std::min(sms, (a.N + kGemvWarps - 1) / kGemvWarps);
    // no more slots than a warp has pieces
    const int pieces = ((a.N - 1) / (ctas * kGemvWarps) + 1) * ((ldq + kPiece - 1) / kPiece);
    const int slots = std::min(std::min(kSlots, pieces), (kGemvSmem - codes) / kSlotBytes);
    LSG_CUDA_TRY(launch_kernel(int8_gemv_kernel<X, MR>, dim3(static_cast<unsigned>(ctas)), dim3(kGemvThreads),
                               static_cast<size_t>(slots) * kSlotBytes + codes, s, true, a, ldq, slots, device_status_word(),
                               wait_limit_cycles()));
    return LSG_OK;
}

template <typename X>
int by_rows(const Int8Gemm& a, cudaStream_t s) {
    if (a.M == 1) return launch<X, 1>(a, s);
    return launch<X, 2>(a, s);
}

}  // namespace

// Two rows only while the weight is small: 4096 x 4096 7.4 us here and 8.2 on the tensor cores, 8192 x 4096
// 11.4 and 11.4, 14336 x 4096 15.6 and 14.4.
bool int8_gemv_takes(int M, int N, int K) {
    return M >= 1 && M <= kGemvRows && static_cast<long long>(M) * ((K + 15) & ~15) <= kGemvCodes &&
           (M == 1 || static_cast<long long>(N) * K < (1 << 25));
}

int int8_gemv(const Int8Gemm& a, int x_dtype, cudaStream_t s) {
    if (x_dtype == LSG_DTYPE_BF16) return by_rows<__nv_bfloat16>(a, s);
    if (x_dtype == LSG_DTYPE_F16) return by_rows<__half>(a, s);
    return by_rows<int8_t>(a, s);
}

}  // namespace lsg
