// The way of a token to its experts and back in fp16, bf16 and fp32, and its gradients.  With
// inv[t, s] the row of pair (token t, slot s), w the routing weights and L the loss:
//
//   permute     x_e[inv[t,s]] = x[t]                    dL/dx[t]          = sum_s dL/dx_e[inv[t,s]]
//   unpermute   out[t] = sum_s w[t,s] y[inv[t,s]]       dL/dy[inv[t,s]]   = w[t,s] dL/dout[t]
//                                                       dL/dw[t,s]        = < y[inv[t,s]], dL/dout[t] >
//   route       w[t,:] = softmax of the k chosen        dL/dl[t,idx[t,s]] = w[t,s] (dL/dw[t,s] - sum_r w[t,r] dL/dw[t,r])
//               logits (renormalising the top k of a                         0 for the experts not chosen
//               softmax leaves just that)
//
// A pair whose entry of inv lies outside [0, rows) has no row: it adds nothing, and its weight's
// gradient is 0.  Every sum is taken in fp32 in the order of the slots or by one CTA in a fixed
// order, without atomics: the same inputs give the same bits.
#include "common.cuh"
#include "host.h"

#include <type_traits>

namespace lsg {

namespace {

constexpr int kMaxSlots = 16;

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

// P values as one load or store: 16 bytes held as they are (as an array of 16-bit values the compiler
// gives every value a register of its own), or a single value where rows are not whole pieces.
template <typename T, int P> struct Piece {
    uint4 raw;
    __device__ __forceinline__ void zero() { raw = make_uint4(0, 0, 0, 0); }
    __device__ __forceinline__ void get(float (&f)[P]) const {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(w[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (std::is_same<T, __half>::value) {
                    const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                    f[2 * i] = h.x;
                    f[2 * i + 1] = h.y;
                } else {
                    f[2 * i] = __uint_as_float(w[i] << 16);
                    f[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
                }
            }
        }
    }
    __device__ __forceinline__ void set(const float (&f)[P]) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                w[i] = __float_as_uint(f[i]);
            } else if constexpr (std::is_same<T, __half>::value) {
                const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        raw = make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <typename T> struct Piece<T, 1> {
    T raw;
    __device__ __forceinline__ void zero() { raw = from_f<T>(0.0f); }
    __device__ __forceinline__ void get(float (&f)[1]) const { f[0] = to_f(raw); }
    __device__ __forceinline__ void set(const float (&f)[1]) { raw = from_f<T>(f[0]); }
};

// Pieces of a row that a thread has under way for every slot.  Single values are few bytes each, so up to
// 16 of them: 65000 tokens, two slots, 1001 bf16 values 375 us with one, 309 with four; 16384 tokens,
// eight slots 258 with one, 252 with two, 368 with four (registers).
template <int P, int K> constexpr int kAtOnce = P > 1 || K > 8 ? 1 : (K > 4 ? 2 : 4);

// The rows of a token's slots; -1: no row.
template <int K>
__device__ __forceinline__ void slot_rows(const int32_t* inv, size_t at, int rows, int k, int (&row)[K]) {
#pragma unroll
    for (int s = 0; s < K; ++s) {
        row[s] = s < k ? __ldg(inv + at + s) : -1;
        if (row[s] >= rows) row[s] = -1;
    }
}
// Four values of a 16-bit type, rounded from fp32 and stored as one: 16 bytes of fp32 rows leave as 8.
template <typename O>
__device__ __forceinline__ void store4(O* p, const float (&f)[4]) {
    alignas(8) O v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = from_f<O>(f[i]);
    *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(v);
}

// out[t] = sum over slots, in order, of (w ? w[t,s] : 1) * y[inv[t,s]], rounded once to O; k <= K.
template <typename T, typename O, int P, int K>
__global__ void __launch_bounds__(256)
moe_sum_slots_kernel(const Piece<T, P>* __restrict__ y, const int32_t* __restrict__ inv, const float* __restrict__ w,
                     int rows, int k, int per_row, O* __restrict__ out) {
    pdl_launch_dependents();
    pdl_wait_prior();
    const size_t t = blockIdx.x;
    int row[K];
    float ws[K];
    slot_rows(inv, t * k, rows, k, row);
#pragma unroll
    for (int s = 0; s < K; ++s) ws[s] = row[s] < 0 ? 0.0f : (w ? __ldg(w + t * k + s) : 1.0f);
    constexpr int U = kAtOnce<P, K>;
    for (int c0 = threadIdx.x; c0 < per_row; c0 += U * blockDim.x) {
        Piece<T, P> v[U][K];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = c0 + u * blockDim.x;
#pragma unroll
            for (int s = 0; s < K; ++s) {
                if (row[s] >= 0 && c < per_row) v[u][s] = y[static_cast<size_t>(row[s]) * per_row + c];
                else v[u][s].zero();
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = c0 + u * blockDim.x;
            if (c >= per_row) break;
            float acc[P];
#pragma unroll
            for (int i = 0; i < P; ++i) acc[i] = 0.0f;
#pragma unroll
            for (int s = 0; s < K; ++s) {
                float f[P];
                v[u][s].get(f);
#pragma unroll
                for (int i = 0; i < P; ++i) acc[i] = fmaf(ws[s], f[i], acc[i]);
            }
            if constexpr (P > 1 && !std::is_same<T, O>::value) {
                store4(out + (t * per_row + c) * P, acc);
            } else {
                Piece<O, P> o;
                o.set(acc);
                reinterpret_cast<Piece<O, P>*>(out)[t * per_row + c] = o;
            }
        }
    }
}

// out[row] = x[perm[row] / k]
template <typename T, int P>
__global__ void __launch_bounds__(256)
moe_copy_rows_kernel(const Piece<T, P>* __restrict__ x, const int32_t* __restrict__ perm, int tokens, int k, int per_row,
                     Piece<T, P>* __restrict__ out) {
    pdl_launch_dependents();
    pdl_wait_prior();
    const size_t row = blockIdx.x;
    const int pair = __ldg(perm + row);
    if (pair < 0 || pair / k >= tokens) return;
    const size_t src = static_cast<size_t>(pair / k) * per_row;
    for (int c = threadIdx.x; c < per_row; c += blockDim.x) out[row * per_row + c] = x[src + c];
}

// One CTA per token: grad_out[t] is read once for all its slots.  Bound by bytes (y read, grad_y
// written); small CTAs keep loads of other tokens under way while one sums its products: 16384 tokens
// of 2048 bf16 values, eight slots, 5.0 TB/s with 256 threads, 6.1 with 64.  Few tokens take 256
// threads (100 tokens: 64 would make the whole backward pass 12.0 us instead of 7.7).  Nine to sixteen
// slots do not fit the 80 registers of three CTAs: their pieces spill (240 bytes a thread), 4096 tokens of
// 2048 bf16 values, 16 slots 4.4 TB/s.
template <typename T, int P, int K>
__global__ void __launch_bounds__(256, 3)
moe_unpermute_backward_kernel(const Piece<T, P>* __restrict__ grad_out, const Piece<T, P>* __restrict__ y,
                              const int32_t* __restrict__ inv, const float* __restrict__ w,
                              const int32_t* __restrict__ rows_used, int rows, int k, int per_row,
                              Piece<T, P>* __restrict__ grad_y, float* __restrict__ grad_w) {
    pdl_launch_dependents();
    pdl_wait_prior();
    __shared__ float part[8][K];
    __shared__ float ws[K];
    const size_t t = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int row[K];
    float dot[K];
    if (threadIdx.x < K) ws[threadIdx.x] = threadIdx.x < k ? __ldg(w + t * k + threadIdx.x) : 0.0f;
    slot_rows(inv, t * k, rows, k, row);
#pragma unroll
    for (int s = 0; s < K; ++s) dot[s] = 0.0f;
    __syncthreads();
    constexpr int U = kAtOnce<P, K>;
    for (int c0 = threadIdx.x; c0 < per_row; c0 += U * blockDim.x) {
        Piece<T, P> v[U][K], g[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = c0 + u * blockDim.x;
            if (c < per_row) g[u] = grad_out[t * per_row + c];
            else g[u].zero();
#pragma unroll
            for (int s = 0; s < K; ++s) {
                if (row[s] >= 0 && c < per_row) v[u][s] = y[static_cast<size_t>(row[s]) * per_row + c];
                else v[u][s].zero();
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = c0 + u * blockDim.x;
            if (c >= per_row) break;
            float gf[P];
            g[u].get(gf);
#pragma unroll
            for (int s = 0; s < K; ++s) {
                if (row[s] >= 0) {
                    Piece<T, P> o;
                    float f[P], d[P];
                    v[u][s].get(f);
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        dot[s] = fmaf(f[i], gf[i], dot[s]);
                        d[i] = ws[s] * gf[i];
                    }
                    o.set(d);
                    grad_y[static_cast<size_t>(row[s]) * per_row + c] = o;
                }
            }
        }
    }
    // K sums over the warp at once: in the first log2(K) steps a lane hands over the half of the slots
    // that its partner keeps, so the sums take K - 1 + log2(32 / K) exchanges instead of 5 K
    int slot = 0;
#pragma unroll
    for (int h = K / 2, o = 16; h > 0; h >>= 1, o >>= 1) {
        const bool upper = (lane & o) != 0;
#pragma unroll
        for (int s = 0; s < h; ++s) {
            const float give = upper ? dot[s] : dot[s + h];
            const float keep = upper ? dot[s + h] : dot[s];
            dot[s] = keep + __shfl_xor_sync(0xffffffffu, give, o);
        }
        slot += upper ? h : 0;
    }
#pragma unroll
    for (int o = 16 / K; o > 0; o >>= 1) dot[0] += __shfl_xor_sync(0xffffffffu, dot[0], o);
    if ((lane & (32 / K - 1)) == 0) part[warp][slot] = dot[0];
    __syncthreads();
    if (threadIdx.x < k) {
        float v = 0.0f;
        for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) v += part[i][threadIdx.x];
        grad_w[t * k + threadIdx.x] = v;
    }
    // rows behind the last expert's belong to no pair
    if (rows_used) {
        const size_t used = static_cast<size_t>(max(__ldg(rows_used), 0));
        const size_t end = min((t + 1) * k, static_cast<size_t>(rows));
        for (size_t r = max(t * k, used); r < end; ++r) {
            Piece<T, P> z;
            z.zero();
            for (int c = threadIdx.x; c < per_row; c += blockDim.x) grad_y[r * per_row + c] = z;
        }
    }
}

// One warp per token.  Lanes 0..k-1 form the chosen experts' gradients, each with the other slots that name
// its expert added in order (routing names an expert once; a caller's own indices may name it twice); the
// row is cleared by whole warps and the k values go over it.
__global__ void __launch_bounds__(256)
moe_route_backward_kernel(const int32_t* __restrict__ idx, const float* __restrict__ w, const float* __restrict__ grad_w,
                          int T, int E, int k, float* __restrict__ grad_logits) {
    pdl_launch_dependents();
    pdl_wait_prior();
    const int lane = threadIdx.x & 31;
    const long long t = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    if (t >= T) return;
    const float wl = lane < k ? w[t * k + lane] : 0.0f;
    const float gl = lane < k ? grad_w[t * k + lane] : 0.0f;
    const int el = lane < k ? idx[t * k + lane] : -1;
    float* row = grad_logits + t * E;
    if ((reinterpret_cast<uintptr_t>(row) & 15) == 0) {
        for (int e = lane; e < E / 4; e += 32) reinterpret_cast<float4*>(row)[e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (lane < (E & 3)) row[(E & ~3) + lane] = 0.0f;
    } else {
        for (int e = lane; e < E; e += 32) row[e] = 0.0f;
    }
    float dot = wl * gl;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
    const float d = wl * (gl - dot);
    float sum = 0.0f;
    for (int s = 0; s < k; ++s) {
        const int es = __shfl_sync(0xffffffffu, el, s);
        const float ds = __shfl_sync(0xffffffffu, d, s);
        if (es == el) sum += ds;
    }
    __syncwarp();   // the zeros are written before the values
    if (el >= 0 && el < E) row[el] = sum;
}

// Threads of a token's CTA, at most `most`: the row's pieces in as few rounds, evenly.
int threads_for(int per_row, int most = 256) {
    const int rounds = (per_row + most - 1) / most;
    return rounds < 1 ? 32 : ((per_row + rounds - 1) / rounds + 31) / 32 * 32;
}

bool whole_pieces(int H, size_t size, uintptr_t at) { return (static_cast<size_t>(H) * size) % 16 == 0 && (at & 15) == 0; }

template <typename T, int P, int K, typename O>
int launch_sum(const void* y, const int32_t* inv, const float* w, int rows, int tokens, int k, int per_row, O* out, cudaStream_t s) {
    LSG_CUDA_TRY(launch_kernel(moe_sum_slots_kernel<T, O, P, K>, dim3(static_cast<unsigned>(tokens)), dim3(threads_for(per_row, tokens >= 2048 ? 128 : 256)), 0, s,
                               true, static_cast<const Piece<T, P>*>(y), inv, w, rows, k, per_row, out));
    return LSG_OK;
}
template <typename T, int P, int K>
int launch_unpermute_backward(const void* grad_out, const void* y, const int32_t* inv, const float* w, const int32_t* used, int rows,
                              int tokens, int k, int per_row, void* grad_y, float* grad_w, cudaStream_t s) {
    LSG_CUDA_TRY(launch_kernel(moe_unpermute_backward_kernel<T, P, K>, dim3(static_cast<unsigned>(tokens)),
                               dim3(threads_for(per_row, tokens >= 2048 ? 64 : 256)), 0, s, true, static_cast<const Piece<T, P>*>(grad_out),
                               static_cast<const Piece<T, P>*>(y), inv, w, used, rows, k, per_row,
                               static_cast<Piece<T, P>*>(grad_y), grad_w));
    return LSG_OK;
}

// K: slots held in registers, the next of 2, 4, 8, 16.
#define LSG_BY_SLOTS(fn, P, ...)                                                                       \
    (k <= 2 ? fn<T, P, 2>(__VA_ARGS__)                                                                 \
            : (k <= 4 ? fn<T, P, 4>(__VA_ARGS__) : (k <= 8 ? fn<T, P, 8>(__VA_ARGS__) : fn<T, P, 16>(__VA_ARGS__))))

// O: what the sums are rounded to, the rows' own type or 16 bits from fp32 rows.
template <typename T, typename O = T>
int sum_slots(const void* y, const int32_t* inv, const float* w, int rows, int tokens, int k, int H, void* out,
              cudaStream_t s) {
    constexpr int P = 16 / sizeof(T);
    O* o = static_cast<O*>(out);
    if (whole_pieces(H, sizeof(T), reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(out)))
        return LSG_BY_SLOTS(launch_sum, P, y, inv, w, rows, tokens, k, H / P, o, s);
    return LSG_BY_SLOTS(launch_sum, 1, y, inv, w, rows, tokens, k, H, o, s);
}

template <typename T>
int copy_rows(const void* x, const int32_t* perm, int rows, int tokens, int k, int H, void* out, cudaStream_t s) {
    constexpr int P = 16 / sizeof(T);
    const dim3 grid(static_cast<unsigned>(rows));
    if (whole_pieces(H, sizeof(T), reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)))
        LSG_CUDA_TRY(launch_kernel(moe_copy_rows_kernel<T, P>, grid, dim3(threads_for(H / P)), 0, s, true,
                                   static_cast<const Piece<T, P>*>(x), perm, tokens, k, H / P, static_cast<Piece<T, P>*>(out)));
    else
        LSG_CUDA_TRY(launch_kernel(moe_copy_rows_kernel<T, 1>, grid, dim3(threads_for(H)), 0, s, true,
                                   static_cast<const Piece<T, 1>*>(x), perm, tokens, k, H, static_cast<Piece<T, 1>*>(out)));
    return LSG_OK;
}

template <typename T>
int unpermute_backward(const void* grad_out, const void* y, const int32_t* inv, const float* w, const int32_t* used, int rows,
                       int tokens, int k, int H, void* grad_y, float* grad_w, cudaStream_t s) {
    constexpr int P = 16 / sizeof(T);
    if (whole_pieces(H, sizeof(T), reinterpret_cast<uintptr_t>(grad_out) | reinterpret_cast<uintptr_t>(y) | reinterpret_cast<uintptr_t>(grad_y)))
        return LSG_BY_SLOTS(launch_unpermute_backward, P, grad_out, y, inv, w, used, rows, tokens, k, H / P, grad_y, grad_w, s);
    return LSG_BY_SLOTS(launch_unpermute_backward, 1, grad_out, y, inv, w, used, rows, tokens, k, H, grad_y, grad_w, s);
}

int check_moe(const char* op, int dtype, int tokens, int k, int H, const void* a, const void* b, const void* c = nullptr,
              int most_slots = kMaxSlots) {
    if (dtype != LSG_DTYPE_BF16 && dtype != LSG_DTYPE_F16 && dtype != LSG_DTYPE_F32)
        return fail(LSG_ERR_UNSUPPORTED, "%s: dtype must be bf16, fp16 or f32", op);
    if (tokens < 0 || H < 0) return fail(LSG_ERR_INVALID, "%s: negative shape", op);
    if (k < 1 || k > most_slots) return fail(LSG_ERR_INVALID, "%s: need 1 <= top_k <= %d (k=%d)", op, most_slots, k);
    if (static_cast<long long>(tokens) * k > 0x7fffffffll)
        return fail(LSG_ERR_INVALID, "%s: more than 2^31 - 1 pairs", op);
    const uintptr_t size = dtype == LSG_DTYPE_F32 ? 4 : 2;
    if (((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c)) & (size - 1)) != 0)
        return fail(LSG_ERR_ALIGNMENT, "%s: a buffer is not aligned to its type", op);
    return LSG_OK;
}

}  // namespace

}  // namespace lsg

using namespace lsg;

#define LSG_BY_DTYPE(call)                                        \
    (dtype == LSG_DTYPE_F32 ? call<float> : dtype == LSG_DTYPE_F16 ? call<__half> : call<__nv_bfloat16>)

extern "C" int lsg_moe_permute_dtype(const void* hidden, int dtype, const int32_t* perm, int rows, int num_tokens,
                                     int top_k, int H, void* out, void* stream) {
    const int rc = check_moe("moe_permute", dtype, num_tokens, top_k, H, hidden, out, nullptr, 0x7fffffff);
    if (rc != LSG_OK) return rc;
    if (rows <= 0 || H == 0) return rows < 0 ? fail(LSG_ERR_INVALID, "moe_permute: negative shape") : LSG_OK;
    if (!hidden || !perm || !out) return fail(LSG_ERR_INVALID, "moe_permute: null pointer");
    // a thread a piece: 4096 x 8 rows of 768 bf16 13.9 us, 34.7 with a CTA a row
    if (dtype == LSG_DTYPE_BF16 && moe_gather_bf16_takes(hidden, out, H))
        return moe_gather_bf16(hidden, perm, rows, num_tokens, top_k, H, out, static_cast<cudaStream_t>(stream));
    return LSG_BY_DTYPE(copy_rows)(hidden, perm, rows, num_tokens, top_k, H, out, static_cast<cudaStream_t>(stream));
}

extern "C" int lsg_moe_unpermute_dtype(const void* y, int dtype, const int32_t* inv_perm, const float* topk_weights, int rows,
                                       int num_tokens, int top_k, int H, void* out, void* stream) {
    // bf16 in pairs: any number of slots, and 512 x 6 rows of 2048 take 2.7 us (3.8 with the slots in registers)
    const bool pairs = dtype == LSG_DTYPE_BF16 && moe_combine_bf16_takes(y, out, H);
    const int rc = check_moe("moe_unpermute", dtype, num_tokens, top_k, H, y, out, nullptr, pairs ? 0x7fffffff : kMaxSlots);
    if (rc != LSG_OK) return rc;
    if (rows < 0) return fail(LSG_ERR_INVALID, "moe_unpermute: negative shape");
    if (num_tokens == 0 || H == 0) return LSG_OK;
    if ((rows > 0 && !y) || !inv_perm || !topk_weights || !out) return fail(LSG_ERR_INVALID, "moe_unpermute: null pointer");
    if (pairs)
        return moe_combine_bf16(y, inv_perm, topk_weights, rows, num_tokens, top_k, H, out, static_cast<cudaStream_t>(stream));
    return LSG_BY_DTYPE(sum_slots)(y, inv_perm, topk_weights, rows, num_tokens, top_k, H, out, static_cast<cudaStream_t>(stream));
}

extern "C" int lsg_moe_unpermute_to(const void* y, int dtype, const int32_t* inv_perm, const float* topk_weights, int rows,
                                    int num_tokens, int top_k, int H, void* out, int out_dtype, void* stream) {
    if (out_dtype == dtype)
        return lsg_moe_unpermute_dtype(y, dtype, inv_perm, topk_weights, rows, num_tokens, top_k, H, out, stream);
    if (dtype != LSG_DTYPE_F32 || (out_dtype != LSG_DTYPE_BF16 && out_dtype != LSG_DTYPE_F16))
        return fail(LSG_ERR_UNSUPPORTED, "moe_unpermute: the output is of the rows' type, or bf16 or fp16 from f32 rows");
    int rc = check_moe("moe_unpermute", dtype, num_tokens, top_k, H, y, nullptr);
    if (rc == LSG_OK) rc = check_moe("moe_unpermute", out_dtype, num_tokens, top_k, H, out, nullptr);
    if (rc != LSG_OK) return rc;
    if (rows < 0) return fail(LSG_ERR_INVALID, "moe_unpermute: negative shape");
    if (num_tokens == 0 || H == 0) return LSG_OK;
    if ((rows > 0 && !y) || !inv_perm || !topk_weights || !out) return fail(LSG_ERR_INVALID, "moe_unpermute: null pointer");
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (out_dtype == LSG_DTYPE_F16)
        return sum_slots<float, __half>(y, inv_perm, topk_weights, rows, num_tokens, top_k, H, out, s);
    return sum_slots<float, __nv_bfloat16>(y, inv_perm, topk_weights, rows, num_tokens, top_k, H, out, s);
}

extern "C" int lsg_moe_permute_backward(const void* grad_rows, int dtype, const int32_t* inv_perm, int rows, int num_tokens,
                                        int top_k, int H, void* grad_hidden, void* stream) {
    const int rc = check_moe("moe_permute_backward", dtype, num_tokens, top_k, H, grad_rows, grad_hidden);
    if (rc != LSG_OK) return rc;
    if (rows < 0) return fail(LSG_ERR_INVALID, "moe_permute_backward: negative shape");
    if (num_tokens == 0 || H == 0) return LSG_OK;
    if ((rows > 0 && !grad_rows) || !inv_perm || !grad_hidden)
        return fail(LSG_ERR_INVALID, "moe_permute_backward: null pointer");
    return LSG_BY_DTYPE(sum_slots)(grad_rows, inv_perm, nullptr, rows, num_tokens, top_k, H, grad_hidden,
                                   static_cast<cudaStream_t>(stream));
}

extern "C" int lsg_moe_unpermute_backward(const void* grad_out, const void* y, int dtype, const int32_t* inv_perm,
                                          const float* topk_weights, const int32_t* expert_offsets, int num_experts, int rows,
                                          int num_tokens, int top_k, int H, void* grad_y, float* grad_weights, void* stream) {
    const int rc = check_moe("moe_unpermute_backward", dtype, num_tokens, top_k, H, grad_out, y, grad_y);
    if (rc != LSG_OK) return rc;
    if (rows < 0) return fail(LSG_ERR_INVALID, "moe_unpermute_backward: negative shape");
    if (rows > static_cast<long long>(num_tokens) * top_k)
        return fail(LSG_ERR_INVALID, "moe_unpermute_backward: more rows than (token, slot) pairs");
    if (expert_offsets && num_experts < 1) return fail(LSG_ERR_INVALID, "moe_unpermute_backward: num_experts must be positive");
    if (num_tokens == 0) return LSG_OK;
    if (!inv_perm || !topk_weights || !grad_weights || (H > 0 && (!grad_out || (rows > 0 && (!y || !grad_y)))))
        return fail(LSG_ERR_INVALID, "moe_unpermute_backward: null pointer");
    return LSG_BY_DTYPE(unpermute_backward)(grad_out, y, inv_perm, topk_weights,
                                            expert_offsets ? expert_offsets + num_experts : nullptr, rows, num_tokens, top_k, H,
                                            grad_y, grad_weights, static_cast<cudaStream_t>(stream));
}

extern "C" int lsg_moe_route_backward(const int32_t* topk_idx, const float* topk_weights, const float* grad_weights,
                                      int num_tokens, int num_experts, int top_k, float* grad_logits, void* stream) {
    if (num_tokens < 0) return fail(LSG_ERR_INVALID, "moe_route_backward: negative shape");
    if (num_experts < 1 || num_experts > 1024 || top_k < 1 || top_k > kMaxSlots || top_k > num_experts)
        return fail(LSG_ERR_INVALID, "moe_route_backward: need 1 <= top_k <= min(16, E) and E <= 1024 (E=%d, k=%d)",
                    num_experts, top_k);
    if (num_tokens == 0) return LSG_OK;
    if (!topk_idx || !topk_weights || !grad_weights || !grad_logits)
        return fail(LSG_ERR_INVALID, "moe_route_backward: null pointer");
    LSG_CUDA_TRY(launch_kernel(moe_route_backward_kernel, dim3(static_cast<unsigned>((static_cast<long long>(num_tokens) + 7) / 8)),
                               dim3(256), 0, static_cast<cudaStream_t>(stream), true, topk_idx, topk_weights, grad_weights,
                               num_tokens, num_experts, top_k, grad_logits));
    return LSG_OK;
}
