// The 8-bit expert block for up to eight rows (one token with its experts, or a few): two streaming mat-vecs.
//
//   h[r] = silu(g) * u,  (g, u) = codes(hidden[token of r]) . gate_up[expert of r]      fp32
//   D[r] = codes(h[r]) . down[expert of r]
//
// Bound by the weight bytes of the rows' experts, read once per row.  Jobs of two weight rows (a gate and its up
// row, or two channels of down) go round the SMs; a warp streams those of its jobs by bulk copies of 1 KB into a
// ring of 6 KB of its own and forms exact int32 sums with dp4a, so the bits are those of the tensor-core route.
// Every CTA quantizes the activations for itself while its first weights arrive: two launches instead of four.
// CTAs of the second product start beside those of the first one and have up to 14 MB of their weights in shared
// memory when h is there.
// One token, with the combination, 2 experts of 2048 / 2048: 13.7 us (four launches 19.5), 8 of 1024 / 512: 12.4
// (15.7), 8 of 2048 / 768: 17.9 (20.1), 8 of 4096 / 1536: 38.6 (42); 4 tokens, 2 of 8 of 1024 / 1024 each: 14.4 (17.7).
// The look at h values in doubt (settle) is 0.3 to 1 us of these.
// Tried: copies of 512 bytes (18.6 for the third), one weight row a job (20), the jobs of a CTA side by side, which
// needs the codes of fewer rows (19.0; 2 experts of 4096 / 8192 52 instead of 42), a scale loaded for each job (17.9).
#include "common.cuh"
#include "host.h"
#include "int8.cuh"

#include <algorithm>
#include <atomic>

namespace lsg {

namespace {

constexpr int kRows = 8;                   // rows (pairs of a token and an expert) at most
constexpr int kWarps = 16;
constexpr int kThreads = kWarps * 32;
constexpr int kBlock = 2;                  // weight rows of a job: a gate and an up row, or two channels
constexpr int kPiece = 1024;               // bytes of a weight row in a slot at most
constexpr int kSlots = 3;
constexpr int kSlotBytes = kBlock * kPiece;
constexpr int kRing = kSlots * kSlotBytes; // of a warp
// Shared memory of a CTA of the second product: over half of an SM's, and under what a CTA of the first leaves while its
// tokens are up to 13000 values (96 KB of ring and the codes, of 228 KB that hold both CTAs' 1.6 KB of their own too).
// So every SM takes one of them while the first product runs (behind it, with more values); where two fit, SMs that are
// done early take two.  48 registers for
// the same reason: one token, 2 experts of 4096 / 8192 42 us, with up to 64 registers 48, and 54 where two fit as well.
constexpr int kAlone = 116 * 1024;
constexpr int kCodes = 16384;              // bytes of codes at most

static_assert(kWarps * kRing + kCodes <= kAlone);

struct Args {
    Int8Gemm g;              // A: hidden [tokens, K] or h [M, K]; N: output channels; B: [E, N or 2 N, K]
    const int32_t* inv;      // row of a pair (first product)
    int top_k, tokens;       // rows of A
    unsigned int* status;
    long long limit;
};

// One row of activations and this thread's place in it: the warps are shared out evenly among the rows.
template <typename T>
struct RowPart {
    static constexpr int kVecs = Int8In<T>::kVecs;
    const T* row;
    int m, share, t, step;
    bool have, whole;

    __device__ __forceinline__ RowPart(const Int8Gemm& g, int rows) {
        share = kWarps;
        while (share > 1 && share * rows > kWarps) share >>= 1;
        const int warp = threadIdx.x >> 5;
        m = warp / share;
        t = (warp % share) * 32 + (threadIdx.x & 31);
        step = share * 32;
        have = m < rows;
        row = reinterpret_cast<const T*>(g.A) + (have ? m : 0) * g.lda;
        whole = ((reinterpret_cast<uintptr_t>(g.A) | static_cast<uintptr_t>(g.lda * sizeof(T))) & 15) == 0;
    }
    __device__ __forceinline__ void load(int v, uint4 (&raw)[kVecs]) const {
#pragma unroll
        for (int i = 0; i < kVecs; ++i) raw[i] = reinterpret_cast<const uint4*>(row)[v * kVecs + i];
    }
    // this thread's part of the row's largest magnitude (as bits)
    __device__ __forceinline__ uint32_t top(int K) const {
        uint32_t most = 0;
        if (have && whole) {
#pragma unroll 2
            for (int v = t; v < K / 8; v += step) {
                uint4 raw[kVecs];
                load(v, raw);
                most = Int8In<T>::top(most, raw);
            }
            most = Int8In<T>::top_bits(most);
        } else if (have) {
            for (int k = t; k < K; k += step) most = max(most, __float_as_uint(fabsf(Int8In<T>::get(row, k))));
        }
        return most;
    }
    __device__ __forceinline__ void codes(int K, const RowScale& r, int8_t* q) const {
        if (have && whole) {
#pragma unroll 2
            for (int v = t; v < K / 8; v += step) {
                uint4 raw[kVecs];
                load(v, raw);
                float f[8];
                Int8In<T>::unpack(raw, f);
                reinterpret_cast<uint2*>(q)[v] = code8<T>(f, r);
            }
        } else if (have) {
            for (int k = t; k < K; k += step) q[k] = static_cast<int8_t>(code1<T>(Int8In<T>::get(row, k), r));
        }
    }
};

// X: bf16 or fp16, the first product (hidden rows, silu(g) * u in fp32); float, the second one (rows of h).
// K is a multiple of 16.
template <typename X>
__global__ void __maxnreg__(48) int8_moe_gemv_kernel(const Args a) {
    constexpr bool kFirst = sizeof(X) == 2;
    constexpr int kOuts = kFirst ? kBlock / 2 : kBlock;   // output channels of a job
    extern __shared__ __align__(128) uint8_t smem[];   // [kWarps][kSlots][kBlock][kPiece], then codes [tokens][K]
    __shared__ uint64_t full[kWarps][kSlots];
    __shared__ float scale[kRows];
    __shared__ uint32_t part[kWarps];
    __shared__ int expert_of[kRows], source_of[kRows];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int M = a.g.M, N = a.g.N, K = a.g.K;
    uint8_t* ring = smem + warp * kRing;
    int8_t* codes = reinterpret_cast<int8_t*>(smem + kWarps * kRing);

    if (lane == 0) {
        for (int s = 0; s < kSlots; ++s) mbar_init(&full[warp][s], 1);
        mbar_fence_init();
    }
    // The first product waits here, then lets the second one start: that one finds offsets and weights in
    // place (all launches before the first product have ended) and waits for h alone.
    const RowPart<X> mine_of(a.g, a.tokens);
    if (kFirst) {
        pdl_wait_prior();
        pdl_launch_dependents();
    }
    // Warp r: the expert of row r.  Offsets are taken as a rising sequence: the first expert that ends behind r.
    if (warp < M) {
        const int below = __ldg(a.g.expert_offsets);
        int pair = 0;
        if constexpr (kFirst) pair = __ldg(a.inv + min(lane, M - 1));
        int found = a.g.E;
        for (int e0 = 0; e0 < a.g.E && found == a.g.E; e0 += 128) {
            int end[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) end[i] = __ldg(a.g.expert_offsets + min(e0 + i * 32 + lane, a.g.E - 1) + 1);
#pragma unroll
            for (int i = 3; i >= 0; --i)
                if (e0 + i * 32 + lane < a.g.E && end[i] > warp) found = e0 + i * 32 + lane;
            found = __reduce_min_sync(0xffffffffu, found);
        }
        if constexpr (kFirst) {
            const uint32_t hits = __ballot_sync(0xffffffffu, lane < M && pair == warp);
            pair = hits ? __ffs(hits) - 1 : 0;
        }
        if (lane == 0) {
            expert_of[warp] = found < a.g.E && below <= warp ? found : -1;
            source_of[warp] = kFirst ? pair / a.top_k : warp;
        }
    }
    if (kFirst) {
        const uint32_t top = __reduce_max_sync(0xffffffffu, mine_of.top(K));
        if (lane == 0) part[warp] = top;
    }
    __syncthreads();
    // rows with an expert lie side by side
    const uint32_t live = __ballot_sync(0xffffffffu, lane < M && expert_of[min(lane, M - 1)] >= 0);
    const int row0 = live ? __ffs(live) - 1 : 0, across = N / kOuts, jobs = __popc(live) * across;
    const int first = warp * gridDim.x + blockIdx.x, stride = kWarps * gridDim.x;   // round the SMs
    const int mine = first < jobs ? (jobs - 1 - first) / stride + 1 : 0;
    const int per_job = (K + kPiece - 1) / kPiece, pieces = mine * per_job;
    const int rows_on = stride / across, on = stride - rows_on * across;      // a step from job to job

    struct Place {
        int row, block, c;
    };
    Place p = {row0 + first / across, first % across, 0};
    auto next = [&](Place& at) {
        if (++at.c < per_job) return;
        at.c = 0;
        at.row += rows_on;
        at.block += on;
        if (at.block >= across) {
            at.block -= across;
            ++at.row;
        }
    };
    // lane i < kBlock: its weight row of a job, among those of all experts
    auto weight_row = [&](const Place& at) {
        const int base = at.block * kOuts;
        if (kFirst) return static_cast<long long>(expert_of[at.row]) * 2 * N + (lane / kOuts) * N + base + lane % kOuts;
        return static_cast<long long>(expert_of[at.row]) * N + base + lane;
    };
    auto copy = [&](const Place& at, int slot) {
        const int bytes = min(kPiece, K - at.c * kPiece);
        if (lane == 0) mbar_arrive_expect_tx(&full[warp][slot], bytes * kBlock);
        __syncwarp();
        if (lane < kBlock)
            bulk_g2s(ring + slot * kSlotBytes + lane * kPiece, a.g.B + weight_row(at) * K + at.c * kPiece, bytes,
                     &full[warp][slot]);
    };
    Place ahead = p;
    for (int i = 0; i < min(kSlots, pieces); ++i) {
        copy(ahead, i);
        next(ahead);
    }
    // lane i: the scale of weight row i % kBlock of this warp's job i / kBlock (of 16; a load per job would be waited for)
    auto channel_scales = [&](int job) {
        const int at = first + (job + lane / kBlock) * stride, on = lane % kBlock;
        if (at >= jobs) return 0.0f;
        const int row = at / across, base = (at - row * across) * kOuts;
        const long long w = static_cast<long long>(expert_of[row0 + row]) * (N * (kBlock / kOuts));
        return __ldg(a.g.scale_B + w + (on / kOuts) * N + base + on % kOuts);
    };
    float sb = channel_scales(0);
    if (!kFirst) {
        pdl_wait_prior();
        pdl_launch_dependents();
        const uint32_t top = __reduce_max_sync(0xffffffffu, mine_of.top(K));
        if (lane == 0) part[warp] = top;
        __syncthreads();
    }
    {
        const int m = mine_of.m;
        const uint32_t theirs = lane < mine_of.share ? part[min(m * mine_of.share + lane, kWarps - 1)] : 0u;
        const RowScale r = row_scale(__reduce_max_sync(0xffffffffu, theirs));
        if (mine_of.have && mine_of.t == 0) scale[m] = r.scale;
        mine_of.codes(K, r, codes + m * K);
    }
    __syncthreads();

    int acc[kBlock], slot = 0, job = 0;
    uint32_t lap = 0;
#pragma unroll
    for (int j = 0; j < kBlock; ++j) acc[j] = 0;
    for (int i = 0; i < pieces; ++i) {
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(&full[warp][slot], lap & 1, a.status, kDevWaitFull, 2000u, a.limit))) {
            // give up, but not before this copy and the ones behind it have landed
            for (int j = 0; j < kSlots && i + j < pieces; ++j) {
                const int other = (slot + j) % kSlots;
                mbar_wait_bounded(&full[warp][other], (lap + (slot + j >= kSlots ? 1 : 0)) & 1, a.status, kDevWaitFull);
            }
            return;
        }
        const int source = source_of[p.row];
        const int bytes = min(kPiece, K - p.c * kPiece);
        const int8_t* x = codes + source * K + p.c * kPiece;
        const uint8_t* w = ring + slot * kSlotBytes;
#pragma unroll
        for (int part_k = 0; part_k < kPiece; part_k += 512) {
            const int k = part_k + lane * 16;
            if (k < bytes) {
                const int4 xv = *reinterpret_cast<const int4*>(x + k);
#pragma unroll
                for (int j = 0; j < kBlock; ++j) {
                    const int4 wv = *reinterpret_cast<const int4*>(w + j * kPiece + k);
                    acc[j] = dp4a_ss(wv.x, xv.x, dp4a_ss(wv.y, xv.y, dp4a_ss(wv.z, xv.z, dp4a_ss(wv.w, xv.w, acc[j]))));
                }
            }
        }
        __syncwarp();
        if (i + kSlots < pieces) {
            copy(ahead, slot);
            next(ahead);
        }
        if (++slot == kSlots) {
            slot = 0;
            ++lap;
        }
        const Place done = p;
        next(p);
        if (p.c == 0) {
            // lane j: weight row j of the job
            int sum = 0;
#pragma unroll
            for (int j = 0; j < kBlock; ++j) {
                const int all = __reduce_add_sync(0xffffffffu, acc[j]);
                if (lane == j) sum = all;
                acc[j] = 0;
            }
            const float sb_own = __shfl_sync(0xffffffffu, sb, (job & (32 / kBlock - 1)) * kBlock + (lane & (kBlock - 1)));
            float v = __fmul_rn(__fmul_rn(static_cast<float>(sum), scale[source]), sb_own);
            if (kFirst) v = silu_mul(v, __shfl_down_sync(0xffffffffu, v, kOuts));
            if (lane < kOuts) store_out(a.g.D, a.g.out_dtype, static_cast<size_t>(done.row) * N + done.block * kOuts + lane, v);
            if ((++job & (32 / kBlock - 1)) == 0) sb = channel_scales(job);
        }
    }
}

template <typename X>
int launch(Args a, cudaStream_t s) {
    static std::atomic<bool> configured[64];
    int dev = 0;
    LSG_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_relaxed)) {
        LSG_CUDA_TRY(cudaFuncSetAttribute(int8_moe_gemv_kernel<X>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                          kAlone));
        if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_relaxed);
    }
    const long long jobs = static_cast<long long>(a.g.M) * a.g.N / (sizeof(X) == 2 ? kBlock / 2 : kBlock);
    const int ctas = static_cast<int>(std::min<long long>(sm_count(), jobs));
    a.status = device_status_word();
    a.limit = wait_limit_cycles();
    size_t smem = kWarps * kRing + static_cast<size_t>(a.tokens) * a.g.K;
    if (sizeof(X) == 4) smem = std::max(smem, static_cast<size_t>(kAlone));
    LSG_CUDA_TRY(launch_kernel(int8_moe_gemv_kernel<X>, dim3(static_cast<unsigned>(ctas)), dim3(kThreads), smem, s, true, a));
    return LSG_OK;
}

}  // namespace

// Rows that share an expert read its weights once each, and every CTA quantizes all tokens: with several tokens, only
// while at most a quarter of the weights (or 25 MB) is expected to be read again and the tokens are up to 8192 values.
// 4 tokens, 2 of 16 experts of 2048 / 2048 27.3 us here, 29.6 in four launches, 2 of 4 experts 26.3 and 23.5;
// 8 tokens of 2048, 1 of 64 experts of 2048 / 1024 23.1 and 21.9.
bool int8_moe_gemv_takes(int tokens, int top_k, int E, int H, int I) {
    const long long rows = static_cast<long long>(tokens) * top_k;
    if (rows > kRows || static_cast<long long>(tokens) * H > kCodes || rows * I > kCodes) return false;
    if (tokens == 1) return true;
    double missed = 1.0;                                        // that an expert is no token's
    for (int t = 0; t < tokens; ++t) missed *= std::max(0.0, 1.0 - static_cast<double>(top_k) / E);
    const double again = static_cast<double>(rows) - E * (1.0 - missed);
    return static_cast<long long>(tokens) * H <= kCodes / 2 && (4.0 * again <= rows || again * 3.0 * H * I <= 3 << 23);
}

int int8_moe_gemv(const Int8Gemm& first, int x_dtype, const int32_t* inv, int top_k, const Int8Gemm& second, cudaStream_t s) {
    Args a = {};
    a.g = first;
    a.inv = inv;
    a.top_k = top_k;
    a.tokens = first.M / top_k;
    const int rc = x_dtype == LSG_DTYPE_BF16 ? launch<__nv_bfloat16>(a, s) : launch<__half>(a, s);
    if (rc != LSG_OK) return rc;
    a.g = second;
    a.tokens = second.M;
    return launch<float>(a, s);
}

}  // namespace lsg
