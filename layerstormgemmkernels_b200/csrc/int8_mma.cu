// The 8-bit integer products on the tensor cores: tcgen05.mma.kind::i8, int32 accumulators in tensor
// memory, scales and rounding on the way out.
//
// The weight is the M operand of the instruction and the tokens are its N operand, so a lane of
// tensor memory is an output channel and a column is a token.  One kernel then serves every row
// count: N is 16 to 256 tokens in steps of 16, few tokens cost few tensor cycles, and a warp's
// store of one token is contiguous whatever N and M are.
//
//   first warps epilogue: warp w owns tensor-memory lanes 32 (w % 4).. and the pieces of 16 columns
//               (tokens) w / 4, w / 4 + groups, ..
//   next warp   TMA producer: 128 weight rows and the tile's tokens, one to four K blocks of 128 bytes a stage
//   last warp   MMA issuer: 4 instructions (K = 32 each) for 128 bytes of K
//
// Three forms of the same kernel:
//   pair    two CTAs share a 256 x 256 tile (cta_group::2): each loads 128 weight rows and half of
//           the tokens, 32 KB a stage for what takes 48 KB in one CTA
//   single  one CTA, 128 weight rows x up to 256 tokens
//   split   few tiles: K divided among the CTAs of a cluster, the int32 partial sums added through
//           distributed shared memory (exactly, so the cut does not show in the result)
// SwiGLU: of every 32 lanes 16 are gate rows and 16 the up rows of the same channels (one
// five-dimensional box of the stacked weight puts them there), a shuffle brings g and u together and
// silu(g) * u is stored in fp32: the quantizer that follows reads 4 bytes instead of 8.
// Persistent except for split; every wait is time-limited.  A CTA whose wait runs out records it, tells the other CTA
// of its pair and leaves its loops; what it and its pair have under way (copies into the stages, MMAs) is waited for
// behind the closing barrier, so that nothing lands in shared or tensor memory that has been handed on.
//
// What bounds it.  Large products: the tensor pipe, busy nine tenths of the time (4096 x 14336 x 4096 in 153 us
// as a burst, 3.1 Pop/s; 180 us when the power limit has taken the clock to 1.5 GHz), with operands coming
// out of L2 at 12 TB/s: single CTAs, which load half as much again, take 36 us for 2048 x 4096 x 4096 where
// pairs take 31.  The two wide dimensions are 256 because tensor memory holds two accumulators of 256
// columns.  Few tokens: the weight bytes (64 tokens through 128 experts 5.2 to 5.7 TB/s).
// A few dense tiles: 2 us for adding the partial sums, which splitting saves several times over (77 x 4096 x
// 14336: 16.6 us with four CTAs a tile, 31 with one).
#include "common.cuh"
#include "host.h"
#include "int8.cuh"
#include "tcgen05.cuh"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace lsg {

using namespace tc;

namespace {

constexpr int kRows = 128;                   // weight rows of a CTA
constexpr int kKB = 128;                     // bytes of K in a stage
constexpr int kABytes = kRows * kKB;
template <bool WIDE> constexpr int kPairBlocks = WIDE ? 2 : 1;   // K blocks of a pair's stage
constexpr int kEpiGroups = 2;               // of four warps: 128 lanes of tensor memory
constexpr int kEpiWarps = 4 * kEpiGroups;
constexpr int kPieces = 16 * kEpiGroups;     // columns from one piece of a warp to its next
constexpr int kThreads = (kEpiWarps + 2) * 32;
constexpr int kMaxStages = 12;
constexpr int kTailBytes = 512 + kEpiWarps * 128 + 2 * 1025 * 4 + 64;    // barriers, flags; token scales; the experts' tiles and rows
constexpr int kSmemMax = 227 * 1024 - 1024 - kTailBytes;

struct MmaArgs {
    void* D;
    int out_dtype;
    const float* sA;
    const float* sB;
    const int32_t* offsets;   // null: dense
    int M, N, E, kblocks;     // N: output columns (of silu(g) * u for SwiGLU)
    int tn;                   // tokens of the tensor map's box (of a CTA: half of a pair's)
    int tile;                 // tokens of a tile at most
    int n_tiles, stages, sub, block_bytes, tmem_cols;   // stages of `sub` K blocks of block_bytes
    int early;   // the kernel in front is the row quantizer: weights and offsets are there before it ends
    unsigned int* status;
    long long limit;
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ uint32_t load_remote(uint32_t cluster_addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(cluster_addr) : "memory");
    return v;
}
__device__ __forceinline__ void store_remote(uint32_t cluster_addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}
// Takes bytes that no copy will bring off a barrier's count.
__device__ __forceinline__ void mbar_complete_tx(uint64_t* bar, uint32_t bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
// Release at CTA scope: what the arrival hands over are tensor-memory reads that have completed.  At cluster
// scope it would wait for the epilogue's stores to global memory (a quarter of the time of short-K tiles).
__device__ __forceinline__ void arrive_remote(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// cta_group::2: the barrier may be the other CTA's of the pair.
template <int CG>
__device__ __forceinline__ void tma_5d(void* dst, const CUtensorMap* map, int x, int y, int z, int v, int w, uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile(
            "cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
            ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(v), "r"(w), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
            ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(v), "r"(w), "r"(bar)
            : "memory");
}
template <int CG>
__device__ __forceinline__ void tma_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
    if constexpr (CG == 2)
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
            ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
            ::"r"(smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar)
            : "memory");
}
template <int CG>
__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    if constexpr (CG == 2)
        asm volatile(
            "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
            "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
}
// Completion of the MMAs so far, to this barrier (of both CTAs of a pair).
template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar) {
    if constexpr (CG == 2)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)),
            "h"(static_cast<uint16_t>(3))
            : "memory");
    else
        tc_commit(bar);
}
template <int CG>
__device__ __forceinline__ void alloc_tmem(uint32_t* slot, uint32_t cols) {
    if constexpr (CG == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
        tmem_alloc(slot, cols);
    }
}
template <int CG>
__device__ __forceinline__ void free_tmem(uint32_t addr, uint32_t cols) {
    if constexpr (CG == 2)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
    else
        tmem_dealloc(addr, cols);
}

// int8 x int8 -> int32, both operands K-major.
__device__ __forceinline__ uint32_t idesc_i8(int m, int n) {
    return (2u << 4) | (1u << 7) | (1u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[16]) {
    // the registers pass through, so that nothing reads them earlier
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

// Sixteen tokens (rows of D) of one output column to p, p + N, ...; the first `count` of them.
template <typename T>
__device__ __forceinline__ void store_column(T* p, size_t ld, const float (&v)[16], int count) {
    if (count >= 16) {
#pragma unroll
        for (int i = 0; i < 16; ++i, p += ld) *p = out_of<T>(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i, p += ld)
            if (i < count) *p = out_of<T>(v[i]);
    }
}

// The tile a CTA (or pair) works on next.
struct Tile {
    int expert, row0, rows, height, n;   // height: tokens the MMA multiplies, a multiple of `step`
};

// Tiles of an expert share its rows evenly, in multiples of `step`; the last one multiplies what is left.
__device__ __forceinline__ Tile tile_of(const MmaArgs& a, const int* cum, const int* start, int w, int step) {
    Tile t;
    int r0, rows, units, local;
    if (a.offsets) {
        int lo = 0, hi = a.E - 1;            // the last expert whose first tile is at most w
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (cum[mid] * a.n_tiles <= w) lo = mid;
            else hi = mid - 1;
        }
        t.expert = lo;
        units = cum[lo + 1] - cum[lo];
        local = w - cum[lo] * a.n_tiles;
        r0 = start[lo];
        rows = start[lo + 1] - r0;
    } else {
        t.expert = 0;
        units = (a.M + a.tile - 1) / a.tile;
        local = w;
        r0 = 0;
        rows = a.M;
    }
    t.n = local / units;
    const int u = local - t.n * units;
    const int even = (rows + units - 1) / units;
    const int apart = (even + step - 1) / step * step;
    t.row0 = r0 + u * apart;
    t.rows = min(apart, rows - u * apart);
    t.height = (t.rows + step - 1) / step * step;
    return t;
}

template <int CG, bool SWIGLU, int SPLIT, bool WIDE>
__global__ void __launch_bounds__(kThreads, 1)
int8_mma_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const MmaArgs a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const int sub = CG == 2 ? kPairBlocks<WIDE> : a.sub;
    const int stage_bytes = sub * a.block_bytes;
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + a.stages * stage_bytes);
    uint64_t* empty = full + kMaxStages;
    uint64_t* acc_full = empty + kMaxStages;   // [2]
    uint64_t* acc_empty = acc_full + 2;        // [2]
    uint64_t* drained = acc_empty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drained + 1);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* scan = reinterpret_cast<int*>(tmem_slot + 2);                           // [16]
    uint32_t* filled = tmem_slot + 18;                                           // stages filled; with weights at least
    float* scales = reinterpret_cast<float*>(smem + a.stages * stage_bytes + 512);   // [epilogue warps][2][16] of the tokens
    int* cum = reinterpret_cast<int*>(smem + a.stages * stage_bytes + 512 + kEpiWarps * 128);   // [E + 1] tiles of tokens before expert e
    int* start = cum + 1025;                                                      // [E + 1] first row

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = (CG == 2 || SPLIT > 1) ? cluster_rank() : 0;
    constexpr int kStep = CG == 2 ? 32 : 16;

    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        for (int s = 0; s < a.stages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], kEpiWarps * CG);
        }
        mbar_init(drained, 1);
        *abort_flag = 0;
        mbar_fence_init();
    }
    if (warp == kEpiWarps + 1) alloc_tmem<CG>(tmem_slot, a.tmem_cols);
    if (warp == kEpiWarps && elect_one()) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmW) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&tmX) : "memory");
    }
    if (!a.early) pdl_wait_prior();
    if (a.offsets && threadIdx.x < 256) {
        // Tiles per expert, summed; offsets are taken as a rising sequence inside [0, M].  A thread has
        // `per` consecutive experts: a running maximum over the starts, then a running sum of the tiles.
        const int per = (a.E + 255) >> 8, e0 = threadIdx.x * per;
        int lo[4], hi[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool have = j < per && e0 + j < a.E;
            lo[j] = have ? min(max(__ldg(a.offsets + e0 + j), 0), a.M) : 0;
            hi[j] = have ? min(max(__ldg(a.offsets + e0 + j + 1), 0), a.M) : 0;
        }
        int top = max(max(lo[0], lo[1]), max(lo[2], lo[3]));
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, top, o);
            if (lane >= o) top = max(top, v);
        }
        if (lane == 31) scan[warp] = top;
        int before = __shfl_up_sync(0xffffffffu, top, 1);
        if (lane == 0) before = 0;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        for (int i = 0; i < warp; ++i) before = max(before, scan[i]);
        int units = 0, n[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            lo[j] = before = max(before, lo[j]);
            hi[j] = max(hi[j], lo[j]);
            n[j] = j < per && e0 + j < a.E ? (hi[j] - lo[j] + a.tile - 1) / a.tile : 0;
            units += n[j];
        }
        int incl = units;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) scan[8 + warp] = incl;
        asm volatile("bar.sync 1, 256;" ::: "memory");
        int at = incl - units;
        for (int i = 0; i < warp; ++i) at += scan[8 + i];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j < per && e0 + j < a.E) {
                cum[e0 + j] = at;
                start[e0 + j] = lo[j];
                at += n[j];
                if (e0 + j == a.E - 1) {
                    cum[a.E] = at;
                    start[a.E] = hi[j];
                }
            }
        }
    }
    tc_fence_before();
    if constexpr (CG == 2 || SPLIT > 1) cluster_sync();
    else __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;

    const int total = (a.offsets ? cum[a.E] : (a.M + a.tile - 1) / a.tile) * a.n_tiles;
    const int first = blockIdx.x / (CG * SPLIT);
    const int stride = gridDim.x / (CG * SPLIT);
    // this CTA's K blocks
    const int kb0 = SPLIT > 1 ? static_cast<int>(a.kblocks * rank / SPLIT) : 0;
    const int kb1 = SPLIT > 1 ? static_cast<int>(a.kblocks * (rank + 1) / SPLIT) : a.kblocks;

    // before the closing barrier: behind it both CTAs of a pair find their flag set
    auto give_up = [&] {
        *abort_flag = 1;
        if constexpr (CG == 2) store_remote(map_to_rank(smem_u32(const_cast<int*>(abort_flag)), rank ^ 1), 1);
    };
    if (warp == kEpiWarps) {
        // ------------------------------ TMA producer ------------------------------
        int s = 0;
        uint32_t lap = 0;
        bool ok = true;
        const uint32_t full_at = CG == 2 ? map_to_rank(smem_u32(full), 0) : smem_u32(full);   // the leader's barriers
        // the weights of stage i, K blocks kb.., and the bytes that its barrier waits for
        auto load_weights = [&](int i, int kb, const Tile& t, int n_cta, int blocks) {
            uint8_t* dst = smem + i * stage_bytes;
            const uint32_t bar = full_at + 8 * i;
            // the leader's barrier counts the bytes of both CTAs
            if (CG == 1 || rank == 0) mbar_arrive_expect_tx(&full[i], CG * (WIDE ? sub : blocks) * (kABytes + a.tn * kKB));
            if constexpr (WIDE) {
                if constexpr (SWIGLU) tma_5d<CG>(dst, &tmW, 0, 0, 2 * t.expert, n_cta * (kRows / 32), kb, bar);
                else tma_5d<CG>(dst, &tmW, 0, n_cta * kRows, t.expert, kb, 0, bar);
            } else {
                for (int j = 0; j < blocks; ++j) {
                    if constexpr (SWIGLU)
                        tma_5d<CG>(dst + j * kABytes, &tmW, (kb + j) * kKB, 0, 0, n_cta * (kRows / 32), t.expert, bar);
                    else
                        tma_5d<CG>(dst + j * kABytes, &tmW, (kb + j) * kKB, n_cta * kRows, t.expert, 0, 0, bar);
                }
            }
        };
        int ahead = 0;   // stages whose weights are under way before the kernel in front has ended
        if (a.early) {
            if (first < total) {
                const Tile t = tile_of(a, cum, start, first, kStep);
                const int n_cta = t.n * CG + (CG == 2 ? static_cast<int>(rank) : 0);
                for (int kb = kb0; kb < kb1 && ahead < a.stages; kb += sub, ++ahead)
                    if (elect_one()) load_weights(ahead, kb, t, n_cta, min(sub, kb1 - kb));
                __syncwarp();
            }
            pdl_wait_prior();
        }
        for (int w = first; w < total && ok && !*abort_flag; w += stride) {
            const Tile t = tile_of(a, cum, start, w, kStep);
            const int x_row = t.row0 + (CG == 2 ? static_cast<int>(rank) * (t.height >> 1) : 0);
            const int n_cta = t.n * CG + (CG == 2 ? static_cast<int>(rank) : 0);
            for (int kb = kb0; kb < kb1; kb += sub) {
                if (lap > 0)
                    ok = __all_sync(0xffffffffu, mbar_wait_bounded(&empty[s], (lap - 1) & 1, a.status, kDevWaitEmpty, 2000u, a.limit));
                if (!ok) break;
                if (elect_one()) {
                    const int blocks = min(sub, kb1 - kb);
                    if (lap > 0 || s >= ahead) load_weights(s, kb, t, n_cta, blocks);
                    uint8_t* dst = smem + s * stage_bytes + sub * kABytes;
                    const uint32_t bar = full_at + 8 * s;
                    if constexpr (WIDE) {
                        tma_3d<CG>(dst, &tmX, 0, x_row, kb, bar);
                    } else {
                        for (int j = 0; j < blocks; ++j) tma_3d<CG>(dst + j * a.tn * kKB, &tmX, (kb + j) * kKB, x_row, 0, bar);
                    }
                }
                __syncwarp();
                if (++s == a.stages) {
                    s = 0;
                    ++lap;
                }
            }
        }
        if (!ok) give_up();
        if (lane == 0) {
            filled[0] = lap * a.stages + s;
            filled[1] = max(filled[0], static_cast<uint32_t>(ahead));
        }
    } else if (warp == kEpiWarps + 1) {
        // ------------------------------ MMA issuer --------------------------------
        if (a.early) pdl_wait_prior();
        int s = 0, ab = 0;
        uint32_t lap = 0, acc_lap = 0;
        bool ok = true;
        if (CG == 1 || rank == 0) {
            for (int w = first; w < total && ok && !*abort_flag; w += stride) {
                const Tile t = tile_of(a, cum, start, w, kStep);
                const uint32_t idesc = idesc_i8(CG * kRows, t.height);
                if (acc_lap > 0)
                    ok = __all_sync(0xffffffffu, mbar_wait_bounded(&acc_empty[ab], (acc_lap - 1) & 1, a.status, kDevWaitTmem, 2000u, a.limit));
                if (!ok) break;
                tc_fence_after();
                const uint32_t d = tmem_base + ab * (a.tmem_cols >> 1);
                for (int kb = kb0; kb < kb1; kb += sub) {
                    ok = __all_sync(0xffffffffu, mbar_wait_bounded(&full[s], lap & 1, a.status, kDevWaitFull, 2000u, a.limit));
                    if (!ok) break;
                    tc_fence_after();
                    const int blocks = min(sub, kb1 - kb);
                    if (elect_one()) {
                        for (int j = 0; j < blocks; ++j) {
                            const uint32_t at = smem_u32(smem + s * stage_bytes);
                            const uint64_t adesc = smem_desc_sw128(at + j * kABytes);
                            const uint64_t bdesc = smem_desc_sw128(at + sub * kABytes + j * a.tn * kKB);
#pragma unroll
                            for (int k = 0; k < kKB / 32; ++k)
                                mma_i8<CG>(d, adesc + 2 * k, bdesc + 2 * k, idesc, (kb + j > kb0 || k != 0) ? 1u : 0u);
                        }
                        commit<CG>(&empty[s]);
                        if (kb + sub >= kb1) commit<CG>(&acc_full[ab]);
                    }
                    __syncwarp();
                    if (++s == a.stages) {
                        s = 0;
                        ++lap;
                    }
                }
                ab ^= 1;
                acc_lap += ab == 0;
            }
            if (!ok) give_up();
        }
    } else {
        // ------------------------------ epilogue ---------------------------------
        if (a.early) pdl_wait_prior();
        const int q = warp & 3, group = warp >> 2;
        const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(q * 32) << 16);
        int ab = 0;
        uint32_t acc_lap = 0;
        bool ok = true;
        for (int w = first; w < total && ok && !*abort_flag; w += stride) {
            const Tile t = tile_of(a, cum, start, w, kStep);
            const int n_cta = t.n * CG + (CG == 2 ? static_cast<int>(rank) : 0);
            // output column of this lane, and where its weight scale lies
            int n, sb_at, n_scales;
            if constexpr (SWIGLU) {
                n = n_cta * (kRows / 2) + q * 16 + (lane & 15);
                sb_at = n + (lane >= 16 ? a.N : 0);
                n_scales = 2 * a.N;
            } else {
                n = n_cta * kRows + q * 32 + lane;
                sb_at = n;
                n_scales = a.N;
            }
            const bool in = n < a.N;
            const float sb = SPLIT == 1 && in ? __ldg(a.sB + static_cast<size_t>(t.expert) * n_scales + sb_at) : 0.0f;
            // the scales of a piece's 16 tokens, fetched a piece ahead and handed round through shared memory
            auto token_scale = [&](int c) { return __ldg(a.sA + min(t.row0 + c + (lane & 15), a.M - 1)); };
            float sa_next = SPLIT > 1 ? 0.0f : token_scale(group * 16);
            ok = __all_sync(0xffffffffu, mbar_wait_bounded(&acc_full[ab], acc_lap & 1, a.status, kDevWaitMma, 2000u, a.limit));
            if (!ok) break;
            tc_fence_after();
            const uint32_t src = t_lane + ab * (a.tmem_cols >> 1);
            if constexpr (SPLIT > 1) {
                // partial sums to this CTA's shared memory, [token][128 channels]; the stages are free:
                // every MMA that reads them has completed
                int* part = reinterpret_cast<int*>(smem);
                for (int c = group * 16; c < t.height; c += kPieces) {
                    uint32_t r[16];
                    tmem_ld16(src + c, r);
                    tmem_ld_wait(r);
#pragma unroll
                    for (int i = 0; i < 16; ++i) part[(c + i) * kRows + q * 32 + lane] = static_cast<int>(r[i]);
                }
            } else {
                int flip = 0;
                auto piece = [&](const uint32_t (&r)[16], int c) {
                    float* sa_buf = scales + warp * 32 + flip;
                    flip ^= 16;   // the other half for the next piece
                    if (lane < 16) sa_buf[lane] = sa_next;
                    __syncwarp();
                    sa_next = token_scale(c + kPieces);
                    float v[16];
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const float4 sa = *reinterpret_cast<const float4*>(sa_buf + i);
                        v[i] = __fmul_rn(__fmul_rn(static_cast<float>(static_cast<int>(r[i])), sa.x), sb);
                        v[i + 1] = __fmul_rn(__fmul_rn(static_cast<float>(static_cast<int>(r[i + 1])), sa.y), sb);
                        v[i + 2] = __fmul_rn(__fmul_rn(static_cast<float>(static_cast<int>(r[i + 2])), sa.z), sb);
                        v[i + 3] = __fmul_rn(__fmul_rn(static_cast<float>(static_cast<int>(r[i + 3])), sa.w), sb);
                    }
                    if constexpr (SWIGLU) {
                        float* p = static_cast<float*>(a.D) + static_cast<size_t>(t.row0 + c + (lane >> 4)) * a.N + n;
                        const int left = t.rows - c - (lane >> 4);
#pragma unroll
                        for (int i = 0; i < 16; i += 2, p += 2 * static_cast<size_t>(a.N)) {
                            // lanes 0-15 take token i, lanes 16-31 token i + 1
                            const float got = __shfl_xor_sync(0xffffffffu, lane < 16 ? v[i + 1] : v[i], 16);
                            const float g = lane < 16 ? v[i] : got, u = lane < 16 ? got : v[i + 1];
                            if (in && i < left) *p = silu_mul(g, u);
                        }
                    } else if (in) {
                        const size_t at = static_cast<size_t>(t.row0 + c) * a.N + n;
                        const int count = t.rows - c;
                        if (a.out_dtype == LSG_DTYPE_BF16) store_column(static_cast<__nv_bfloat16*>(a.D) + at, a.N, v, count);
                        else if (a.out_dtype == LSG_DTYPE_F16) store_column(static_cast<__half*>(a.D) + at, a.N, v, count);
                        else store_column(static_cast<float*>(a.D) + at, a.N, v, count);
                    }
                };
                // the accumulator is free for the next tile but one when its last piece is in registers
                auto hand_back = [&] {
                    tc_fence_before();
                    __syncwarp();
                    if (elect_one()) {
                        if (CG == 2) arrive_remote(map_to_rank(smem_u32(&acc_empty[ab]), 0));
                        else mbar_arrive(&acc_empty[ab]);
                    }
                    __syncwarp();
                };
                // two pieces in registers: one is read while the other is worked on
                uint32_t r0[16], r1[16];
                int c = group * 16;
                if (c < t.rows) {
                    tmem_ld16(src + c, r0);
                    tmem_ld_wait(r0);
                }
                if (c + kPieces >= t.rows) hand_back();
                while (c < t.rows) {
                    if (c + kPieces < t.rows) tmem_ld16(src + c + kPieces, r1);
                    piece(r0, c);
                    c += kPieces;
                    if (c >= t.rows) break;
                    tmem_ld_wait(r1);
                    if (c + kPieces < t.rows) tmem_ld16(src + c + kPieces, r0);
                    else hand_back();
                    piece(r1, c);
                    c += kPieces;
                    if (c >= t.rows) break;
                    tmem_ld_wait(r0);
                    if (c + kPieces >= t.rows) hand_back();
                }
                __syncwarp();
                ab ^= 1;
                acc_lap += ab == 0;
            }
        }
        if (!ok) give_up();
    }

    // Behind the closing barrier of a CTA (pair) that gave up: the issuer waits for its MMAs, the producer for every
    // stage's last copies.  The leader's barriers count both CTAs' bytes, and one of the two may have gone a stage
    // further: the leader arms what it has not yet, and takes off what was never asked for.
    auto drain = [&] {
        const bool leads = CG == 1 || rank == 0;
        if (warp == kEpiWarps + 1) {
            if (leads && elect_one()) commit<CG>(drained);
            __syncwarp();
            mbar_wait_bounded(drained, 0, a.status, kDevWaitMma);
        } else if (leads && warp == kEpiWarps && lane == 0) {
            const uint32_t f0 = filled[0], w0 = filled[1];
            uint32_t f1 = f0, w1 = w0;
            if constexpr (CG == 2) {
                const uint32_t theirs = map_to_rank(smem_u32(filled), 1);
                f1 = load_remote(theirs);
                w1 = load_remote(theirs + 4);
            }
            const uint32_t stages = a.stages, end = max(w0, w1), per_tile = (kb1 - kb0 + sub - 1) / sub;
            for (uint32_t f = end > stages ? end - stages : 0; f < end; ++f) {
                uint64_t* bar = &full[f % stages];
                const uint32_t blocks = WIDE ? sub : min(sub, kb1 - kb0 - static_cast<int>(f % per_tile) * sub);
                const uint32_t weights = blocks * kABytes, tokens = blocks * a.tn * kKB;
                uint32_t never = (f >= w0 ? weights : 0) + (f >= f0 ? tokens : 0);
                if (CG == 2) never += (f >= w1 ? weights : 0) + (f >= f1 ? tokens : 0);
                if (f >= w0) mbar_arrive_expect_tx(bar, CG * (weights + tokens));
                if (never > 0) mbar_complete_tx(bar, never);
                mbar_wait_bounded(bar, (f / stages) & 1, a.status, kDevWaitFull);
            }
        }
        __syncwarp();
    };

    tc_fence_before();
    __syncwarp();
    if constexpr (SPLIT > 1) {
        // Every rank adds and writes its share of the tokens: a warp U tokens at a time, four channels a
        // lane, all loads of the partial sums under way together.
        constexpr int U = SPLIT == 8 ? 1 : (SPLIT == 4 ? 2 : 4);
        constexpr int kApart = SPLIT * (kThreads / 32);
        const Tile t = tile_of(a, cum, start, first, kStep);
        const int n = t.n * kRows + lane * 4;
        float sb[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) sb[i] = n + i < a.N ? __ldg(a.sB + n + i) : 0.0f;
        const size_t size = a.out_dtype == LSG_DTYPE_F32 ? 4 : 2;
        const bool whole = n + 3 < a.N && (a.N & 3) == 0 && (reinterpret_cast<uintptr_t>(a.D) & (4 * size - 1)) == 0;
        cluster_sync();
        if (*abort_flag) drain();
        for (int c0 = static_cast<int>(rank) + SPLIT * warp; c0 < t.rows; c0 += U * kApart) {
            float4 p[U][SPLIT];
            float sa[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = min(c0 + u * kApart, t.rows - 1);
                sa[u] = __ldg(a.sA + t.row0 + c);
                const uint32_t at = smem_u32(smem) + static_cast<uint32_t>((c * kRows + lane * 4) * 4);
#pragma unroll
                for (int r = 0; r < SPLIT; ++r) p[u][r] = ld_cluster_f4(at, r);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int c = c0 + u * kApart;
                if (c >= t.rows) break;
                int v[4] = {0, 0, 0, 0};
#pragma unroll
                for (int r = 0; r < SPLIT; ++r) {
                    v[0] += __float_as_int(p[u][r].x);
                    v[1] += __float_as_int(p[u][r].y);
                    v[2] += __float_as_int(p[u][r].z);
                    v[3] += __float_as_int(p[u][r].w);
                }
                float o[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) o[i] = __fmul_rn(__fmul_rn(static_cast<float>(v[i]), sa[u]), sb[i]);
                const size_t at = static_cast<size_t>(t.row0 + c) * a.N + n;
                if (whole) {
                    store_out4(a.D, a.out_dtype, at, o);
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (n + i < a.N) store_out(a.D, a.out_dtype, at + i, o[i]);
                }
            }
        }
        __syncwarp();
        cluster_sync();      // nobody leaves while its sums are read
    } else if constexpr (CG == 2) {
        cluster_sync();
        if (*abort_flag) {
            drain();
            cluster_sync();      // the leader has waited for the other CTA's copies
        }
    } else {
        __syncthreads();
        if (*abort_flag) drain();
    }
    if (warp == kEpiWarps + 1) {
        tc_fence_after();
        free_tmem<CG>(tmem_base, a.tmem_cols);
    }
}

int encode(CUtensorMap* map, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return fail(LSG_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const cuuint32_t one[5] = {1, 1, 1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides, box, one,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(LSG_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", static_cast<int>(r));
    return LSG_OK;
}

// The weight [E, N, K] (or [E, 2 N, K], gate rows in front of up rows): boxes of 128 rows by 128 bytes, or by
// `blocks` times 128 bytes, block after block (0: K is not a multiple of 128, and reads as zeros behind it).
int weight_map(CUtensorMap* map, const Int8Gemm& g, bool swiglu, int blocks) {
    const cuuint64_t ld = static_cast<cuuint64_t>(g.ldb), n = static_cast<cuuint64_t>(g.N), e = static_cast<cuuint64_t>(g.E);
    const cuuint64_t k = static_cast<cuuint64_t>(g.K), kb = k / kKB;
    if (swiglu && blocks) {
        const cuuint64_t dims[5] = {kKB, 16, 2 * e, n / 16, kb};
        const cuuint64_t strides[4] = {ld, ld * n, ld * 16, kKB};
        const cuuint32_t box[5] = {kKB, 16, 2, 4, static_cast<cuuint32_t>(blocks)};
        return encode(map, 5, g.B, dims, strides, box);
    }
    if (swiglu) {
        const cuuint64_t dims[5] = {k, 16, 2, n / 16, e};
        const cuuint64_t strides[4] = {ld, ld * n, ld * 16, ld * n * 2};
        const cuuint32_t box[5] = {kKB, 16, 2, 4, 1};
        return encode(map, 5, g.B, dims, strides, box);
    }
    if (blocks) {
        const cuuint64_t dims[5] = {kKB, n, e, kb, 1};
        const cuuint64_t strides[4] = {ld, ld * n, kKB, ld * n};
        const cuuint32_t box[5] = {kKB, kRows, 1, static_cast<cuuint32_t>(blocks), 1};
        return encode(map, 5, g.B, dims, strides, box);
    }
    const cuuint64_t dims[5] = {k, n, e, 1, 1};
    const cuuint64_t strides[4] = {ld, ld * n, ld * n, ld * n};
    const cuuint32_t box[5] = {kKB, kRows, 1, 1, 1};
    return encode(map, 5, g.B, dims, strides, box);
}

// The tokens [M, K]: boxes of `rows` by 128 bytes, or as above.
int token_map(CUtensorMap* map, const Int8Gemm& g, int rows, int blocks) {
    const cuuint64_t ld = static_cast<cuuint64_t>(g.lda), m = static_cast<cuuint64_t>(g.M), k = static_cast<cuuint64_t>(g.K);
    const cuuint64_t dims[3] = {blocks ? kKB : k, m, blocks ? k / kKB : 1};
    const cuuint64_t strides[2] = {ld, blocks ? kKB : ld * m};
    const cuuint32_t box[3] = {kKB, static_cast<cuuint32_t>(rows), static_cast<cuuint32_t>(blocks ? blocks : 1)};
    return encode(map, 3, g.A, dims, strides, box);
}

template <int CG, bool SWIGLU, int SPLIT, bool WIDE>
int launch(const CUtensorMap& tmW, const CUtensorMap& tmX, const MmaArgs& a, int grid, int cluster, cudaStream_t s) {
    static std::atomic<bool> configured[64];
    int dev = 0;
    LSG_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_relaxed)) {
        LSG_CUDA_TRY(cudaFuncSetAttribute(int8_mma_kernel<CG, SWIGLU, SPLIT, WIDE>, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_relaxed);
    }
    const size_t smem = static_cast<size_t>(a.stages) * a.sub * a.block_bytes + 1024 + kTailBytes;
    LSG_CUDA_TRY(launch_clusters(int8_mma_kernel<CG, SWIGLU, SPLIT, WIDE>, cluster, dim3(static_cast<unsigned>(grid)), dim3(kThreads), smem, s,
                                 true, tmW, tmX, a));
    return LSG_OK;
}

// Clusters of CTAs that take an SM each (all forms do) that the device holds at a time.
template <int CTAS>
int resident(ClusterSlots& seen) {
    return cluster_slots(int8_mma_kernel<1, false, CTAS, true>, CTAS, kThreads, 227 * 1024, seen);
}

int round_up(int v, int step) { return (v + step - 1) / step * step; }

struct Plan {
    int tile;       // tokens of a tile
    bool pair;
    int split;
};

// One product: the tile, the form and the cut of K of the least estimated time, in SM cycles.  A K block of a
// tile takes what the tensor pipe needs (2 cycles a token, nine tenths of the time) or what its operands need to
// arrive, whichever is longer: 68 bytes a cycle out of L2 in single CTAs, 58 in pairs, weight rows that only this
// tile of tokens reads 48, as they come from memory.  All weights take the memory's 3300 bytes a cycle once.
// Behind the last K block come the epilogue (13 cycles a token) and, where K is cut, adding the partial sums
// (2200 and 37 a token); what does not fit the stages at once waits for memory once more (1000).
// Against one rule per row count (even tiles of up to 256 tokens, cut when fewer than half the SMs have one):
// 1001 x 1024 x 4096 12.9 -> 9.7 us, 512 x 4096 x 4096 15.2 -> 11.5, 600 x 2000 x 1024 9.0 -> 5.5, 1500 x 4096 x
// 4096 25.6 -> 22.3.
// slots: clusters of 1, 2, 4, 8 CTAs that are resident at a time.
Plan plan_dense(int M, int N, int kblocks, const int (&slots)[4]) {
    const int sms = slots[0];
    const long long ctas = (N + kRows - 1) / kRows;
    const long long bytes = static_cast<long long>(N) * kblocks * kKB;
    Plan best = {256, false, 1};
    long long least = -1;
    const auto consider = [&](int tile, bool pair, int split, long long units, long long active, long long rounds) {
        const int from = units == 1 ? 48 : (pair ? 58 : (units == 2 ? 58 : 68));
        const long long kbs = (kblocks + split - 1) / split;
        const long long mma = tile * 2 * 10 / 9, load = kABytes / from + (pair ? tile * 64 / 58 : tile * 128 / 68);
        const long long stream = bytes / std::min(3300ll, 48 * std::min(active, static_cast<long long>(sms)));
        const long long laps = rounds * kbs * (kABytes + (pair ? tile * 64 : tile * 128)) / (216 * 1024);
        const long long t = std::max(rounds * kbs * std::max(mma, load), stream) + tile * 13 +
                            (split > 1 ? 2200 + tile * 37 : 0) + (laps > 0 ? 1000 : 0);
        if (least < 0 || t < least) {
            least = t;
            best = {tile, pair, split};
        }
    };
    int last = 0;
    for (long long units = (static_cast<long long>(M) + 255) / 256, tries = 0; tries < 32; ++tries, ++units) {
        const int tile = round_up(static_cast<int>((M + units - 1) / units), 16);
        if (tile == last) continue;
        last = tile;
        const long long n = (M + tile - 1) / tile;
        consider(tile, false, 1, n, n * ctas, (n * ctas + sms - 1) / sms);
        for (int c = 1; c < 4; ++c)
            if (n * ctas <= slots[c] && kblocks >= (2 << c)) consider(tile, false, 1 << c, n, n * ctas << c, 1);
        const int even = round_up(tile, 32);
        const long long m = (M + even - 1) / even, pairs = m * ((ctas + 1) / 2);
        if (tile >= 32 && slots[1] > 0) consider(even, true, 1, m, 2 * pairs, (pairs + slots[1] - 1) / slots[1]);
        if (tile <= 32) break;
    }
    return best;
}

}  // namespace

// D = A B^T with both scales; swiglu: B is [E, 2 N, K] and D fp32 silu(gate) * up.  early: A comes from
// the row quantizer launched right in front.  That kernel lets this one start only after its own wait,
// so everything launched before it has ended: offsets are read and weights loaded while it still runs.
int int8_mma(const Int8Gemm& g, bool swiglu, bool early, cudaStream_t s) {
    if (g.M > 0x7fffffff - 512 || g.N > 0x7fffffff - 512) return fail(LSG_ERR_UNSUPPORTED, "int8 product: too many rows");
    // K a multiple of 128: one copy loads all K blocks of a stage (experts of 4096 tokens 1319 -> 1295 us)
    const bool wide = g.K % kKB == 0;
    MmaArgs a = {};
    a.D = g.D; a.out_dtype = g.out_dtype; a.sA = g.scale_A; a.sB = g.scale_B; a.offsets = g.expert_offsets;
    a.M = g.M; a.N = g.N; a.E = g.E; a.kblocks = (g.K + kKB - 1) / kKB;
    a.early = early ? 1 : 0;
    a.status = device_status_word();
    a.limit = wait_limit_cycles();
    static ClusterSlots seen;
    const int slots[4] = {sm_count(), resident<2>(seen), resident<4>(seen), resident<8>(seen)};
    const int sms = slots[0];
    const int per_cta = swiglu ? kRows / 2 : kRows;             // output columns of a CTA
    const int cta_tiles = (g.N + per_cta - 1) / per_cta;
    Plan plan;
    if (g.expert_offsets) {
        // 1.4 times the average rows of an expert, so that most experts are one tile: 1024 tokens, 128 experts of
        // 2048 / 768, top 8 (64 rows each): 148.7 us with 96, 154 with 128; 2048 tokens 188 with 160, 194 with 256.
        // Pairs from 96 tokens on (256 tokens, 8 experts of 4096 / 14336: 266.7 us with pairs, 274 without).
        const long long share = (static_cast<long long>(g.M) + g.E - 1) / g.E, most = share + share * 2 / 5;
        plan.tile = most >= 256 ? 256 : (most > 64 ? round_up(static_cast<int>(most), 32) : round_up(static_cast<int>(most), 16));
        plan.split = 1;
        plan.pair = slots[1] > 0 && plan.tile > 64 && (g.M / plan.tile + static_cast<long long>(std::min(g.E, g.M))) * cta_tiles >= sms / 2;
    } else {
        plan = plan_dense(g.M, g.N, a.kblocks, slots);
    }
    const int tile = plan.tile, split = plan.split;
    const bool pair = plan.pair;
    const long long units = g.expert_offsets ? g.M / tile + static_cast<long long>(std::min(g.E, g.M))
                                             : (static_cast<long long>(g.M) + tile - 1) / tile;
    a.tile = tile;
    a.tn = pair ? tile / 2 : tile;
    a.n_tiles = pair ? (cta_tiles + 1) / 2 : cta_tiles;
    a.block_bytes = kABytes + round_up(a.tn * kKB, 1024);
    // Up to 128 tokens: two to four K blocks a stage, so that what is asked of a weight row at a time is 256
    // to 512 bytes (256 tokens, 8 experts of 4096 / 14336: 278 us with stages of 56 KB, 261 with 74 KB, 272
    // with 110 KB; 128 x 14336 x 4096 20.6 with one block, then 18.3, 16.2, 18.2).
    a.sub = pair ? (wide ? kPairBlocks<true> : kPairBlocks<false>) : std::min(4, std::max(1, 74 * 1024 / a.block_bytes));
    a.stages = kSmemMax / (a.sub * a.block_bytes) < kMaxStages ? kSmemMax / (a.sub * a.block_bytes) : kMaxStages;
    int cols = 64;
    while (cols < 2 * tile) cols *= 2;
    a.tmem_cols = cols;
    const long long tiles = units * a.n_tiles;
    if (tiles > 0x7fffffffll) return fail(LSG_ERR_UNSUPPORTED, "int8 product: too many tiles");

    CUtensorMap tmW, tmX;
    int rc = weight_map(&tmW, g, swiglu, wide ? a.sub : 0);
    if (rc != LSG_OK) return rc;
    rc = token_map(&tmX, g, a.tn, wide ? a.sub : 0);
    if (rc != LSG_OK) return rc;

    const int count = static_cast<int>(tiles);
    const auto go = [&](auto w) {
        constexpr bool W = decltype(w)::value;
        if (pair) {
            const int grid = 2 * std::min(count, slots[1]);
            return swiglu ? launch<2, true, 1, W>(tmW, tmX, a, grid, 2, s) : launch<2, false, 1, W>(tmW, tmX, a, grid, 2, s);
        }
        if (split == 8) return launch<1, false, 8, W>(tmW, tmX, a, count * 8, 8, s);
        if (split == 4) return launch<1, false, 4, W>(tmW, tmX, a, count * 4, 4, s);
        if (split == 2) return launch<1, false, 2, W>(tmW, tmX, a, count * 2, 2, s);
        const int grid = std::min(count, sms);
        return swiglu ? launch<1, true, 1, W>(tmW, tmX, a, grid, 1, s) : launch<1, false, 1, W>(tmW, tmX, a, grid, 1, s);
    };
    return wide ? go(std::true_type{}) : go(std::false_type{});
}

}  // namespace lsg
