// gemm16_tc.cu -- the 16-bit products on the tensor cores (tcgen05.mma
// kind::f16, f32 accumulators in tensor memory).
//
// The weights are the MMA's M side and the tokens its N side: an expert's
// weights stream through 128-row tiles whatever its number of tokens, and the
// number of columns follows the tokens in steps of 16, so a short list
// of tokens costs no padded rows of 128. A tensor-memory lane is an output
// feature and its columns are tokens: the bias is one register, and a warp's
// store of one column is 32 consecutive features of one row.
//
//   k_gemm16_pair   256 weight rows x up to 256 tokens per pair of SMs
//                   (cta_group::2), persistent, for work bound by the MMA
//                   (8192 x 4096 x 11008, gelu: 480 us = 1540 TFLOP/s at full
//                   clocks, 555 us = 1330 where the power limit holds them)
//   k_gemm16_split  128 weight rows x up to 128 tokens per SM, k split over a
//                   cluster, for work bound by the weights' stream
//                   (64 x 4096 x 11008: 92 MB in 21.5 us = 4.3 TB/s)
//
// Gated layers: each 32-lane quarter holds 16 gate rows and the 16 up rows of
// the same features (one TMA box over the two halves of W), so the two meet
// by one exchange between lanes l and l + 16.
//
// Every wait is bounded; a wait that runs out raises the CTA's abort and the
// context's timeout word, the roles leave, copies and MMAs in flight are
// drained (bounded), tensor memory is freed and the kernel returns.

#include "gemm16.cuh"
#include "pair_settle.h"

namespace tpt {
namespace {
using namespace tc;

constexpr int BK = 64;           // k values per stage: one 128-byte swizzled row
constexpr int ROW_BYTES = 128;
constexpr int W_ROWS = 128;      // weight rows of one CTA's tile
constexpr int W_BYTES = W_ROWS * ROW_BYTES;

struct Args {
    int rows, n, k;
    int ftiles;                  // feature tiles
    int tile_n;                  // dense: tokens per tile
    int group;                   // dense: token tiles that share a sweep over the features
    uint32_t fmt;                // 0 f16, 1 bf16
    int gate16;                  // gated: n is a multiple of 16 (see weight_map)
    const int *row_token;
    const Tile16 *tiles;
    const int *n_tiles;
    const void *bias;
    int act;
    const void *residual;
    size_t ldr;
    void *y;
    size_t ldy;
    size_t low;                  // y's second plane (elements on) takes what y's rounding left; 0: none
    int x_low;                   // X's second plane (rows on), added to the first in the products
    unsigned *gflags;
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *tm, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
        "[%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *tm, uint32_t bar, int x, int y, int z,
                                            int u) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, "
        "%6}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(u)
        : "memory");
}
// four rows of a 2-D map (box one row high)
__device__ __forceinline__ void tma_gather4(uint32_t dst, const CUtensorMap *tm, uint32_t bar, int x, const int (&r)[4]) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
        "%4, %5, %6, %7}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(x), "r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3])
        : "memory");
}
// The same loads of an SM pair: the bytes count on the barrier at `bar`, the
// leader CTA's (a shared::cluster address).
__device__ __forceinline__ void tma_load_2d_p(uint32_t dst, const CUtensorMap *tm, uint32_t bar, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, "
        "{%3, %4}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(x), "r"(y)
        : "memory");
}
__device__ __forceinline__ void tma_load_3d_p(uint32_t dst, const CUtensorMap *tm, uint32_t bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, "
        "{%3, %4, %5}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void tma_load_4d_p(uint32_t dst, const CUtensorMap *tm, uint32_t bar, int x, int y, int z,
                                              int u) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, "
        "{%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(x), "r"(y), "r"(z),
        "r"(u)
        : "memory");
}
__device__ __forceinline__ void tma_load_5d_p(uint32_t dst, const CUtensorMap *tm, uint32_t bar, int x, int y, int z,
                                              int u, int v) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, "
        "{%3, %4, %5, %6, %7}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(x), "r"(y),
        "r"(z), "r"(u), "r"(v)
        : "memory");
}
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap *tm, uint32_t bar, int x, int y, int z,
                                            int u, int v) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, "
        "%6, %7}], [%2];" ::"r"(dst), "l"(reinterpret_cast<uint64_t>(tm)), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(u),
        "r"(v)
        : "memory");
}

// The producer and the MMA issuer run as whole warps with uniform control flow
// and elect one lane for the issue itself: descriptors, addresses and
// coordinates then stay in uniform registers. (One diverged lane doing it all
// moved each of them over again: 75 cycles an MMA, 600 a stage, twice the
// tensor cores' own time.)
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(r));
    return r != 0;
}
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag, unsigned *gflags,
                                          bool honour_abort) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, gflags, honour_abort));
}

template <int GROUP>
__device__ __forceinline__ void mma_f16(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                                        uint32_t accumulate) {
    if constexpr (GROUP == 2)
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
            " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
            " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d_tmem),
            "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
            : "memory");
}
// counts `bytes` on this CTA's barrier as a copy of that size would
__device__ __forceinline__ void mbar_complete_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t cluster_addr, int v) {
    asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(cluster_addr), "r"(v) : "memory");
}
__device__ __forceinline__ int ld_cluster(uint32_t cluster_addr) {
    int v;
    asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(cluster_addr) : "memory");
    return v;
}
// f32 accumulator, both operands K-major of type fmt, M x N
__device__ __forceinline__ uint32_t idesc_f16(uint32_t fmt, uint32_t m, uint32_t n) {
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
__device__ __forceinline__ void commit_both(uint32_t bar) {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
        "h"((uint16_t)3)
        : "memory");
}

// The residual's values of C columns (tokens col0 .. col0 + C - 1 of the tile)
// of this thread's feature f. A chunk whose columns are all rows takes the
// branch-free path, here and below, so that its loads and stores go out back to
// back.
template <typename TY, int C>
__device__ __forceinline__ void load_residual(const Args &a, TY (&rv)[C], int f, size_t row0, int col0, int rows) {
    const int n = f < a.n ? rows - col0 : 0;
    const TY *r = static_cast<const TY *>(a.residual) + (row0 + col0) * a.ldr + f;
    if (n >= C) {
#pragma unroll
        for (int i = 0; i < C; i++, r += a.ldr) rv[i] = *r;
    } else {
#pragma unroll
        for (int i = 0; i < C; i++, r += a.ldr) rv[i] = i < n ? *r : from_f32<TY>(0.0f);
    }
}

// One output, and with `low` what its rounding left, for a product that reads both
// (a template argument too: the test alone makes the pair kernel's epilogue a
// quarter longer)
template <bool LOW, typename TY>
__device__ __forceinline__ void store16(TY *y, float v, size_t low) {
    const TY upper = from_f32<TY>(v);
    *y = upper;
    if (LOW && low) {
        const float rest = v - to_f32(upper);
        y[low] = from_f32<TY>(isfinite(rest) ? rest : 0.0f);  // inf - inf stays out
    }
}

// The epilogue of C columns of this thread's lane. Ungated: lane l of the warp
// is feature f0 + l, b its bias, rv its residual values.
template <bool LOW, typename TY, int C>
__device__ __forceinline__ void epilogue16(const Args &a, float (&v)[C], const TY (&rv)[C], float b, int f, size_t row0,
                                           int col0, int rows) {
    const int n = f < a.n ? rows - col0 : 0;
#pragma unroll
    for (int i = 0; i < C; i++) v[i] += b;
    act16<!std::is_same<TY, float>::value>(v, a.act);
    if (a.residual) {
#pragma unroll
        for (int i = 0; i < C; i++) v[i] += to_f32(rv[i]);
    }
    TY *y = static_cast<TY *>(a.y) + (row0 + col0) * a.ldy + f;
    if (n >= C) {
#pragma unroll
        for (int i = 0; i < C; i++, y += a.ldy) store16<LOW>(y, v[i], a.low);
    } else {
#pragma unroll
        for (int i = 0; i < C; i++, y += a.ldy)
            if (i < n) store16<LOW>(y, v[i], a.low);
    }
}
// Gated: lanes l and l + 16 are the gate and the up product of feature f0 + l;
// each of them finishes half of the columns.
template <bool LOW, typename TY, int C>
__device__ __forceinline__ void epilogue16_gated(const Args &a, const float (&v)[C], int f0, size_t row0, int col0,
                                                 int rows, int lane) {
    const bool hi = lane >= 16;
    const int f = f0 + (lane & 15);
    float g[C / 2], u[C / 2];
#pragma unroll
    for (int i = 0; i < C / 2; i++) {
        const float got = __shfl_xor_sync(0xffffffffu, hi ? v[i] : v[C / 2 + i], 16);
        g[i] = hi ? got : v[i];
        u[i] = hi ? v[C / 2 + i] : got;
    }
    act16<true>(g, a.act);
    const int c0 = col0 + (hi ? C / 2 : 0);
    TY *y = static_cast<TY *>(a.y) + (row0 + c0) * a.ldy + f;
    const int n = f < a.n ? rows - c0 : 0;
    if (n >= C / 2) {
#pragma unroll
        for (int i = 0; i < C / 2; i++, y += a.ldy) store16<LOW>(y, g[i] * u[i], a.low);
    } else {
#pragma unroll
        for (int i = 0; i < C / 2; i++, y += a.ldy)
            if (i < n) store16<LOW>(y, g[i] * u[i], a.low);
    }
}
// the bias of feature f (0: none)
template <typename T>
__device__ __forceinline__ float bias_at(const Args &a, int f) {
    return a.bias && f < a.n ? to_f32(static_cast<const T *>(a.bias)[f]) : 0.0f;
}

// ---------------------------------------------------------------------------
// The SM-pair kernel. Barriers as in the pair's INT8 kernel:
//   full[s]   (leader)  both CTAs' bytes of stage s
//   empty[s]  (each)    the leader's MMAs have read stage s
//   tfull[b]  (each)    accumulator b is complete
//   tempty[b] (leader)  both CTAs' epilogue warps have read accumulator b
// ---------------------------------------------------------------------------
constexpr int P_STAGES = 6;
constexpr int P_STAGE_BYTES = 2 * W_BYTES;  // 128 weight rows + up to 128 token rows
constexpr int P_EPI_WARPS = 8;
constexpr int P_THREADS = (2 + P_EPI_WARPS) * 32;
constexpr int P_SMEM = P_STAGES * P_STAGE_BYTES + (2 * P_STAGES + 5) * 8 + 1024;

// X's maps with boxes of 128, 64 and 32 rows: a stage's token rows are one box,
// the smallest that holds them. (Rows past the tile land in columns that nothing
// reads; a box costs the issuing thread more than its extra rows cost the L2.)
struct XMaps {
    CUtensorMap box[3];
};
struct TileAt {
    int expert, row0, rows, cols, ft;
};
// Tile t of the product: sweeps of several token tiles over all the features, so
// that the tiles in flight share both operands in L2. Dense: `group` token tiles
// a sweep; grouped: the schedule's runs of tiles of one expert (a run's tiles and
// its feature tiles take the same place in the order of t as tile by tile).
__device__ __forceinline__ TileAt tile_at(const Args &a, int t) {
    TileAt r;
    if (a.tiles) {
        const int4 *tiles = reinterpret_cast<const int4 *>(a.tiles);
        const int i = t / a.ftiles;
        const int run = __ldcg(tiles + i).w, place = run >> 8, wide = run & 255;
        const int in = t - (i - place) * a.ftiles;
        r.ft = in / wide;
        const int4 q = __ldcg(tiles + (i - place) + in - r.ft * wide);
        r.expert = q.x;
        r.row0 = q.y;
        r.rows = q.z;
        r.cols = (q.z + TILE_STEP - 1) & ~(TILE_STEP - 1);
    } else {
        const int ttiles = (a.rows + a.tile_n - 1) / a.tile_n;
        const int sweep = a.group * a.ftiles;
        const int s = t / sweep, in = t - s * sweep;
        const int wide = min(a.group, ttiles - s * a.group);
        r.ft = in / wide;
        const int tt = s * a.group + in - r.ft * wide;
        r.expert = 0;
        r.row0 = tt * a.tile_n;
        r.rows = min(a.tile_n, a.rows - r.row0);
        r.cols = a.tile_n;
    }
    return r;
}

// X's box of a tile of cols tokens, half of them a CTA's, and the bytes of one CTA's stage
__device__ __forceinline__ int pair_box(int cols) { return cols > 128 ? 0 : cols > 64 ? 1 : 2; }
__device__ __forceinline__ uint32_t pair_cta_bytes(int cols) { return W_BYTES + (W_BYTES >> pair_box(cols)); }

// An aborting pair leaves no copy in flight behind it. Its two producers (the leader's
// issued `mine` stages, the other `theirs`) may have stopped at different ones; the
// leader evens out the counts of its full barriers (pair_settle.h) and waits, bounded,
// for the copies of both. Out of line: the kernels' usual end stays short.
__device__ __noinline__ void pair_drain(const Args &a, uint32_t full_bars, int mine, int theirs, int cluster,
                                        int nclusters, volatile int *abort_p) {
    const int last = max(mine, theirs), kblocks = (a.k + BK - 1) / BK;
    for (int i = max(0, last - P_STAGES); i < last; i++) {
        const uint32_t bar = full_bars + 8u * (i % P_STAGES);
        const PairSettle p =
            pair_settle(i, mine, theirs, pair_cta_bytes(tile_at(a, cluster + i / kblocks * nclusters).cols));
        if (elect_one()) {
            if (p.arrive) mbar_arrive_expect_tx(bar, p.expect);
            if (p.complete) mbar_complete_tx(bar, p.complete);
        }
        __syncwarp();
        warp_wait(bar, (uint32_t)(i / P_STAGES) & 1u, abort_p, a.gflags, false);
    }
}

template <typename T, typename TY, bool GATED>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(P_THREADS, 1)
    k_gemm16_pair(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ XMaps tmX,
                  const __grid_constant__ Args a) {
    constexpr int S = P_STAGES;
    extern __shared__ uint8_t smem_raw[];
    __shared__ int abort_flag;
    __shared__ int pair_abort, pair_issued;  // a CTA of the pair gave up; stages that this CTA's producer issued
    __shared__ uint32_t tmem_slot;
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bars = ring + S * P_STAGE_BYTES;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (S + s); };
    auto tfull_bar = [&](int b) { return bars + 8u * (2 * S + b); };
    auto tempty_bar = [&](int b) { return bars + 8u * (2 * S + 2 + b); };
    const uint32_t drain_bar = bars + 8u * (2 * S + 4);

    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const bool leader = rank == 0;
    const int cluster = blockIdx.x >> 1, nclusters = gridDim.x >> 1;
    const int kblocks = (a.k + BK - 1) / BK;

    if (threadIdx.x == 0) {
        abort_flag = pair_abort = 0;
        for (int s = 0; s < S; s++) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(tfull_bar(b), 1);
            mbar_init(tempty_bar(b), 2 * P_EPI_WARPS);
        }
        mbar_init(drain_bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmW)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmX.box[0])) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    pdl_wait();
    pdl_trigger();
    const uint32_t tmem = tmem_slot;
    volatile int *abort_p = &abort_flag;
    const int ntiles = a.tiles ? __ldcg(a.n_tiles) * a.ftiles : ((a.rows + a.tile_n - 1) / a.tile_n) * a.ftiles;

    if (warp == 0) {
        // ---------------- producer ----------------
        const uint32_t full_leader = map_to_rank(full_bar(0), 0);
        int stage = 0;
        uint32_t phase = 0;
        int issued = 0;
        bool ok = true;
        for (int t = cluster; t < ntiles && ok; t += nclusters) {
            const TileAt tl = tile_at(a, t);
            const int half = tl.cols >> 1;
            const int box = pair_box(tl.cols);
            const uint32_t bytes = 2u * pair_cta_bytes(tl.cols);
            const int xrow = tl.row0 + (int)rank * half;
            const CUtensorMap *xmap = &tmX.box[box];
            for (int kb = 0; kb < kblocks; kb++) {
                if (!warp_wait(empty_bar(stage), phase ^ 1u, abort_p, a.gflags, true)) {
                    ok = false;
                    break;
                }
                const uint32_t w_dst = ring + stage * P_STAGE_BYTES, x_dst = w_dst + W_BYTES;
                const uint32_t fb = full_leader + 8u * stage;
                if (elect_one()) {
                    if (leader) mbar_arrive_expect_tx(full_bar(stage), bytes);
                    if (GATED && a.gate16) {
                        tma_load_5d_p(w_dst, &tmW, fb, kb * BK, 0, 0, tl.ft * 8 + (int)rank * 4, tl.expert);
                    } else if (GATED) {
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            tma_load_4d_p(w_dst + q * 4096, &tmW, fb, kb * BK, tl.ft * 128 + (int)rank * 64 + q * 16,
                                          0, tl.expert);
                    } else {
                        tma_load_3d_p(w_dst, &tmW, fb, kb * BK, tl.ft * 256 + (int)rank * 128, tl.expert);
                    }
                    tma_load_2d_p(x_dst, xmap, fb, kb * BK, xrow);
                }
                __syncwarp();
                issued++;
                if (++stage == S) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
        if (lane == 0) pair_issued = issued;
    } else if (warp == 1) {
        if (leader) {
            // ---------------- MMA issuer ----------------
            int stage = 0;
            uint32_t phase = 0;
            int acc = 0;
            uint32_t acc_phase = 0;
            bool ok = true;
            for (int t = cluster; t < ntiles && ok; t += nclusters) {
                const uint32_t idesc = idesc_f16(a.fmt, 256, tile_at(a, t).cols);
                if (!warp_wait(tempty_bar(acc), acc_phase ^ 1u, abort_p, a.gflags, true)) break;
                tc_fence_after();
                const uint32_t d_tmem = tmem + (uint32_t)(acc * 256);
                for (int kb = 0; kb < kblocks; kb++) {
                    if (!warp_wait(full_bar(stage), phase, abort_p, a.gflags, true)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t w_addr = ring + stage * P_STAGE_BYTES, x_addr = w_addr + W_BYTES;
                    const uint64_t wd = sw128_desc(w_addr), xd = sw128_desc(x_addr);
                    if (elect_one()) {
#pragma unroll
                        for (int kk = 0; kk < BK / 16; kk++)
                            mma_f16<2>(d_tmem, wd + 2 * kk, xd + 2 * kk, idesc, (kb | kk) != 0 ? 1u : 0u);
                        commit_both(empty_bar(stage));
                    }
                    __syncwarp();
                    if (++stage == S) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (!ok) break;
                if (elect_one()) commit_both(tfull_bar(acc));
                __syncwarp();
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
            // drain: every MMA issued completes before tensor memory is freed
            if (elect_one())
                asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                                 drain_bar)
                             : "memory");
            __syncwarp();
            warp_wait(drain_bar, 0, abort_p, a.gflags, false);
        }
    } else {
        // ---------------- epilogue: two warps per lane quarter, alternate 32-column chunks ----------------
        const int q = warp & 3, half = (warp - 2) >> 2;
        const uint32_t tempty_leader0 = map_to_rank(tempty_bar(0), 0);
        const uint32_t tempty_leader1 = map_to_rank(tempty_bar(1), 0);
        int acc = 0;
        uint32_t acc_phase = 0;
        for (int t = cluster; t < ntiles; t += nclusters) {
            const TileAt tl = tile_at(a, t);
            const int f0 = GATED ? tl.ft * 128 + (int)rank * 64 + q * 16 : tl.ft * 256 + (int)rank * 128 + q * 32;
            const float b = GATED ? 0.0f : bias_at<T>(a, f0 + lane);
            // the first chunk's residual values and the L2 lines of the others
            // come while the MMAs run, each further chunk's while the one before
            // it is finished
            TY rv[2][32];
            const bool res = !GATED && a.residual;
            if (res) {
                if (half * 32 < tl.rows) load_residual<TY, 32>(a, rv[0], f0 + lane, (size_t)tl.row0, half * 32, tl.rows);
                for (int c = half * 32 + 64 + lane; c < tl.rows; c += 64)
                    if (f0 < a.n)
                        asm volatile("prefetch.global.L2 [%0];" ::"l"(static_cast<const TY *>(a.residual) +
                                                                      (size_t)(tl.row0 + c) * a.ldr + f0));
            }
            int okw = 0;
            if (lane == 0) okw = mbar_wait(tfull_bar(acc), acc_phase, abort_p, a.gflags, true) ? 1 : 0;
            okw = __shfl_sync(0xffffffffu, okw, 0);
            if (!okw) break;
            tc_fence_after();
            const uint32_t t_base = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * 256);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int c = half * 32 + i * 64;
                if (c >= tl.rows) break;
                if (res && c + 64 < tl.rows)
                    load_residual<TY, 32>(a, rv[(i + 1) & 1], f0 + lane, (size_t)tl.row0, c + 64, tl.rows);
                float v[32];
                __syncwarp();
                tmem_ld32(t_base + (uint32_t)c, reinterpret_cast<uint32_t(&)[32]>(v));
                tmem_wait_ld();
                if constexpr (GATED)
                    epilogue16_gated<false, TY, 32>(a, v, f0, (size_t)tl.row0, c, tl.rows, lane);
                else
                    epilogue16<false, TY, 32>(a, v, rv[i & 1], b, f0 + lane, (size_t)tl.row0, c, tl.rows);
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(acc == 0 ? tempty_leader0 : tempty_leader1);
            if (++acc == 2) {
                acc = 0;
                acc_phase ^= 1u;
            }
        }
        __syncwarp();
    }
    // both CTAs stay until neither needs the other's memory or barriers
    tc_fence_before();
    __syncthreads();
    if (threadIdx.x < 2 && abort_flag) st_cluster(map_to_rank(smem_u32(&pair_abort), threadIdx.x), 1);
    __syncwarp();
    cluster_sync();
    if (pair_abort) {  // the same in both
        if (leader && warp == 0)
            pair_drain(a, bars, pair_issued, ld_cluster(map_to_rank(smem_u32(&pair_issued), 1)), cluster, nclusters,
                       abort_p);
        __syncwarp();
        cluster_sync();
    }
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// ---------------------------------------------------------------------------
// The split kernel: one tile of 128 weight rows x NT tokens per cluster of KS
// CTAs, each on its share of k. The CTAs' partial sums meet in distributed
// shared memory: CTA r adds the columns [r NT / KS, (r + 1) NT / KS) of all of
// them in rank order (a fixed order) and finishes those. Two CTAs fit on an
// SM, so one streams while the other starts or finishes.
// ---------------------------------------------------------------------------
constexpr int S_THREADS = 6 * 32;

// LOW: X has two planes, the tokens' values and what their rounding left; the second
// one's rows are further columns, added to the first's.
template <int NT, bool LOW>
struct SplitCfg {
    static constexpr int COLS = LOW ? 2 * NT : NT;  // the MMA's
    static constexpr int STAGE_BYTES = W_BYTES + COLS * ROW_BYTES;
    static constexpr int STAGES = COLS == 16 ? 6 : COLS == 32 ? 5 : COLS == 64 ? 4 : 3;
    static constexpr int TMEM_COLS = COLS < 32 ? 32 : COLS;
    static constexpr int SMEM = STAGES * STAGE_BYTES + (2 * STAGES + 1) * 8 + 1024;
    static_assert(2 * (SMEM + 1024) <= 233472, "two CTAs per SM");
};

// 16 columns of this thread's lane, with LOW the second plane's added
template <bool LOW>
__device__ __forceinline__ void load16(uint32_t taddr, float (&v)[16]) {
    float w[16];
    tmem_ld16(taddr, reinterpret_cast<uint32_t *>(v));
    if (LOW) tmem_ld16(taddr + 16, reinterpret_cast<uint32_t *>(w));
    tmem_wait_ld();
    if (LOW) {
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = add_low(v[i], w[i]);
    }
}

template <typename T, typename TY, bool GATED, int NT, int KS, bool LOW>
__global__ void __launch_bounds__(S_THREADS, 2)
    k_gemm16_split(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                   const __grid_constant__ Args a) {
    using Cfg = SplitCfg<NT, LOW>;
    constexpr int S = Cfg::STAGES;
    constexpr bool LOW_OUT = NT == 16 && std::is_same<T, TY>::value;  // may write a second plane
    static_assert(!LOW || NT == 16, "the epilogue adds columns i and i + 16");
    extern __shared__ uint8_t smem_raw[];
    __shared__ int abort_flag;
    __shared__ uint32_t tmem_slot;
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t ring = (raw + 1023u) & ~1023u;
    const uint32_t bars = ring + S * Cfg::STAGE_BYTES;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (S + s); };
    const uint32_t done_bar = bars + 8u * (2 * S);
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int rank = KS > 1 ? (int)cluster_rank() : 0;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < S; s++) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(done_bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmW)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tmX)) : "memory");
    }
    // Tensor memory is taken after the wait: a CTA of the kernel before that has yet
    // to allocate its own may share this SM, and would wait for this one while this
    // one waited for it. And before the trigger, for the kernel after in turn. (The
    // pair kernel's shared memory leaves no room for such a neighbour.)
    pdl_wait();
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "r"((uint32_t)Cfg::TMEM_COLS)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_trigger();
    const uint32_t tmem = tmem_slot;
    volatile int *abort_p = &abort_flag;

    const int t = (int)blockIdx.x / KS;
    const int ti = t / a.ftiles, ft = t - ti * a.ftiles;
    int expert = 0, row0, rows;
    if (a.tiles) {
        const bool in = ti < __ldcg(a.n_tiles);  // the grid has room for the longest schedule
        const int4 q = in ? __ldcg(reinterpret_cast<const int4 *>(a.tiles) + ti) : make_int4(0, 0, 0, 0);
        expert = q.x;
        row0 = q.y;
        rows = q.z;
    } else {
        row0 = ti * NT;
        rows = min(NT, a.rows - row0);
    }
    const int all_kb = (a.k + BK - 1) / BK;
    const int kb0 = all_kb * rank / KS, kb1 = all_kb * (rank + 1) / KS;  // KS <= all_kb
    int issued = 0;  // the producer's stages
    if (rows > 0) {  // the same for every CTA of the cluster
        if (warp == 0) {
            // ---------------- producer ----------------
            int r4[4];
            if (a.row_token) {
#pragma unroll
                for (int i = 0; i < 4; i++) {  // past the tile's rows: its first row, into columns that nothing reads
                    const int c = lane * 4 + i;
                    r4[i] = __ldcg(a.row_token + row0 + (c < rows ? c : 0));
                }
            }
            int stage = 0;
            uint32_t phase = 0;
            for (int kb = kb0; kb < kb1; kb++) {
                if (!warp_wait(empty_bar(stage), phase ^ 1u, abort_p, a.gflags, true)) break;
                const uint32_t w_dst = ring + stage * Cfg::STAGE_BYTES, x_dst = w_dst + W_BYTES;
                const uint32_t fb = full_bar(stage);
                if (elect_one()) {
                    mbar_arrive_expect_tx(fb, Cfg::STAGE_BYTES);
                    if (GATED && a.gate16) {
                        tma_load_5d(w_dst, &tmW, fb, kb * BK, 0, 0, ft * 4, expert);
                    } else if (GATED) {
#pragma unroll
                        for (int q = 0; q < 4; q++)
                            tma_load_4d(w_dst + q * 4096, &tmW, fb, kb * BK, ft * 64 + q * 16, 0, expert);
                    } else {
                        tma_load_3d(w_dst, &tmW, fb, kb * BK, ft * 128, expert);
                    }
                    if (!a.row_token) tma_load_2d(x_dst, &tmX, fb, kb * BK, row0);
                    if (LOW) tma_load_2d(x_dst + NT * ROW_BYTES, &tmX, fb, kb * BK, row0 + a.x_low);
                }
                __syncwarp();
                if (a.row_token && lane * 4 < NT) tma_gather4(x_dst + lane * 4 * ROW_BYTES, &tmX, fb, kb * BK, r4);
                issued++;
                if (++stage == S) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        } else if (warp == 1) {
            // ---------------- MMA issuer ----------------
            const uint32_t idesc = idesc_f16(a.fmt, 128, Cfg::COLS);
            int stage = 0;
            uint32_t phase = 0;
            for (int kb = kb0; kb < kb1; kb++) {
                if (!warp_wait(full_bar(stage), phase, abort_p, a.gflags, true)) break;
                tc_fence_after();
                const uint32_t w_addr = ring + stage * Cfg::STAGE_BYTES, x_addr = w_addr + W_BYTES;
                const uint64_t wd = sw128_desc(w_addr), xd = sw128_desc(x_addr);
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < BK / 16; kk++)
                        mma_f16<1>(tmem, wd + 2 * kk, xd + 2 * kk, idesc, kb > kb0 || kk > 0 ? 1u : 0u);
                    tc_commit(empty_bar(stage));
                }
                __syncwarp();
                if (++stage == S) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (elect_one()) tc_commit(done_bar);
            __syncwarp();
            warp_wait(done_bar, 0, abort_p, a.gflags, false);
        }
        // ---------------- epilogue (warps 2 to 5) ----------------
        const int q = warp & 3;
        const int f0 = GATED ? ft * 64 + q * 16 : ft * 128 + q * 32;
        const float b = GATED ? 0.0f : bias_at<T>(a, f0 + lane);
        int go = 0;
        if (warp >= 2) {
            if (lane == 0) go = mbar_wait(done_bar, 0, abort_p, a.gflags, true) ? 1 : 0;
            go = __shfl_sync(0xffffffffu, go, 0);
            tc_fence_after();
        }
        __syncwarp();
        const uint32_t t_base = tmem + ((uint32_t)(q * 32) << 16);
        if constexpr (KS == 1) {
            if (go) {
                constexpr int C = NT < 32 ? NT : 32;
#pragma unroll 1
                for (int c = 0; c < NT && c < rows; c += C) {
                    TY rv[C];
                    if (!GATED && a.residual) load_residual<TY, C>(a, rv, f0 + lane, (size_t)row0, c, rows);
                    float v[C];
                    __syncwarp();
                    if constexpr (C == 32) {
                        tmem_ld32(t_base + (uint32_t)c, reinterpret_cast<uint32_t(&)[32]>(v));
                        tmem_wait_ld();
                    } else {
                        load16<LOW>(t_base + (uint32_t)c, v);
                    }
                    if constexpr (GATED)
                        epilogue16_gated<LOW_OUT, TY, C>(a, v, f0, (size_t)row0, c, rows, lane);
                    else
                        epilogue16<LOW_OUT, TY, C>(a, v, rv, b, f0 + lane, (size_t)row0, c, rows);
                }
            }
        } else {
            // CTA o finishes the columns from o CW on; they lie in its ring as
            // [source CTA][column][128 features]
            constexpr int CW = (NT + 4 * KS - 1) / (4 * KS) * 4;
            constexpr int C = CW % 16 == 0 ? 16 : CW % 8 == 0 ? 8 : 4;
            static_assert(KS * CW * W_ROWS * 4 <= S * Cfg::STAGE_BYTES, "the partial sums reuse the ring");
            cluster_sync();  // every CTA's MMAs and copies are done: the rings are free
            if (warp >= 2) {
#pragma unroll 1
                for (int c = 0; c < NT && c < rows; c += 16) {
                    float v[16];
                    load16<LOW>(t_base + (uint32_t)c, v);
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int o = (c + i) / CW, oc = (c + i) % CW;
                        const uint32_t dst = map_to_rank(ring, (uint32_t)o) +
                                             (uint32_t)(((rank * CW + oc) * W_ROWS + q * 32 + lane) * 4);
                        asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(dst), "f"(v[i]) : "memory");
                    }
                }
            }
            __syncwarp();
            cluster_sync();
            const int c0 = rank * CW, c1 = min(min(c0 + CW, NT), rows);
            if (go) {
                const float *part = reinterpret_cast<const float *>(smem_raw + (ring - raw)) + q * 32 + lane;
#pragma unroll 1
                for (int c = c0; c < c1; c += C) {
                    TY rv[C];
                    if (!GATED && a.residual) load_residual<TY, C>(a, rv, f0 + lane, (size_t)row0, c, rows);
                    float v[C];
#pragma unroll
                    for (int i = 0; i < C; i++) {
                        v[i] = part[(c - c0 + i) * W_ROWS];
#pragma unroll
                        for (int s = 1; s < KS; s++) v[i] += part[(s * CW + c - c0 + i) * W_ROWS];
                    }
                    if constexpr (GATED)
                        epilogue16_gated<LOW_OUT, TY, C>(a, v, f0, (size_t)row0, c, rows, lane);
                    else
                        epilogue16<LOW_OUT, TY, C>(a, v, rv, b, f0 + lane, (size_t)row0, c, rows);
                    __syncwarp();
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    // An aborting CTA leaves no copy in flight behind it, whichever role gave up (the
    // MMA issuer may do so when every stage has been issued).
    if (warp == 0 && abort_flag)
        for (int i = max(0, issued - S); i < issued; i++)
            warp_wait(full_bar(i % S), (uint32_t)(i / S) & 1u, abort_p, a.gflags, false);
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)Cfg::TMEM_COLS)
                     : "memory");
    }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------

// Tensor map of 16-bit elements with 64-wide, 128B-swizzled boxes; dims and
// strides from the innermost out, strides of the outer dims in elements.
bool make_map(CUtensorMap *tm, int dtype, const void *base, int rank, const size_t *dims, const size_t *strides,
              const unsigned *box) {
    auto fn = encode_fn();
    if (!fn || ((uintptr_t)base & 15)) return false;
    cuuint64_t d[5], s[4];
    cuuint32_t b[5], e[5] = {1, 1, 1, 1, 1};
    for (int i = 0; i < rank; i++) {
        d[i] = dims[i];
        b[i] = box[i];
        if (i) {
            s[i - 1] = strides[i - 1] * 2;
            if (s[i - 1] & 15) return false;
        }
    }
    return fn(tm, dtype == TPT_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
              (cuuint32_t)rank, const_cast<void *>(base), d, s, b, e, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

bool weight_map(CUtensorMap *tm, int dtype, const Gemm16 &g) {
    const size_t ldw = g.n > 1 || g.gated ? g.ldw : (size_t)(g.k + 7) / 8 * 8;
    const size_t we = g.experts > 1 ? g.w_expert : (size_t)(g.gated ? 2 : 1) * g.n * ldw;
    // Gated: a tile's rows are 16 gate rows, the 16 up rows of the same features,
    // and so on. With n a multiple of 16 the features are a dimension of 16 and
    // one of n / 16, and one box brings all 128 rows; otherwise a box of 16 + 16
    // rows whose feature dimension ends at n (rows past it read as zero).
    if (g.gated && g.n % 16 == 0) {
        const size_t dims[5] = {(size_t)g.k, 16, 2, (size_t)g.n / 16, (size_t)g.experts};
        const size_t st[4] = {ldw, (size_t)g.n * ldw, 16 * ldw, we};
        const unsigned box[5] = {BK, 16, 2, 4, 1};
        return make_map(tm, dtype, g.w, 5, dims, st, box);
    }
    if (g.gated) {
        const size_t dims[4] = {(size_t)g.k, (size_t)g.n, 2, (size_t)g.experts}, st[3] = {ldw, (size_t)g.n * ldw, we};
        const unsigned box[4] = {BK, 16, 2, 1};
        return make_map(tm, dtype, g.w, 4, dims, st, box);
    }
    const size_t dims[3] = {(size_t)g.k, (size_t)g.n, (size_t)g.experts}, st[2] = {ldw, we};
    const unsigned box[3] = {BK, W_ROWS, 1};
    return make_map(tm, dtype, g.w, 3, dims, st, box);
}
bool token_map(CUtensorMap *tm, int dtype, const Gemm16 &g, unsigned box_rows) {
    const size_t ldx = g.x_rows > 1 ? g.ldx : (size_t)(g.k + 7) / 8 * 8;
    const size_t dims[2] = {(size_t)g.k, (size_t)g.x_rows}, st[1] = {ldx};
    const unsigned box[2] = {BK, g.row_token ? 1u : box_rows};
    return make_map(tm, dtype, g.x, 2, dims, st, box);
}

Args make_args(tpt_cuda_ctx *ctx, int dtype, const Gemm16 &g) {
    Args a = {};
    a.rows = g.rows;
    a.n = g.n;
    a.k = g.k;
    a.fmt = dtype == TPT_DT_BF16 ? 1 : 0;
    a.gate16 = g.n % 16 == 0;
    a.row_token = g.row_token;
    a.tiles = g.tiles;
    a.n_tiles = g.n_tiles;
    a.bias = g.bias;
    a.act = g.act;
    a.residual = g.residual;
    a.ldr = g.ldr;
    a.y = g.y;
    a.ldy = g.ldy;
    a.low = g.y_low;
    a.x_low = g.x_low;
    a.gflags = ctx->d_flags;
    return a;
}

template <typename T, typename TY, bool GATED>
int launch_pair(tpt_cuda_ctx *ctx, int dtype, const Gemm16 &g, int tile_n) {
    auto kern = k_gemm16_pair<T, TY, GATED>;
    static int cached[64] = {};  // pairs of SMs that hold a cluster at the same time
    const int dev = ctx->device & 63;
    if (!cached[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, P_SMEM);
        if (e != cudaSuccess) return cuda_fail(ctx, e, "gemm16_pair smem attribute");
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2 * (ctx->sm_count / 2), 1, 1);
        cfg.blockDim = dim3(P_THREADS, 1, 1);
        cfg.dynamicSmemBytes = P_SMEM;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = 2;
        at[0].val.clusterDim.y = 1;
        at[0].val.clusterDim.z = 1;
        cfg.attrs = at;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
            cudaGetLastError();
            n = ctx->sm_count / 2;
        }
        cached[dev] = n;
    }
    const int pairs = cached[dev];
    Args a = make_args(ctx, dtype, g);
    a.ftiles = (g.n + (GATED ? 127 : 255)) / (GATED ? 128 : 256);
    a.tile_n = tile_n;
    a.group = 8;
    CUtensorMap tw;
    XMaps tx;
    if (!weight_map(&tw, dtype, g) || !token_map(&tx.box[0], dtype, g, 128) || !token_map(&tx.box[1], dtype, g, 64) ||
        !token_map(&tx.box[2], dtype, g, 32))
        return cuda_fail(ctx, cudaErrorInvalidValue, "gemm16_pair tensor map");
    const long long tiles = (g.tiles ? (long long)g.max_tiles : ((long long)g.rows + tile_n - 1) / tile_n) * a.ftiles;
    if (tiles > 0x7fffffffLL) return TPT_UNSUPPORTED;
    const int clusters = tiles < pairs ? (int)tiles : pairs;
    launch_pdl(kern, 2 * clusters, P_THREADS, P_SMEM, ctx->stream, tw, tx, a);
    return after_launch(ctx, "gemm16_pair");
}

// Tokens per tile of a dense product: the fewest cycles by a model of the pair
// kernel. A stage of 64 k values takes ~240 + 1.1 N cycles (521 at N = 256,
// where the MMAs alone take 512), a tile's epilogue ~20 N (more with a residual
// or a smooth activation) and runs beside the next tile's stages; what counts
// are the rounds of tiles over the pairs and the last tile's epilogue.
// Measured: 8192 x 768 x 768 with residual 18.4 us at 256, 15.3 at 176, 14.9 at
// 128, 18.9 at 64; 512 x 4096 x 4096 25.1 at 256, 19.3 at 128; 4096^3 97 at 256,
// 119 at 128.
int pair_tile_n(tpt_cuda_ctx *ctx, const Gemm16 &g) {
    const long long pairs = ctx->sm_count / 2 > 0 ? ctx->sm_count / 2 : 1;
    const long long ft = (g.n + 255) / 256, kb = (g.k + BK - 1) / BK;
    int best_n = 256;
    double best = 0.0;
    for (int n : {256, 224, 192, 176, 160, 128, 96, 64, 32}) {
        const long long tiles = ((g.rows + n - 1) / n) * ft, rounds = (tiles + pairs - 1) / pairs;
        const double main = (double)kb * (240 + 1.1 * n);
        const double epi = n * (20.0 + (g.residual ? 5 : 0) + (g.act == TPT_ACT_GELU || g.act == TPT_ACT_SILU ? 12 : 0));
        const double t = main + (double)(rounds - 1) * (main > epi ? main : epi) + epi;
        if (n == 256 || t < best) {
            best = t;
            best_n = n;
        }
    }
    return best_n;
}

template <typename T, typename TY, bool GATED, int NT, int KS, bool LOW>
int launch_split(tpt_cuda_ctx *ctx, int dtype, const Gemm16 &g) {
    using Cfg = SplitCfg<NT, LOW>;
    auto kern = k_gemm16_split<T, TY, GATED, NT, KS, LOW>;
    static bool done[64] = {};
    const int dev = ctx->device & 63;
    if (!done[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::SMEM);
        // the largest carveout, or only one CTA would fit per SM
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(kern, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        if (e != cudaSuccess) return cuda_fail(ctx, e, "gemm16_split smem attribute");
        done[dev] = true;
    }
    Args a = make_args(ctx, dtype, g);
    a.ftiles = (g.n + (GATED ? 63 : 127)) / (GATED ? 64 : 128);
    CUtensorMap tw, tx;
    if (!weight_map(&tw, dtype, g) || !token_map(&tx, dtype, g, NT))
        return cuda_fail(ctx, cudaErrorInvalidValue, "gemm16_split tensor map");
    const long long tiles = (g.tiles ? (long long)g.max_tiles : ((long long)g.rows + NT - 1) / NT) * a.ftiles;
    if (tiles * KS > 0x7fffffffLL) return TPT_UNSUPPORTED;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * KS));
    cfg.blockDim = dim3(S_THREADS);
    cfg.dynamicSmemBytes = Cfg::SMEM;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = KS;
    at[1].val.clusterDim.y = 1;
    at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = KS > 1 ? 2 : 1;
    (void)cudaLaunchKernelEx(&cfg, kern, tw, tx, a);
    return after_launch(ctx, "gemm16_split");
}

template <typename T, typename TY, bool GATED, int NT, bool LOW = false>
int launch_split_k(tpt_cuda_ctx *ctx, int dtype, const Gemm16 &g, int ks) {
    if constexpr (NT < 128) {  // the wide tile's k is split over 4 CTAs at most (launch_tc)
        if (ks == 8) return launch_split<T, TY, GATED, NT, 8, LOW>(ctx, dtype, g);
        if (ks == 6) return launch_split<T, TY, GATED, NT, 6, LOW>(ctx, dtype, g);
    }
    switch (ks) {
        case 4: return launch_split<T, TY, GATED, NT, 4, LOW>(ctx, dtype, g);
        case 3: return launch_split<T, TY, GATED, NT, 3, LOW>(ctx, dtype, g);
        case 2: return launch_split<T, TY, GATED, NT, 2, LOW>(ctx, dtype, g);
        default: return launch_split<T, TY, GATED, NT, 1, LOW>(ctx, dtype, g);
    }
}

template <typename T, typename TY, bool GATED>
int launch_tc(tpt_cuda_ctx *ctx, int dtype, const Gemm16 &g) {
    const int fw = GATED ? 64 : 128;  // features of a split tile
    const long long ft = (g.n + fw - 1) / fw;
    const int kb = (g.k + BK - 1) / BK;
    // More than 128 tokens go to the pair kernel; 65 to 128 do where its tiles
    // reach half of the pairs or k is too short to be worth splitting (80 x 1024 x
    // 11008: 8.7 us against 11.4, 128 x 768 x 768: 5.3 against 6.1; but 128 x 4096
    // x 4096: 16.9 against 13.9).
    const bool pair = g.tiles ? g.tile_rows > 128
                              : g.rows > 128 || (g.rows > 64 && (((g.n + 255LL) / 256) * 4 >= ctx->sm_count || kb <= 16));
    if (pair) return launch_pair<T, TY, GATED>(ctx, dtype, g, g.tiles ? 256 : pair_tile_n(ctx, g));
    const int nt = g.tiles ? g.tile_rows : g.rows <= 16 ? 16 : g.rows <= 32 ? 32 : g.rows <= 64 ? 64 : 128;
    const long long tiles = (g.tiles ? (long long)g.max_tiles : ((long long)g.rows + nt - 1) / nt) * ft;
    // How many CTAs share a tile's k: as many as are resident at once, three steps
    // each at least. Measured at 32 tiles of 4096 values: 1 25 us, 2 15, 4 and up
    // 10.3; at 86 tiles: 1 27.6, 2 21.9, 3 20.9, 4 27.1 (a third round). The wide
    // tile's exchange costs more than its eighth share saves.
    int ks = 1;
    for (int s : {2, 3, 4, 6, 8})
        if (tiles * s <= 2LL * ctx->sm_count && kb / s >= 3 && (nt < 128 || s <= 4)) ks = s;
    if constexpr (!GATED && std::is_same<TY, float>::value)
        if (g.x_low) return launch_split_k<T, TY, GATED, 16, true>(ctx, dtype, g, ks);  // tiles of 16: the caller's choice
    if (nt == 16) return launch_split_k<T, TY, GATED, 16>(ctx, dtype, g, ks);
    if constexpr (!GATED) {  // gated products are the experts', in tiles of 16, 32 or 256
        if (nt == 64) return launch_split_k<T, TY, GATED, 64>(ctx, dtype, g, ks);
        if (nt == 128) return launch_split_k<T, TY, GATED, 128>(ctx, dtype, g, ks);
    }
    return launch_split_k<T, TY, GATED, 32>(ctx, dtype, g, ks);
}

template <typename T>
int launch_typed(tpt_cuda_ctx *ctx, int dtype, const Gemm16 &g) {
    if (g.gated) return launch_tc<T, T, true>(ctx, dtype, g);
    if (g.y_f32) return launch_tc<T, float, false>(ctx, dtype, g);
    return launch_tc<T, T, false>(ctx, dtype, g);
}

}  // namespace

int launch_gemm16(tpt_cuda_ctx *ctx, int dtype, const Gemm16 &g) {
    return dtype == TPT_DT_BF16 ? launch_typed<__nv_bfloat16>(ctx, dtype, g) : launch_typed<__half>(ctx, dtype, g);
}

}  // namespace tpt
