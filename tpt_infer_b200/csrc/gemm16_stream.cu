// gemm16_stream.cu -- the 16-bit products of a few tokens, bound by the stream
// of the weights: a decoding step's linear layers and its tokens' experts.
//
// The weights go from memory to registers in 128-bit loads, several per thread
// in flight, and straight into mma.sync m16n8k16 as the A operand (16 weight
// rows; the tokens are the 8 columns). The k order within 32 values is permuted
// the same way in both operands, so that a thread's 16 bytes of a row are its
// fragments of two MMAs; the tokens' rows wait in shared memory. Every block
// takes an equal range of weight rows, so the SMs' shares of the stream differ
// by one row at most; its eight warps split k (and, summing over experts, the
// experts), and their partial sums meet in shared memory in a fixed order.
//
// 1 x 4096 x 4096 (33.5 MB, 5.1 us at the copy rate) takes 6.3 us, the two products
// of one token's 8 experts of 2048 x 768 (75.5 MB, 11.5 us) 22. The tcgen05 split kernel
// takes 10.3 at the first: there a single SM draws ~50 GB/s through TMA boxes of
// 128-byte lines, and 256 tiles over 148 SMs leave some with twice the work.
#include "gemm16.cuh"

namespace tpt {
namespace {

constexpr int ST_WARPS = 8;
constexpr int ST_T = ST_WARPS * 32;
constexpr int ST_ROWS = 16;   // weight rows of one MMA
constexpr int ST_CHUNK = 64;  // k values of one step of a warp

struct StreamArgs {
    const void *x;
    size_t ldx;
    int tokens;
    const void *w;
    size_t ldw, w_expert;
    int n, k;
    // grouped: the distinct experts of `pairs` ids take one tile each
    const int *ids;
    const float *weights;
    int pairs, top_k, experts;
    int compact;  // w has the tiles' experts only, in the order of the tiles
    const void *bias;
    int act;
    const void *residual;
    size_t ldr;
    void *y;
    size_t ldy;
    unsigned *gflags;
};

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    if constexpr (std::is_same<T, __nv_bfloat16>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                     "{%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight weights where `in` holds (0 elsewhere), read once and not kept in L1
__device__ __forceinline__ uint4 load8(const uint16_t *p, bool in) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (in)
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                     : "l"(p));
    return v;
}

// GATED: y = act(W x) * (W2 x). SUM: y[token] = sum over the experts of
// weight * W_e h_e, h the tiles' rows [tile][token]; otherwise a tile's products go
// to h's rows [tile][token] (dense: to y). Up to 4 tokens. A row of h is two rows of
// 16-bit values, the products rounded and what that rounding left, and they take two
// of the MMA's 8 columns: a token's result comes from a few thousand values of h, and
// how the largest of them happen to round would show in it (up to 1.55 times the
// error of one rounded y).
template <typename T, typename TY, bool GATED, bool SUM>
__global__ void __launch_bounds__(ST_T, 2) k_gemm16_stream(const __grid_constant__ StreamArgs a) {
    constexpr int H = GATED ? 2 : 1;
    constexpr int DEPTH = GATED ? 2 : 4;  // steps in flight: 16 loads of 16 bytes a thread
    constexpr int COLS = 8;
    __shared__ float red[2][ST_WARPS][H][ST_ROWS][COLS];
    __shared__ int tile_expert[32];
    // SUM: per tile the tokens that chose the expert, per tile and token its weight
    // and its staged row, per staged row its tile * 4 + token
    __shared__ int tile_used[SUM ? 32 : 1], slot_of[SUM ? 128 : 1], slot_row[SUM ? 32 : 1];
    __shared__ float tile_w[SUM ? 128 : 1];
    extern __shared__ __align__(16) uint8_t xs[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t = lane & 3;
    const uint16_t *w = static_cast<const uint16_t *>(a.w);
    const uint16_t *x = static_cast<const uint16_t *>(a.x);
    // this block's equal share of `rows`: rows [first, end) (32-bit: a 64-bit
    // division is hundreds of cycles)
    auto share = [](int rows, int &first, int &end) {
        const int q = rows / (int)gridDim.x, r = rows - q * (int)gridDim.x, b = (int)blockIdx.x;
        first = b * q + min(b, r);
        end = first + q + (b < r ? 1 : 0);
    };
    int at = 0, end = 0;  // the block's rows; `at` is the first row of its group
    if (SUM || !a.ids) share(a.n, at, end);
    if (!a.ids) {
        // a dense layer's rows start towards the L2 while the kernel before it ends
        for (int r = at + (int)threadIdx.x; r < end && a.k >= 8; r += ST_T)
            prefetch_l2_bulk(w + (size_t)r * a.ldw, (uint32_t)(a.k & ~7) * 2);
    }
    const int kch = (a.k + ST_CHUNK - 1) / ST_CHUNK;  // steps of one product
    // SUM waits for the kernel before it only where it reads h. That kernel, the
    // first product of the same call, let this one start after its own wait, so what
    // earlier kernels wrote (ids, weights, W) is complete; and it writes only h.
    if (!SUM) {
        pdl_wait();
        pdl_trigger();
    }
    int n_tiles = 1, x_rows = a.tokens;
    if (a.ids) {
        // lane p is pair p; every warp finds the distinct experts (in the order of
        // their first choice), the first one writes the tables
        const int id = lane < a.pairs ? __ldcg(a.ids + lane) : -1;
        const float weight = SUM && lane < a.pairs ? a.weights[lane] : 0.0f;
        const int tok = lane / a.top_k;
        const bool valid = id >= 0 && id < a.experts;
        if (warp == 0 && id >= a.experts) atomicOr(a.gflags + TPT_FLAG_CHECK, 1u);
        const unsigned below = (1u << lane) - 1;
        const unsigned same = __match_any_sync(0xffffffffu, valid ? id : -1 - lane);
        const int leader = __ffs(same) - 1;
        const unsigned firsts = __ballot_sync(0xffffffffu, valid && leader == lane);
        n_tiles = __popc(firsts);
        const int tile = __popc(firsts & ((1u << leader) - 1));
        if (warp == 0 && valid && leader == lane) tile_expert[tile] = a.compact ? tile : id;
        if (SUM) {
            // a token that chose the expert twice takes it once, with both weights
            const unsigned twin = __match_any_sync(0xffffffffu, valid ? id * 4 + tok : -1 - lane);
            const bool row = valid && __ffs(twin) - 1 == lane;
            const unsigned slots = __ballot_sync(0xffffffffu, row);
            x_rows = __popc(slots);
            float sum = weight;
            if (__any_sync(0xffffffffu, valid && __popc(twin) > 1)) {
                sum = 0.0f;
                for (int j = 0; j < 32; j++) {
                    const float v = __shfl_sync(0xffffffffu, weight, j);
                    if (twin >> j & 1) sum += v;
                }
            }
            if (warp == 0 && row) {
                const int slot = __popc(slots & below);
                slot_row[slot] = tile * 4 + tok;
                slot_of[tile * 4 + tok] = slot;
                tile_w[tile * 4 + tok] = sum;
            }
            if (warp == 0 && valid && leader == lane) {
                int used = 0;
                for (unsigned m = same; m; m &= m - 1) used |= 1 << ((__ffs(m) - 1) / a.top_k);
                tile_used[tile] = used;
            }
        }
        __syncthreads();
        if (!SUM) share(n_tiles * a.n, at, end);
    }
    const int chunks = SUM ? kch * n_tiles : kch;  // steps of one output, split over the warps
    const int c0 = chunks * warp / ST_WARPS, c1 = chunks * (warp + 1) / ST_WARPS;
    const size_t half = (size_t)a.n * a.ldw;
    // The warp's walk: groups of up to 16 rows of one expert's features; in a
    // group, the warp's steps [c0, c1) as segments of one expert's k; in a segment,
    // rounds of DEPTH steps. A round's loads go out as soon as the one before it
    // has been consumed, across the ends of segments and groups, so that a group's
    // sums meet while the next group's weights come.
    int rows = 0, out_tile = 0, f = 0;
    int c = c1, tile = 0, kc = 0, last = 0;  // segment of expert `tile`: steps [kc, last) are left
    const uint16_t *p0 = w;
    auto segment = [&]() {
        if (c >= c1) {  // the warp has no step (left) in this group
            kc = last = 0;
            return;
        }
        tile = SUM ? c / kch : out_tile;
        kc = SUM ? c - tile * kch : c;
        last = min(kch, kc + c1 - c);
        c += last - kc;
        p0 = w + (a.ids ? (size_t)tile_expert[tile] * a.w_expert : 0) + (size_t)(f + g) * a.ldw + 8 * t;
    };
    auto group = [&]() {
        rows = 0;
        if (at < end) {
            out_tile = SUM ? 0 : at / a.n;
            f = at - out_tile * a.n;
            const int rem = min(end - at, a.n - f), parts = (rem + ST_ROWS - 1) / ST_ROWS;
            rows = (rem + parts - 1) / parts;
            c = c0;
            segment();
        } else {
            kc = last = 0;
        }
    };
    uint4 buf[DEPTH][4 * H];
    auto fetch = [&]() {
        if (kc >= last) return;
        const bool row0 = g < rows, row1 = g + 8 < rows;
        const uint16_t *p1 = p0 + 8 * a.ldw;
        if (kc + DEPTH <= last && (kc + DEPTH) * ST_CHUNK <= a.k) {
#pragma unroll
            for (int d = 0; d < DEPTH; d++)
#pragma unroll
                for (int h = 0; h < H; h++)
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        const size_t o = h * half + (size_t)(kc + d) * ST_CHUNK + 32 * s;
                        buf[d][h * 4 + s] = load8(p0 + o, row0);
                        buf[d][h * 4 + 2 + s] = load8(p1 + o, row1);
                    }
        } else {
#pragma unroll
            for (int d = 0; d < DEPTH; d++)
#pragma unroll
                for (int h = 0; h < H; h++)
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        const int k0 = (kc + d) * ST_CHUNK + 32 * s;
                        const bool in = kc + d < last && k0 + 8 * t < a.k;  // zeros from k to the word's end
                        const size_t o = h * half + (size_t)k0;
                        buf[d][h * 4 + s] = load8(p0 + o, row0 && in);
                        buf[d][h * 4 + 2 + s] = load8(p1 + o, row1 && in);
                    }
        }
    };
    group();
    if (SUM) {
        fetch();
        pdl_wait();
        pdl_trigger();
    }
    // the tokens' rows, zero past k; 16 bytes more than a multiple of 128 from one
    // to the next, so that eight rows' fragments lie in different banks
    const int xld = kch * ST_CHUNK * 2 + 16;
    const int pieces = kch * (ST_CHUNK / 8);  // of 16 bytes, a row
    // (SUM: the upper halves of h's rows, then the lower ones)
    for (int i = threadIdx.x; i < (SUM ? 2 : 1) * x_rows * pieces; i += ST_T) {  // all in flight together
        const int r = i / pieces, c = (i - r * pieces) * 8;
        const int n = min(max(a.k - c, 0), 8);  // values of this piece
        const int low = SUM && r >= x_rows ? 1 : 0;
        const uint16_t *src = x + (size_t)(SUM ? slot_row[r - low * x_rows] * 2 + low : r) * a.ldx;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(tc::smem_u32(xs) + r * xld + c * 2),
                     "l"(src + (n ? c : 0)), "r"(n * 2)
                     : "memory");
    }
    bool staged = false;  // whether the warp has waited for them
    auto wait_staged = [&]() {
        if (staged) return;
        asm volatile("cp.async.wait_all;" ::: "memory");
        __syncthreads();
        staged = true;
    };

    if (!SUM) fetch();
    int rb = 0;
    while (rows > 0) {
        const int g_rows = rows, g_f = f, g_tile = out_tile;
        float acc[H][4] = {}, sum[4] = {};
        bool more = kc < last;
        while (more) {
            // this lane's column: token g, or, summing, token g % 4 and the upper (g < 4)
            // or lower half of its row
            const int used = SUM ? tile_used[tile] : 0;
            const bool in = SUM ? (used >> (g & 3) & 1) != 0 : g < a.tokens;
            const int xrow = SUM ? (in ? slot_of[tile * 4 + (g & 3)] + (g >> 2) * x_rows : 0) : g;
            const uint8_t *xp = xs + xrow * xld + 16 * t;
            wait_staged();
#pragma unroll
            for (int d = 0; d < DEPTH; d++) {
                if (kc + d >= last) break;
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    uint4 xv = make_uint4(0, 0, 0, 0);
                    if (in) xv = *reinterpret_cast<const uint4 *>(xp + (kc + d) * (ST_CHUNK * 2) + 64 * s);
#pragma unroll
                    for (int h = 0; h < H; h++) {
                        const uint4 lo = buf[d][h * 4 + s], hi = buf[d][h * 4 + 2 + s];
                        mma16816<T>(acc[h], lo.x, hi.x, lo.y, hi.y, xv.x, xv.y);
                        mma16816<T>(acc[h], lo.z, hi.z, lo.w, hi.w, xv.z, xv.w);
                    }
                }
            }
            const int weigh = tile;
            kc += DEPTH;
            const bool seg_end = kc >= last;
            if (seg_end) {
                more = c < c1;
                if (more) {
                    segment();
                } else {
                    at += rows;
                    group();
                }
            }
            fetch();
            if (SUM && seg_end) {  // the warp's share of this expert's products: weigh it
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int tok = (2 * t + (i & 1)) & 3;
                    // a token without this expert takes nothing of it, not 0 x inf
                    if (used >> tok & 1) sum[i] = fmaf(tile_w[weigh * 4 + tok], acc[0][i], sum[i]);
                    acc[0][i] = 0.0f;
                }
            }
        }
        if (c0 >= c1) {  // no share: on to the next group
            at += rows;
            group();
        }
        wait_staged();
#pragma unroll
        for (int h = 0; h < H; h++)
#pragma unroll
            for (int i = 0; i < 2; i++)
                *reinterpret_cast<float2 *>(&red[rb][warp][h][g + 8 * i][2 * t]) =
                    SUM ? make_float2(sum[2 * i], sum[2 * i + 1]) : make_float2(acc[h][2 * i], acc[h][2 * i + 1]);
        __syncthreads();
        // one output a thread: feature g_f + r of token o
        const int r = threadIdx.x & 15, o = threadIdx.x >> 4;
        if (o < COLS && o < a.tokens && r < g_rows) {
            float v[1] = {0.0f}, u = 0.0f, rest = 0.0f;
#pragma unroll
            for (int i = 0; i < ST_WARPS; i++) {
                v[0] += red[rb][i][0][r][o];
                if (SUM) rest += red[rb][i][0][r][o + 4];
                if (GATED) u += red[rb][i][H - 1][r][o];
            }
            if (SUM) v[0] = add_low(v[0], rest);
            if (a.bias) v[0] += to_f32(static_cast<const T *>(a.bias)[g_f + r]);
            act16<!std::is_same<TY, float>::value>(v, a.act);
            if (GATED) v[0] *= u;
            if (a.residual) v[0] += to_f32(static_cast<const TY *>(a.residual)[(size_t)o * a.ldr + g_f + r]);
            if (a.ids && !SUM) {
                TY *h = static_cast<TY *>(a.y) + ((size_t)g_tile * 4 + o) * 2 * a.ldy + g_f + r;
                const TY upper = from_f32<TY>(v[0]);
                const float rest = v[0] - to_f32(upper);
                h[0] = upper;
                h[a.ldy] = from_f32<TY>(isfinite(rest) ? rest : 0.0f);  // inf - inf stays out
            } else {
                static_cast<TY *>(a.y)[(size_t)o * a.ldy + g_f + r] = from_f32<TY>(v[0]);
            }
        }
        rb ^= 1;  // the next group's sums go beside these; the barrier after it frees them
    }
}

template <typename T, typename TY, bool GATED, bool SUM>
int launch(tpt_cuda_ctx *ctx, const StreamArgs &a, long long rows, int x_rows) {
    auto kern = k_gemm16_stream<T, TY, GATED, SUM>;
    static bool done[64] = {};
    const int dev = ctx->device & 63;
    if (!done[dev]) {
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)STREAM_X_BYTES);
        if (e != cudaSuccess) return cuda_fail(ctx, e, "gemm16_stream smem attribute");
        done[dev] = true;
    }
    const long long grid = rows < 2LL * ctx->sm_count ? rows : 2LL * ctx->sm_count;  // two blocks an SM
    launch_pdl(kern, (unsigned)grid, ST_T, stream_x_bytes(x_rows, a.k), ctx->stream, a);
    return after_launch(ctx, "gemm16_stream");
}

StreamArgs base_args(tpt_cuda_ctx *ctx, const Gemm16 &g) {
    StreamArgs a = {};
    a.x = g.x;
    a.ldx = g.ldx;
    a.tokens = g.x_rows;
    a.w = g.w;
    a.ldw = g.ldw;
    a.w_expert = g.w_expert;
    a.compact = g.compact;
    a.n = g.n;
    a.k = g.k;
    a.bias = g.bias;
    a.act = g.act;
    a.residual = g.residual;
    a.ldr = g.ldr;
    a.y = g.y;
    a.ldy = g.ldy;
    a.gflags = ctx->d_flags;
    return a;
}

template <typename T>
int dense_typed(tpt_cuda_ctx *ctx, const Gemm16 &g) {
    const StreamArgs a = base_args(ctx, g);
    return g.y_f32 ? launch<T, float, false, false>(ctx, a, g.n, g.rows) : launch<T, T, false, false>(ctx, a, g.n, g.rows);
}

template <typename T>
int experts_typed(tpt_cuda_ctx *ctx, const Gemm16 &in, const Gemm16 &out, const int *ids, const float *weights,
                  int pairs, int top_k) {
    StreamArgs a = base_args(ctx, in), b = base_args(ctx, out);
    a.ids = b.ids = ids;
    a.weights = b.weights = weights;
    a.pairs = b.pairs = pairs;
    a.top_k = b.top_k = top_k;
    a.experts = b.experts = in.experts;
    b.tokens = a.tokens;
    const long long rows = (long long)in.n * (pairs < in.experts ? pairs : in.experts);
    const int st = in.gated ? launch<T, T, true, false>(ctx, a, rows, a.tokens)
                            : launch<T, T, false, false>(ctx, a, rows, a.tokens);
    return st ? st : launch<T, T, false, true>(ctx, b, out.n, 2 * pairs);
}

}  // namespace

int launch_gemm16_stream(tpt_cuda_ctx *ctx, int dtype, const Gemm16 &g) {
    return dtype == TPT_DT_BF16 ? dense_typed<__nv_bfloat16>(ctx, g) : dense_typed<__half>(ctx, g);
}

int launch_experts_stream(tpt_cuda_ctx *ctx, int dtype, const Gemm16 &in, const Gemm16 &out, const int *ids,
                          const float *weights, int pairs, int top_k) {
    return dtype == TPT_DT_BF16 ? experts_typed<__nv_bfloat16>(ctx, in, out, ids, weights, pairs, top_k)
                                : experts_typed<__half>(ctx, in, out, ids, weights, pairs, top_k);
}

}  // namespace tpt
