// experts.cu -- mixture-of-experts feed-forward layers: the router's choice
// of experts, and the experts' products over the tokens that chose them.
//
// route:   s = softmax(l) or sigmoid(l); the top_k experts by s + bias, within
//          the best groups; weights s of the chosen, renormalised, scaled
// experts: y[t] = r[t] + sum_j w[t, j] W_out[e] h,  e = ids[t, j],
//          h = act(W_in[e] x[t]), or act(gate) * up of W_in[e]'s two halves
//
// The experts' products run over slots: one slot per (token, choice), sorted
// by expert, so that each expert's weights are read once for all its tokens.
// The order of an expert's slots has no influence on the results: a slot's
// sums do not depend on its neighbours, and the sum over a token's experts
// runs in the order of its choices.
#include "gemm16.cuh"

namespace tpt {
namespace {

// ------------------------------------------------------------------ routing

constexpr int ROUTE_WARPS = 4;

// A total order of floats as unsigned integers; NaN does not occur.
__device__ __forceinline__ unsigned order_key(float v) {
    const unsigned b = __float_as_uint(v);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// One warp per token; lane l holds experts l * V .. l * V + V - 1, so that of
// equal values the lowest lane's lowest one is the lowest expert.
template <typename T, int V>
__global__ void __launch_bounds__(ROUTE_WARPS * 32)
    k_route_experts(const T *__restrict__ logits, size_t ld, int tokens, int experts, int score,
                    const float *__restrict__ bias, int groups, int groups_kept, int group_top, int top_k,
                    int renormalise, float scale, const uint8_t *__restrict__ mask, int *__restrict__ ids,
                    float *__restrict__ weights) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int t = blockIdx.x * ROUTE_WARPS + (threadIdx.x >> 5);
    if (t >= tokens) return;
    int *my_ids = ids + (size_t)t * top_k;
    float *my_w = weights + (size_t)t * top_k;
    if (mask && !mask[t]) {
        for (int j = lane; j < top_k; j += 32) {
            my_ids[j] = -1;
            my_w[j] = 0.0f;
        }
        return;
    }
    const float NEG = -INFINITY;
    const T *row = logits + (size_t)t * ld;
    float s[V], c[V];
    float top = NEG;
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int e = lane * V + i;
        const float l = e < experts ? to_f32(row[e]) : NEG;
        s[i] = l > NEG ? l : NEG;  // NaN: an expert that cannot be chosen
        top = fmaxf(top, s[i]);
    }
    if (score == TPT_SCORE_SOFTMAX) {
        top = warp_max(top);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < V; i++) {
            c[i] = s[i];
            // the largest logit itself by comparison: its term is 1 for +inf too
            s[i] = s[i] == NEG ? 0.0f : s[i] == top ? 1.0f : expf(s[i] - top);
            sum += s[i];
        }
        sum = warp_sum(sum);
#pragma unroll
        for (int i = 0; i < V; i++) s[i] = sum > 0.0f ? s[i] / sum : 0.0f;
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) {
            c[i] = s[i];
            s[i] = s[i] == NEG ? 0.0f : 1.0f / (1.0f + expf(-s[i]));
        }
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
        const int e = lane * V + i;
        const float b = c[i] == NEG ? NEG : bias ? s[i] + bias[e] : s[i];
        c[i] = b > NEG ? b : NEG;  // a NaN or -inf bias switches the expert off
    }
    if (groups > 1) {
        // lane q's verdict on group q; each group's best one or two values by
        // warp maxima over the lanes' members
        const int per = experts / groups;
        float mine = NEG;
        for (int q = 0; q < groups; q++) {
            float b1 = NEG, b2 = NEG;
#pragma unroll
            for (int i = 0; i < V; i++) {
                const int e = lane * V + i;
                const float v = e >= q * per && e < (q + 1) * per ? c[i] : NEG;
                if (v > b1) {
                    b2 = b1;
                    b1 = v;
                } else {
                    b2 = fmaxf(b2, v);
                }
            }
            const float m1 = warp_max(b1);
            if (group_top == 2 && m1 > NEG) {
                const int owner = __ffs(__ballot_sync(0xffffffffu, b1 == m1)) - 1;
                const float m2 = warp_max(lane == owner ? b2 : b1);
                b1 = m2 > NEG ? m1 + m2 : m1;
            } else {
                b1 = m1;
            }
            if (lane == q) mine = b1;
        }
        unsigned kept = 0;
        for (int r = 0; r < groups_kept; r++) {
            const unsigned key = lane < groups && !(kept >> lane & 1) ? order_key(mine + 0.0f) : 0u;
            const unsigned best = __reduce_max_sync(0xffffffffu, key);
            kept |= 1u << (__ffs(__ballot_sync(0xffffffffu, key == best && lane < groups && !(kept >> lane & 1))) - 1);
        }
#pragma unroll
        for (int i = 0; i < V; i++) {
            const int e = lane * V + i;
            if (e < experts && !(kept >> (e / per) & 1)) c[i] = NEG;
        }
    }
    float w_mine = 0.0f, sum = 0.0f;  // lane j keeps choice j
    int id_mine = -1;
    for (int j = 0; j < top_k; j++) {
        float b = NEG, sv = 0.0f;
        int at = 0;
#pragma unroll
        for (int i = 0; i < V; i++)
            if (c[i] > b) {
                b = c[i];
                sv = s[i];
                at = i;
            }
        const unsigned key = order_key(b + 0.0f);  // -0 counts as 0
        const unsigned best = __reduce_max_sync(0xffffffffu, key);
        if (best == order_key(NEG)) break;  // no expert is left
        const int owner = __ffs(__ballot_sync(0xffffffffu, key == best)) - 1;
        const int e = __shfl_sync(0xffffffffu, lane * V + at, owner);
        const float w = __shfl_sync(0xffffffffu, sv, owner);
        sum += w;
        if (lane == j) {
            id_mine = e;
            w_mine = w;
        }
        if (lane == owner) {
#pragma unroll
            for (int i = 0; i < V; i++)
                if (i == at) c[i] = NEG;
        }
    }
    if (renormalise) w_mine = sum > 0.0f ? w_mine / sum : 0.0f;
    if (lane < top_k) {
        my_ids[lane] = id_mine;
        my_w[lane] = w_mine * scale;
    }
}

template <typename T>
void launch_route(tpt_cuda_ctx *ctx, const void *logits, size_t ld, int tokens, int experts, int score,
                  const float *bias, int groups, int groups_kept, int group_top, int top_k, int renormalise,
                  float scale, const uint8_t *mask, int *ids, float *weights) {
    const dim3 grid((tokens + ROUTE_WARPS - 1) / ROUTE_WARPS);
    auto go = [&](auto kern) {
        launch_pdl(kern, grid, ROUTE_WARPS * 32, 0, ctx->stream, (const T *)logits, ld, tokens, experts, score, bias,
                   groups, groups_kept, group_top, top_k, renormalise, scale, mask, ids, weights);
    };
    if (experts <= 32)
        go(k_route_experts<T, 1>);
    else if (experts <= 64)
        go(k_route_experts<T, 2>);
    else if (experts <= 128)
        go(k_route_experts<T, 4>);
    else if (experts <= 256)
        go(k_route_experts<T, 8>);
    else if (experts <= 512)
        go(k_route_experts<T, 16>);
    else
        go(k_route_experts<T, 32>);
}

// ------------------------------------------------------------------ the slots

// Sorts the (token, choice) pairs by expert: pos[i] is pair i's slot (-1: no
// expert), row_token[slot] its token; tiles lists each expert's slots in runs
// of at most tile_rows. One block.
__global__ void __launch_bounds__(1024)
    k_experts_plan(const int *__restrict__ ids, int pairs, int top_k, int experts, int tile_rows, int *__restrict__ pos,
                   int *__restrict__ row_token, Tile16 *__restrict__ tiles, int *__restrict__ n_tiles,
                   unsigned *gflags) {
    extern __shared__ int plan_smem[];
    int *count = plan_smem, *first = plan_smem + experts;
    pdl_wait();
    pdl_trigger();
    for (int e = threadIdx.x; e < experts; e += 1024) count[e] = 0;
    __syncthreads();
    bool bad = false;
    for (int i = threadIdx.x; i < pairs; i += 1024) {
        const int e = ids[i];
        if (e >= experts)
            bad = true;
        else if (e >= 0)
            atomicAdd(&count[e], 1);
    }
    if (bad) atomicOr(gflags + TPT_FLAG_CHECK, 1u);
    __syncthreads();
    if (threadIdx.x == 0) {
        int at = 0, nt = 0;
        for (int e = 0; e < experts; e++) {
            first[e] = at;
            for (int r = 0; r < count[e]; r += tile_rows)
                tiles[nt++] = Tile16{e, at + r, min(tile_rows, count[e] - r), 0};
            at += count[e];
        }
        *n_tiles = nt;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < pairs; i += 1024) {
        const int e = ids[i];
        int slot = -1;
        if (e >= 0 && e < experts) {
            slot = atomicAdd(&first[e], 1);
            row_token[slot] = i / top_k;
        }
        pos[i] = slot;
    }
}

// y[t, d] = r[t, d] + sum_j w[t, j] P[pos[t, j], d], j in order
template <typename T>
__global__ void __launch_bounds__(256)
    k_experts_combine(const float *__restrict__ p, const int *__restrict__ pos, const float *__restrict__ weights,
                      int tokens, int top_k, int d, const T *residual, size_t ldr, T *y, size_t ldy) {
    pdl_wait();
    pdl_trigger();
    for (int t = blockIdx.x; t < tokens; t += gridDim.x)
        for (int i = threadIdx.x; i < d; i += 256) {
            float v = 0.0f;
            for (int j = 0; j < top_k; j++) {
                const int s = pos[(size_t)t * top_k + j];
                if (s >= 0) v = fmaf(weights[(size_t)t * top_k + j], p[(size_t)s * d + i], v);
            }
            if (residual) v += to_f32(residual[(size_t)t * ldr + i]);
            y[(size_t)t * ldy + i] = from_f32<T>(v);
        }
}

// The products' intermediate results of one chunk of tokens stay under this
// many bytes of workspace.
constexpr size_t EXPERTS_WS_BYTES = (size_t)2 << 30;

template <typename T>
int run_experts(tpt_cuda_ctx *ctx, int dtype, const T *x, size_t ldx, size_t tokens, size_t d, const int *ids,
                const float *weights, size_t top_k, const T *w_in, const T *w_out, size_t experts, size_t f, int act,
                bool gated, const T *residual, size_t ldr, T *y, size_t ldy) {
    const size_t ldh = (f + 7) / 8 * 8;  // rows of h start on 16 bytes
    const size_t per_token = top_k * (ldh * 2 + d * 4 + 8);
    size_t chunk = EXPERTS_WS_BYTES / per_token;
    if (chunk < 1) chunk = 1;
    if (chunk > tokens) chunk = tokens;
    // tokens per tile: what an expert gets on average, up to the pair kernel's 256
    const size_t mean = (tokens * top_k + experts - 1) / experts;
    const int tile_rows = mean <= 16 ? 16 : mean <= 32 ? 32 : mean <= 64 ? 64 : mean <= 128 ? 128 : 256;
    for (size_t t0 = 0; t0 < tokens; t0 += chunk) {
        const size_t tn = tokens - t0 < chunk ? tokens - t0 : chunk;
        const size_t pairs = tn * top_k;
        const size_t max_tiles = pairs / tile_rows + (pairs < experts ? pairs : experts);
        size_t off = 0;
        auto take = [&](size_t bytes) {
            const size_t at = off;
            off += Staging::align_up(bytes);
            return at;
        };
        const size_t o_pos = take(pairs * 4), o_tok = take(pairs * 4), o_tiles = take(max_tiles * sizeof(Tile16)),
                     o_n = take(4), o_h = take(pairs * ldh * 2), o_p = take(pairs * d * 4);
        int st = ensure_ws(ctx, off);
        if (st) return st;
        int *pos = (int *)(ctx->ws + o_pos), *tok = (int *)(ctx->ws + o_tok), *n_tiles = (int *)(ctx->ws + o_n);
        Tile16 *tiles = (Tile16 *)(ctx->ws + o_tiles);
        launch_pdl(k_experts_plan, 1, 1024, experts * 8, ctx->stream, ids + t0 * top_k, (int)pairs, (int)top_k,
                   (int)experts, tile_rows, pos, tok, tiles, n_tiles, ctx->d_flags);
        st = after_launch(ctx, "experts_plan");
        if (st) return st;
        Gemm16 g;
        g.x = x + t0 * ldx;
        g.ldx = ldx;
        g.x_rows = (int)tn;
        g.w = w_in;
        g.ldw = d;
        g.w_expert = (gated ? 2 : 1) * f * d;
        g.rows = (int)pairs;
        g.n = (int)f;
        g.k = (int)d;
        g.experts = (int)experts;
        g.row_token = tok;
        g.tiles = tiles;
        g.n_tiles = n_tiles;
        g.max_tiles = (int)max_tiles;
        g.tile_rows = tile_rows;
        g.act = act;
        g.gated = gated;
        g.y = ctx->ws + o_h;
        g.ldy = ldh;
        st = launch_gemm16(ctx, dtype, g);
        if (st) return st;
        Gemm16 o;
        o.x = g.y;
        o.ldx = ldh;
        o.x_rows = (int)pairs;
        o.w = w_out;
        o.ldw = f;
        o.w_expert = d * f;
        o.rows = (int)pairs;
        o.n = (int)d;
        o.k = (int)f;
        o.experts = (int)experts;
        o.tiles = tiles;
        o.n_tiles = n_tiles;
        o.max_tiles = (int)max_tiles;
        o.tile_rows = tile_rows;
        o.y = ctx->ws + o_p;
        o.ldy = d;
        o.y_f32 = true;
        st = launch_gemm16(ctx, dtype, o);
        if (st) return st;
        launch_pdl(k_experts_combine<T>, (unsigned)(tn < 148 * 16 ? tn : 148 * 16), 256, 0, ctx->stream,
                   (const float *)(ctx->ws + o_p), pos, weights + t0 * top_k, (int)tn, (int)top_k, (int)d,
                   residual ? residual + t0 * ldr : nullptr, ldr, y + t0 * ldy, ldy);
        st = after_launch(ctx, "experts_combine");
        if (st) return st;
    }
    return TPT_OK;
}

}  // namespace
}  // namespace tpt

using namespace tpt;

extern "C" {

int tpt_cuda_route_experts_dev(tpt_cuda_ctx *ctx, const void *logits, int dtype, size_t ld, size_t tokens,
                               size_t experts, int score, const float *bias, size_t groups, size_t groups_kept,
                               size_t group_top, size_t top_k, int renormalise, float scale, const uint8_t *mask,
                               int32_t *ids, float *weights) {
    if (!ctx) return TPT_INVALID;
    cudaSetDevice(ctx->device);
    if (dtype != TPT_DT_F32 && dtype != TPT_DT_BF16 && dtype != TPT_DT_F16) return TPT_UNSUPPORTED;
    if (score != TPT_SCORE_SOFTMAX && score != TPT_SCORE_SIGMOID) return TPT_INVALID;
    if (experts == 0 || top_k == 0 || groups == 0 || groups_kept == 0) return TPT_INVALID;
    if (experts > TPT_ROUTE_MAX_EXPERTS || top_k > TPT_ROUTE_MAX_TOP_K || groups > 32 || tokens > 0x7fffffff)
        return TPT_UNSUPPORTED;
    if (experts % groups || groups_kept > groups || (group_top != 1 && group_top != 2)) return TPT_INVALID;
    if (top_k > groups_kept * (experts / groups)) return TPT_INVALID;
    if (tokens == 0) return TPT_OK;
    if (!logits || !ids || !weights) return TPT_INVALID;
    if (tokens > 1 && ld < experts) return TPT_SHAPE_MISMATCH;
    if (((uintptr_t)logits & (dtype == TPT_DT_F32 ? 3 : 1)) ||
        (((uintptr_t)bias | (uintptr_t)ids | (uintptr_t)weights) & 3))
        return TPT_INVALID;
    auto go = [&](auto tag) {
        launch_route<decltype(tag)>(ctx, logits, ld, (int)tokens, (int)experts, score, bias, (int)groups,
                                    (int)groups_kept, (int)group_top, (int)top_k, renormalise, scale, mask, ids,
                                    weights);
    };
    if (dtype == TPT_DT_F32)
        go(float());
    else if (dtype == TPT_DT_BF16)
        go(__nv_bfloat16());
    else
        go(__half());
    return after_launch(ctx, "route_experts");
}

int tpt_cuda_experts_mlp_dev(tpt_cuda_ctx *ctx, int dtype, const void *x, size_t ldx, size_t tokens, size_t d,
                             const int32_t *ids, const float *weights, size_t top_k, const void *w_in,
                             const void *w_out, size_t experts, size_t f, int act, int gated, const void *residual,
                             size_t ldr, void *y, size_t ldy) {
    if (!ctx) return TPT_INVALID;
    cudaSetDevice(ctx->device);
    if (dtype != TPT_DT_BF16 && dtype != TPT_DT_F16) return TPT_UNSUPPORTED;
    if (act < 0 || act > TPT_ACT_SILU || experts == 0 || top_k == 0 || f == 0) return TPT_INVALID;
    if (tokens > 0x7fffffff || d > 0x3fffffff || f > 0x3fffffff || experts > TPT_EXPERTS_MAX ||
        top_k > TPT_EXPERTS_MAX)
        return TPT_UNSUPPORTED;
    if (tokens == 0 || d == 0) return TPT_OK;
    if (!x || !ids || !weights || !w_in || !w_out || !y) return TPT_INVALID;
    if (tokens > 1 && (ldx < d || ldy < d || (residual && ldr < d))) return TPT_SHAPE_MISMATCH;
    if ((((uintptr_t)x | (uintptr_t)w_in | (uintptr_t)w_out | (uintptr_t)residual | (uintptr_t)y) & 1) ||
        (((uintptr_t)ids | (uintptr_t)weights) & 3))
        return TPT_INVALID;
    if (dtype == TPT_DT_BF16)
        return run_experts<__nv_bfloat16>(ctx, dtype, (const __nv_bfloat16 *)x, ldx, tokens, d, ids, weights, top_k,
                                          (const __nv_bfloat16 *)w_in, (const __nv_bfloat16 *)w_out, experts, f, act,
                                          gated != 0, (const __nv_bfloat16 *)residual, ldr, (__nv_bfloat16 *)y, ldy);
    return run_experts<__half>(ctx, dtype, (const __half *)x, ldx, tokens, d, ids, weights, top_k,
                               (const __half *)w_in, (const __half *)w_out, experts, f, act, gated != 0,
                               (const __half *)residual, ldr, (__half *)y, ldy);
}

}  // extern "C"
