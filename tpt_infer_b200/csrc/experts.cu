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
#include <type_traits>

#include "gemm16.cuh"

namespace tpt {
namespace {

// ------------------------------------------------------------------ routing

constexpr int ROUTE_WARPS = 8;

// V consecutive logits; vec: as 16-, 8- or 4-byte words
template <typename T, int V>
__device__ __forceinline__ void load_logits(const T *p, bool vec, int n, float (&s)[V]) {
    constexpr int B = V * sizeof(T) >= 16 ? 16 : V * sizeof(T);  // bytes of a word
    constexpr int N = B / sizeof(T);
    if (B >= 4 && vec) {
        using W = typename std::conditional<B == 16, uint4, typename std::conditional<B == 8, uint2, uint32_t>::type>::type;
        if (n > 0) {
#pragma unroll
            for (int i = 0; i < V; i += N) {
                union {
                    W w;
                    T t[N];
                } u;
                u.w = *reinterpret_cast<const W *>(p + i);
#pragma unroll
                for (int j = 0; j < N; j++) s[i + j] = to_f32(u.t[j]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; i++) s[i] = -INFINITY;
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) s[i] = i < n ? to_f32(p[i]) : -INFINITY;
    }
}
// A logit's share of the softmax before the division by the sum; the largest
// logit itself by comparison, so that its term is 1 for +inf too.
__device__ __forceinline__ float softmax_term(float l, float top) { return l == top ? 1.0f : expf(l - top); }
// 1 / (1 + e^-l): the hardware's reciprocal and one Newton step. Under -87 (a
// score below 2^-125) it is 0, since e^-l may not be finite there.
__device__ __forceinline__ float sigmoid_score(float l) {
    const float d = 1.0f + expf(-fmaxf(l, -87.0f));
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    return l < -87.0f ? 0.0f : fmaf(r, fmaf(-d, r, 1.0f), r);
}

// The largest of the warp's floats (no NaN among them)
__device__ __forceinline__ float warp_best(float v) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}

// One warp per token. Each group has 2^lane_bits neighbouring lanes and each of
// them V of its `per` experts in order, so a group's best values meet in
// lane_bits exchanges, and of equal values the lowest lane's lowest one is the
// lowest expert. Each lane keeps its best three in order, and the chosen experts
// come out one per round: the warp's largest value, its first lane, that lane's
// next best. What it does is bound by instructions, not by the 4 E bytes it reads:
// 16384 tokens of 256 experts in 8 groups, 8 chosen, 831 instructions a token,
// 16 us (2.7 at the copy rate); with one expert chosen 9.6. Two best values a lane and
// more rescans: 19.4 us; several tokens a warp by sorting networks: 24.7.
template <typename T, int V>
__global__ void __launch_bounds__(ROUTE_WARPS * 32)
    k_route_experts(const T *__restrict__ logits, size_t ld, int tokens, int per, int softmax,
                    const float *__restrict__ bias, int groups, int groups_kept, int group_top, int lane_bits, int vec,
                    int bias_vec, int top_k, int renormalise, float scale, const uint8_t *__restrict__ mask, int *__restrict__ ids,
                    float *__restrict__ weights) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const int t = blockIdx.x * ROUTE_WARPS + (threadIdx.x >> 5);
    if (t >= tokens) return;
    int id_mine = -1;  // lane j keeps choice j
    float w_mine = 0.0f;
    if (!mask || mask[t]) {
        const float NEG = -INFINITY;
        const int lanes = 1 << lane_bits, q = lane >> lane_bits, sub = lane & (lanes - 1);
        const int n = q < groups ? min(V, per - sub * V) : 0;  // this lane's experts (none: n <= 0)
        const int e0 = q * per + sub * V;
        const T *row = logits + (size_t)t * ld;
        float c[V];
        load_logits<T, V>(row + e0, vec, n, c);
        float top = NEG, rsum = 1.0f;
        if (softmax) {
#pragma unroll
            for (int i = 0; i < V; i++) top = fmaxf(top, c[i]);  // NaN: the other operand
            top = warp_best(top);
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float s = c[i] > NEG ? softmax_term(c[i], top) : 0.0f;
                sum += s;
                c[i] = c[i] > NEG ? s : NEG;  // NaN and -inf: experts that cannot be chosen
            }
            sum = warp_sum(sum);
            rsum = sum > 0.0f ? __frcp_rn(sum) : 0.0f;
#pragma unroll
            for (int i = 0; i < V; i++) c[i] = c[i] > NEG ? c[i] * rsum : NEG;
        } else if (!bias) {
#pragma unroll
            for (int i = 0; i < V; i++) c[i] = c[i] > NEG ? sigmoid_score(c[i]) : NEG;
        }
        if (bias) {
            float bv[V];
            load_logits<float, V>(bias + e0, bias_vec, n, bv);
#pragma unroll
            for (int i = 0; i < V; i++) {
                bv[i] += softmax ? c[i] : sigmoid_score(c[i]);
                c[i] = c[i] > NEG && bv[i] > NEG ? bv[i] : NEG;  // a NaN or -inf bias: off, too
            }
        }
        // This lane's best values below (from, from_i), in order, the lower index first
        // among equals; MORE marks the last of them, behind which others may come.
        constexpr int D = V < 3 ? V : 3, MORE = V > D ? 1 << 16 : 0;
        float b[D];
        int at[D];
        auto scan = [&](bool all, float from, int from_i) {
#pragma unroll
            for (int d = 0; d < D; d++) {
                b[d] = NEG;
                at[d] = 0;
            }
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float v = all || c[i] < from || (c[i] == from && i > from_i) ? c[i] : NEG;
                bool over[D];
#pragma unroll
                for (int d = 0; d < D; d++) over[d] = v > b[d];
#pragma unroll
                for (int d = D - 1; d > 0; d--) {
                    at[d] = over[d - 1] ? at[d - 1] : over[d] ? i : at[d];
                    b[d] = fmaxf(b[d], fminf(b[d - 1], v));
                }
                at[0] = over[0] ? i : at[0];
                b[0] = fmaxf(b[0], v);
            }
            at[D - 1] |= MORE;
        };
        scan(true, 0.0f, 0);
        if (groups > 1) {
            float g1 = b[0], g2 = D > 1 ? b[D > 1 ? 1 : 0] : NEG;
            for (int o = 1; o < lanes; o <<= 1) {
                const float p1 = __shfl_xor_sync(0xffffffffu, g1, o), p2 = __shfl_xor_sync(0xffffffffu, g2, o);
                g2 = fmaxf(fminf(g1, p1), fmaxf(g2, p2));
                g1 = fmaxf(g1, p1);
            }
            // a group's lanes share the comparisons with the other groups
            const float mine = group_top == 2 && g2 > NEG ? g1 + g2 : g1;
            int better = 0;
            for (int g0 = 0; g0 < groups; g0 += lanes) {
                const int g = g0 + sub;
                const float o = __shfl_sync(0xffffffffu, mine, (g << lane_bits) & 31);
                better += g < groups && (o > mine || (o == mine && g < q)) ? 1 : 0;
            }
            for (int o = 1; o < lanes; o <<= 1) better += __shfl_xor_sync(0xffffffffu, better, o);
            if (better >= groups_kept) {  // nothing of this lane can be chosen
#pragma unroll
                for (int d = 0; d < D; d++) b[d] = NEG;
            }
        }
        for (int j = 0; j < top_k; j++) {
            const float best = warp_best(b[0]);
            if (best == NEG) break;  // no expert is left
            const int owner = __ffs(__ballot_sync(0xffffffffu, b[0] == best)) - 1;
            const int e = __shfl_sync(0xffffffffu, e0 + at[0], owner);
            if (lane == j) id_mine = e;
            if (lane == owner) {
#pragma unroll
                for (int d = 0; d + 1 < D; d++) {
                    b[d] = b[d + 1];
                    at[d] = at[d + 1];
                }
                b[D - 1] = NEG;
            }
            if (MORE && (e & MORE) && lane == owner) scan(false, best, (e & (MORE - 1)) - e0);
        }
        if (id_mine >= 0) {
            if (MORE) id_mine &= MORE - 1;
            const float l = to_f32(row[id_mine]);
            w_mine = softmax ? softmax_term(l, top) * rsum : sigmoid_score(l);
        }
        if (renormalise) {
            const float sum = warp_sum(w_mine);
            w_mine = sum > 0.0f ? w_mine / sum : 0.0f;
        }
        w_mine *= scale;
    }
    if (lane < top_k) {
        ids[(size_t)t * top_k + lane] = id_mine;
        weights[(size_t)t * top_k + lane] = w_mine;
    }
}

template <typename T>
void launch_route(tpt_cuda_ctx *ctx, const void *logits, size_t ld, int tokens, int experts, int score,
                  const float *bias, int groups, int groups_kept, int group_top, int top_k, int renormalise,
                  float scale, const uint8_t *mask, int *ids, float *weights) {
    const dim3 grid((tokens + ROUTE_WARPS - 1) / ROUTE_WARPS);
    int lane_bits = 5;
    while (groups << lane_bits > 32) lane_bits--;
    const int per = experts / groups, need = (per + (1 << lane_bits) - 1) >> lane_bits;
    int v = 1;
    while (v < need) v *= 2;
    const size_t word = v * sizeof(T) < 16 ? v * sizeof(T) : 16;
    const bool vec = per % v == 0 && ((uintptr_t)logits % word) == 0 && (tokens == 1 || ld * sizeof(T) % word == 0);
    const size_t bword = v * 4 < 16 ? v * 4 : 16;
    const bool bias_vec = per % v == 0 && ((uintptr_t)bias % bword) == 0;
    auto go = [&](auto kern) {
        launch_pdl(kern, grid, ROUTE_WARPS * 32, 0, ctx->stream, (const T *)logits, ld, tokens, per,
                   score == TPT_SCORE_SOFTMAX, bias, groups, groups_kept, group_top, lane_bits, vec, bias_vec, top_k, renormalise,
                   scale, mask, ids, weights);
    };
    // groups <= 32 and experts <= 1024: at most 64 experts a lane (17 groups of 60)
    if (v == 1)
        go(k_route_experts<T, 1>);
    else if (v == 2)
        go(k_route_experts<T, 2>);
    else if (v == 4)
        go(k_route_experts<T, 4>);
    else if (v == 8)
        go(k_route_experts<T, 8>);
    else if (v == 16)
        go(k_route_experts<T, 16>);
    else if (v == 32)
        go(k_route_experts<T, 32>);
    else
        go(k_route_experts<T, 64>);
}

// ------------------------------------------------------------------ the slots

// Sorts the (token, choice) pairs by expert: pos[i] is pair i's slot (-1: no
// expert), row_token[slot] its token (null: not wanted); tiles lists each
// expert's slots in runs of at most tile_rows, an expert's runs of equal
// length up to TILE_STEP.
// One cluster of eight blocks: each counts its share of the pairs in shared
// memory, the blocks add one another's counts, and each places its share (65536
// pairs of 128 experts: 9 us).
constexpr int PLAN_T = 1024, CL = 8;

__global__ void __cluster_dims__(CL, 1, 1) __launch_bounds__(PLAN_T)
    k_experts_plan(const int *__restrict__ ids, int pairs, int top_k, int experts, int tile_rows, int *pos,
                   int *row_token, Tile16 *tiles, int *n_tiles, unsigned *gflags) {
    extern __shared__ int plan_smem[];
    int *count = plan_smem, *first = plan_smem + experts;
    __shared__ int warp_slots[PLAN_T / 32], warp_tiles[PLAN_T / 32];
    __shared__ int run_slots, run_tiles;
    const int rank = (int)tc::cluster_rank();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int e = threadIdx.x; e < experts; e += PLAN_T) count[e] = 0;
    if (threadIdx.x == 0) run_slots = run_tiles = 0;
    pdl_wait();
    pdl_trigger();
    __syncthreads();
    const int i0 = (int)((long long)pairs * rank / CL), i1 = (int)((long long)pairs * (rank + 1) / CL);
    bool bad = false;
    for (int i = i0 + threadIdx.x; i < i1; i += PLAN_T) {
        const int e = ids[i];
        if (e >= experts)
            bad = true;
        else if (e >= 0)
            atomicAdd(&count[e], 1);
    }
    if (bad) atomicOr(gflags + TPT_FLAG_CHECK, 1u);
    __syncwarp();
    tc::cluster_sync();
    // first[e]: the first slot of this block's pairs of expert e. Exclusive sums
    // over the experts, PLAN_T at a time; block 0 writes the tiles on the way.
    for (int e0 = 0; e0 < experts; e0 += PLAN_T) {
        const int e = e0 + threadIdx.x;
        int total = 0, before = 0;
        if (e < experts) {
            const uint32_t at = tc::smem_u32(count + e);
#pragma unroll
            for (int r = 0; r < CL; r++) {
                int v;
                asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(tc::map_to_rank(at, (uint32_t)r)) : "memory");
                if (r < rank) before += v;
                total += v;
            }
        }
        const int nt = (total + tile_rows - 1) / tile_rows;
        int s = total, n = nt;  // inclusive sums over the warp
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int ps = __shfl_up_sync(0xffffffffu, s, o), pn = __shfl_up_sync(0xffffffffu, n, o);
            if (lane >= o) {
                s += ps;
                n += pn;
            }
        }
        if (lane == 31) {
            warp_slots[warp] = s;
            warp_tiles[warp] = n;
        }
        __syncthreads();
        int ws = run_slots, wn = run_tiles;
        for (int w = 0; w < warp; w++) {
            ws += warp_slots[w];
            wn += warp_tiles[w];
        }
        const int at = ws + s - total;
        if (e < experts) first[e] = at + before;
        if (rank == 0 && nt > 0) {
            int each = (total + nt - 1) / nt;
            each = (each + TILE_STEP - 1) / TILE_STEP * TILE_STEP;
            for (int r = 0, k = wn + n - nt; r < nt; r++, k++) {
                // no tile is empty: (nt - 1) * each <= (nt - 1) * tile_rows < total
                const int place = r % TILE_RUN;
                tiles[k] = Tile16{e, at + r * each, min(each, total - r * each),
                                  place << 8 | min(TILE_RUN, nt - (r - place))};
            }
        }
        __syncthreads();
        if (threadIdx.x == PLAN_T - 1) {
            run_slots = ws + s;
            run_tiles = wn + n;
        }
        __syncthreads();
    }
    if (rank == 0 && threadIdx.x == 0) *n_tiles = run_tiles;
    for (int i = i0 + threadIdx.x; i < i1; i += PLAN_T) {
        const int e = ids[i];
        int slot = -1;
        if (e >= 0 && e < experts) {
            slot = atomicAdd(&first[e], 1);
            if (row_token) row_token[slot] = i / top_k;
        }
        pos[i] = slot;
    }
    __syncwarp();
    tc::cluster_sync();  // the counts are read by the other blocks
}

// xs[pos[t, j], :] = x[t, :] for every choice j: each token's row is read once
// and written to its slots, the rows padded to lds (a multiple of 8) with zeros.
// Bound by the slots' bytes (8192 tokens of 2048 to 8 slots each: 302 MB, 49 us, 94 %
// of the copy rate).
template <typename V>
__global__ void __launch_bounds__(256)
    k_experts_spread(const V *__restrict__ x, size_t ldx, int tokens, int d, const int *pos, int top_k, V *xs,
                     size_t lds) {
    pdl_wait();
    pdl_trigger();
    for (int t = blockIdx.y; t < tokens; t += gridDim.y) {
        const int *p = pos + (size_t)t * top_k;
        for (int i = blockIdx.x * 256 + threadIdx.x; i < (int)lds; i += gridDim.x * 256) {
            V v = {};
            if (i < d) v = x[(size_t)t * ldx + i];
            for (int j = 0; j < top_k; j++) {
                const int s = __ldcg(p + j);
                if (s >= 0) xs[(size_t)s * lds + i] = v;
            }
        }
    }
}

// y[t, i] = r[t, i] + sum_j w[t, j] P[pos[t, j], i], j in order; V consecutive
// values per thread, the rows of up to eight choices in flight together. Bound by P's
// bytes (65536 slots of 2048: 537 MB of f32 and y, 123 us).
template <typename T, int V>
__global__ void __launch_bounds__(256)
    k_experts_combine(const float *p, size_t ldp, const int *pos, const float *__restrict__ weights, int tokens,
                      int top_k, int d, const T *residual, size_t ldr, T *y, size_t ldy) {
    pdl_wait();
    pdl_trigger();
    for (int t = blockIdx.y; t < tokens; t += gridDim.y) {
        const int *ps = pos + (size_t)t * top_k;
        const float *w = weights + (size_t)t * top_k;
        for (int i = (blockIdx.x * 256 + threadIdx.x) * V; i < d; i += gridDim.x * 256 * V) {
            float v[V] = {};
            for (int j0 = 0; j0 < top_k; j0 += 8) {
                int s[8];
                float wj[8], pv[8][V];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    s[j] = j0 + j < top_k ? __ldcg(ps + j0 + j) : -1;
                    wj[j] = j0 + j < top_k ? w[j0 + j] : 0.0f;
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if (s[j] < 0) continue;
                    const float *row = p + (size_t)s[j] * ldp + i;
                    if constexpr (V == 4) {
                        const float4 q = __ldcs(reinterpret_cast<const float4 *>(row));
                        pv[j][0] = q.x;
                        pv[j][1] = q.y;
                        pv[j][2] = q.z;
                        pv[j][3] = q.w;
                    } else {
                        pv[j][0] = __ldcs(row);
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if (s[j] < 0) continue;
#pragma unroll
                    for (int c = 0; c < V; c++) v[c] = fmaf(wj[j], pv[j][c], v[c]);
                }
            }
            const T *r = residual ? residual + (size_t)t * ldr + i : nullptr;
            T *o = y + (size_t)t * ldy + i;
            if constexpr (V == 4) {
                union {
                    uint2 u;
                    T t[4];
                } a, b;
                if (r) {
                    b.u = *reinterpret_cast<const uint2 *>(r);
#pragma unroll
                    for (int c = 0; c < 4; c++) v[c] += to_f32(b.t[c]);
                }
#pragma unroll
                for (int c = 0; c < 4; c++) a.t[c] = from_f32<T>(v[c]);
                *reinterpret_cast<uint2 *>(o) = a.u;
            } else {
                if (r) v[0] += to_f32(*r);
                *o = from_f32<T>(v[0]);
            }
        }
    }
}

// The intermediate results of one chunk of tokens stay under this many bytes
// of workspace.
constexpr size_t EXPERTS_WS_BYTES = (size_t)2 << 30;

template <typename T>
int run_experts(tpt_cuda_ctx *ctx, int dtype, const T *x, size_t ldx, size_t tokens, size_t d, const int *ids,
                const float *weights, size_t top_k, const T *w_in, const T *w_out, size_t experts, size_t f, int act,
                bool gated, const T *residual, size_t ldr, T *y, size_t ldy) {
    auto up8 = [](size_t v) { return (v + 7) / 8 * 8; };
    const size_t ldh = up8(f), lds = up8(d), ldp = (d + 3) / 4 * 4;  // rows start on 16 bytes
    const bool x_ok = d % 8 == 0 && rows16_ok(x, ldx, tokens);
    // Tokens per tile of the products, by what an expert gets on average (experts
    // draw unevenly: many get far more). 128 experts of 2048 x 768, 8 chosen, us with
    // tiles of 16 / 32 / 256: 64 tokens (mean 4) 178 / 182 / 193, 256 tokens (16) 220 /
    // 210 / 225, 512 tokens (32) 305 / 239 / 233, 2048 tokens (128) 862 / 494 / 311.
    const size_t mean = (tokens * top_k + experts - 1) / experts;
    // Calls of few hidden values keep 16 bits of them between the products, in two planes:
    // how the largest of them happen to round would show in the results, in up to 1.6
    // times the error of one rounded y. Over many values that settles at 1.41, with a
    // spread of about 1.8 / sqrt(tokens f): 0.02 from 8192 values on. The planes need tiles
    // of 16 tokens, which leave the MMAs idle. In place of one plane in longer tiles: 12
    // tokens, 8 of 8 experts of 2048 x 768, 30.3 -> 27.7 us; 32 tokens, 2 of 2 of 4096 x 256,
    // 30.0 -> 18.5; 256 tokens, 2 of 8 of 4096 x 32, 35.5 -> 31. (More tokens have so few
    // values only where f is under 32, and take longer: 1024 of f = 8 62 -> 76. 64 tokens, 8
    // of 128 of 2048 x 768, would take 5 % longer.)
    const bool few = tokens <= 16 || (tokens <= 256 && tokens * f <= 8192);
    const int tile_rows = few || mean <= 10 ? 16 : mean <= 24 ? 32 : 256;
    // A few tokens: no plan, no slots, one tile per chosen expert (128 experts of
    // 2048 x 768, 8 chosen: 1 token 22 us against 29, 4 tokens 57 against 58; 8 tokens of
    // 64 experts, 4 chosen: 30 against 24).
    const bool stream = tokens <= 4 && tokens * top_k <= STREAM_PAIRS && stream_x_bytes(tokens, d) <= STREAM_X_BYTES &&
                        stream_x_bytes(2 * tokens * top_k, f) <= STREAM_X_BYTES;
    // With tiles of 16 tokens the product gathers x's rows itself (TMA, four rows
    // an instruction, ~20 cycles a row): no launch and no copy. Longer tiles would
    // wait for those rows (8192 tokens: 1192 us gathered, 49 + 355 us spread), and x is
    // spread over the slots first.
    const bool gather = x_ok && tile_rows == 16;
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t at = off;
        off += Staging::align_up(bytes);
        return at;
    };
    // Weights whose rows TMA and 128-bit loads cannot read are copied first: all
    // of them, or, for a few pairs, the named experts'. (A single row starts on 16
    // bytes whatever its length, but its last load would reach past its end.)
    const T *w_src[2] = {w_in, w_out};
    const size_t w_er[2] = {(gated ? 2 : 1) * f, d}, w_k[2] = {d, f};
    bool pad[2];
    size_t o_w[2] = {0, 0};
    for (int i = 0; i < 2; i++) {
        pad[i] = w_k[i] % 8 != 0 || !rows16_ok(w_src[i], w_k[i], experts * w_er[i]);
        // the few-token kernels find the named experts by the order of their choice, so
        // that one decoded token does not reserve room for every expert
        const size_t room = stream && tokens * top_k < experts ? tokens * top_k : experts;
        if (pad[i]) o_w[i] = take(room * w_er[i] * up8(w_k[i]) * 2);
    }
    const int planes = few ? 2 : 1;
    const size_t per_token = top_k * (planes * ldh * 2 + ldp * 4 + (gather ? 0 : lds * 2) + 8);
    size_t chunk = EXPERTS_WS_BYTES / per_token;
    if (chunk < 1) chunk = 1;
    if (chunk > tokens) chunk = tokens;
    const size_t max_pairs = chunk * top_k;
    const size_t max_tiles = max_pairs / tile_rows + (max_pairs < experts ? max_pairs : experts);
    size_t o_pos = 0, o_tok = 0, o_tiles = 0, o_n = 0, o_x = 0, o_h, o_p = 0;
    if (stream) {
        if (!x_ok) o_x = take(tokens * lds * 2);
        o_h = take((tokens * top_k < experts ? tokens * top_k : experts) * 8 * ldh * 2);
    } else {
        o_pos = take(max_pairs * 4);
        o_tok = take(gather ? max_pairs * 4 : 0);
        o_tiles = take(max_tiles * sizeof(Tile16));
        o_n = take(4);
        o_x = take(gather ? 0 : max_pairs * lds * 2);
        o_h = take(planes * max_pairs * ldh * 2);
        o_p = take(max_pairs * ldp * 4);
    }
    int st = ensure_ws(ctx, off);
    if (st) return st;
    const void *w_use[2];
    size_t w_ld[2];
    PadJob job[3];
    for (int i = 0; i < 2; i++) {
        w_use[i] = pad[i] ? (const void *)(ctx->ws + o_w[i]) : (const void *)w_src[i];
        w_ld[i] = pad[i] ? up8(w_k[i]) : w_k[i];
        if (!pad[i]) continue;
        job[i] = PadJob{w_src[i], w_k[i], experts * w_er[i], w_k[i], ctx->ws + o_w[i], nullptr, 0, w_er[i]};
        if (tokens * top_k <= 32) {
            job[i].ids = ids;
            job[i].pairs = (int)(tokens * top_k);
            job[i].compact = stream;
        }
    }
    if (stream && !x_ok) job[2] = PadJob{x, ldx, tokens, d, ctx->ws + o_x, nullptr, 0, 1};
    st = launch_pad_rows16(ctx, job[0], job[1], job[2]);
    if (st) return st;
    Gemm16 g;
    g.w = w_use[0];
    g.ldw = w_ld[0];
    g.w_expert = w_er[0] * w_ld[0];
    g.n = (int)f;
    g.k = (int)d;
    g.experts = (int)experts;
    g.act = act;
    g.gated = gated;
    g.y = ctx->ws + o_h;
    g.ldy = ldh;
    Gemm16 o;
    o.x = g.y;
    o.ldx = ldh;
    o.w = w_use[1];
    o.ldw = w_ld[1];
    o.w_expert = w_er[1] * w_ld[1];
    o.n = (int)d;
    o.k = (int)f;
    o.experts = (int)experts;
    if (stream) {
        g.compact = pad[0];
        o.compact = pad[1];
        g.x = x_ok ? (const void *)x : (const void *)(ctx->ws + o_x);
        g.ldx = x_ok ? ldx : lds;
        g.x_rows = (int)tokens;
        o.x_rows = 8;
        o.residual = residual;
        o.ldr = ldr;
        o.y = y;
        o.ldy = ldy;
        return launch_experts_stream(ctx, dtype, g, o, ids, weights, (int)(tokens * top_k), (int)top_k);
    }
    int *pos = (int *)(ctx->ws + o_pos), *tok = gather ? (int *)(ctx->ws + o_tok) : nullptr;
    int *n_tiles = (int *)(ctx->ws + o_n);
    Tile16 *tiles = (Tile16 *)(ctx->ws + o_tiles);
    float *p = (float *)(ctx->ws + o_p);
    for (size_t t0 = 0; t0 < tokens; t0 += chunk) {
        const size_t tn = tokens - t0 < chunk ? tokens - t0 : chunk;
        const size_t pairs = tn * top_k;
        const T *xt = x + t0 * ldx;
        launch_pdl(k_experts_plan, CL, PLAN_T, experts * 8, ctx->stream, ids + t0 * top_k, (int)pairs, (int)top_k,
                   (int)experts, tile_rows, pos, tok, tiles, n_tiles, ctx->d_flags);
        st = after_launch(ctx, "experts_plan");
        if (st) return st;
        if (!gather) {
            const unsigned rows = (unsigned)(tn < 16384 ? tn : 16384);
            if (x_ok)
                launch_pdl(k_experts_spread<uint4>, dim3((unsigned)((lds / 8 + 255) / 256), rows), 256, 0, ctx->stream,
                           (const uint4 *)xt, ldx / 8, (int)tn, (int)(d / 8), pos, (int)top_k, (uint4 *)(ctx->ws + o_x),
                           lds / 8);
            else
                launch_pdl(k_experts_spread<uint16_t>, dim3((unsigned)((lds + 255) / 256), rows), 256, 0, ctx->stream,
                           (const uint16_t *)xt, ldx, (int)tn, (int)d, pos, (int)top_k, (uint16_t *)(ctx->ws + o_x),
                           lds);
            st = after_launch(ctx, "experts_spread");
            if (st) return st;
        }
        g.x = gather ? (const void *)xt : (const void *)(ctx->ws + o_x);
        g.ldx = gather ? ldx : lds;
        g.x_rows = (int)(gather ? tn : pairs);
        g.row_token = tok;
        o.x_rows = (int)(planes * pairs);
        if (planes == 2) {
            g.y_low = pairs * ldh;
            o.x_low = (int)pairs;
        }
        o.y = p;
        o.ldy = ldp;
        o.y_f32 = true;
        g.rows = o.rows = (int)pairs;
        g.tiles = o.tiles = tiles;
        g.n_tiles = o.n_tiles = n_tiles;
        g.max_tiles = o.max_tiles = (int)(pairs / tile_rows + (pairs < experts ? pairs : experts));
        g.tile_rows = o.tile_rows = tile_rows;
        st = launch_gemm16(ctx, dtype, g);
        if (st) return st;
        st = launch_gemm16(ctx, dtype, o);
        if (st) return st;
        const T *rt = residual ? residual + t0 * ldr : nullptr;
        T *yt = y + t0 * ldy;
        const bool vec = d % 4 == 0 && ldy % 4 == 0 && ((uintptr_t)yt & 7) == 0 &&
                         (!rt || (ldr % 4 == 0 && ((uintptr_t)rt & 7) == 0));
        const unsigned rows = (unsigned)(tn < 16384 ? tn : 16384);
        if (vec)
            launch_pdl(k_experts_combine<T, 4>, dim3((unsigned)((d + 1023) / 1024), rows), 256, 0, ctx->stream, p, ldp,
                       pos, weights + t0 * top_k, (int)tn, (int)top_k, (int)d, rt, ldr, yt, ldy);
        else
            launch_pdl(k_experts_combine<T, 1>, dim3((unsigned)((d + 255) / 256), rows), 256, 0, ctx->stream, p, ldp,
                       pos, weights + t0 * top_k, (int)tn, (int)top_k, (int)d, rt, ldr, yt, ldy);
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
    if (experts > TPT_ROUTE_MAX_EXPERTS || top_k > TPT_ROUTE_MAX_TOP_K || groups > 32 || tokens > TPT_LINEAR_MAX)
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
    if (tokens > TPT_LINEAR_MAX || d > TPT_LINEAR_MAX || f > TPT_LINEAR_MAX || experts > TPT_EXPERTS_MAX ||
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
