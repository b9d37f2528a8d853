// gemm16.cuh -- what the 16-bit matrix products (linear layers and the
// experts' products) share: the description of one product, the experts'
// schedule, and the element helpers of their epilogues.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "tc_common.cuh"

namespace tpt {

// One product Y[row, f] = act(sum_k X[row, k] W[f, k] + bias[f]) + R[row, f],
// or, gated, Y[row, f] = act(gate) * up with gate = W[f, :] x and
// up = W[n + f, :] x. Grouped: the rows of tile t go through the weight of
// tiles[t].expert; X's row of a slot is row_token[slot] (the slot itself
// without a list), Y's row is the slot.
// An expert's tiles lie in runs of up to TILE_RUN: `run` holds the tile's place
// in its run (from bit 8) and the run's length (8 bits).
constexpr int TILE_RUN = 8;
// The step in which the products count a tile's columns (with steps of 32 in place of
// 16: 2048 tokens, 8 experts of 4096 x 11008, 2 chosen: 1280 us against 1200).
constexpr int TILE_STEP = 16;
struct Tile16 {
    int expert, row0, rows, run;
};
struct Gemm16 {
    const void *x = nullptr;
    size_t ldx = 0;
    const void *w = nullptr;
    size_t ldw = 0, w_expert = 0;  // elements from one weight row, one expert, to the next
    int rows = 0, n = 0, k = 0;    // rows of X (dense) or slots (grouped); output features; products per output
    int x_rows = 0;                // rows that X has in memory
    int experts = 1;
    bool compact = false;  // w holds only the experts that the call names, in the order of their first choice
    const int *row_token = nullptr;
    const Tile16 *tiles = nullptr;
    const int *n_tiles = nullptr;
    int max_tiles = 0;  // grouped: no schedule has more
    int tile_rows = 0;  // grouped: no tile has more rows
    const void *bias = nullptr;
    int act = 0;
    bool gated = false;
    const void *residual = nullptr;
    size_t ldr = 0;
    void *y = nullptr;
    size_t ldy = 0;
    bool y_f32 = false;
    // Two planes of 16-bit values for 16 bits of the numbers between two products:
    // y's second plane (y_low elements on) takes what y's rounding left, X's second
    // plane (x_low rows on) is added to the first. X's only with tiles of 16 rows, f32 y.
    size_t y_low = 0;
    int x_low = 0;
};

// Device enqueue; dtype TPT_DT_BF16 or TPT_DT_F16, k > 0. The operands' rows
// must pass rows16_ok (the copies below make them).
int launch_gemm16(tpt_cuda_ctx *ctx, int dtype, const Gemm16 &g);

// The kernels of a few tokens, for operands like launch_gemm16's whose weight rows hold
// k values and then zeros up to a multiple of 8: a dense product of
// up to STREAM_TOKENS rows, and both of the experts' products of as many tokens and
// up to STREAM_PAIRS (token, choice) pairs. `in` reads the tokens' rows and writes
// [tile][4][2][ldy], one tile per distinct expert; `out` reads those and writes the
// tokens' weighted sums. (4 x 4096 x 4096: 8.5 us against the split kernel's 10; 8 x 4096
// x 11008: 21.3 against 18.2, since every block reads and holds every token's row.)
// Those rows have to fit STREAM_X_BYTES of shared memory: it is taken from the L1
// that the weights in flight need (with the largest carveout 1 x 4096 x 4096 takes 11 us
// instead of 7).
constexpr int STREAM_TOKENS = 4, STREAM_PAIRS = 32;
constexpr size_t STREAM_X_BYTES = 52 * 1024;
inline size_t stream_x_bytes(size_t rows, size_t k) { return rows * ((k + 63) / 64 * 128 + 16); }
int launch_gemm16_stream(tpt_cuda_ctx *ctx, int dtype, const Gemm16 &g);
int launch_experts_stream(tpt_cuda_ctx *ctx, int dtype, const Gemm16 &in, const Gemm16 &out, const int *ids,
                          const float *weights, int pairs, int top_k);

// Whether TMA can read `rows` rows of 16-bit values ld apart: base and rows on
// 16 bytes.
inline bool rows16_ok(const void *p, size_t ld, size_t rows) {
    return ((uintptr_t)p & 15) == 0 && (rows <= 1 || ld % 8 == 0);
}
// dst [rows][k rounded up to a multiple of 8, at least 8] = src [rows][k],
// zero-filled; three of them in one launch. With ids only the rows of the experts
// that they name are copied (up to 32 pairs, expert_rows rows an expert), to their own
// places or, compact, one after the other in the order of their first choice.
struct PadJob {
    const void *src = nullptr;
    size_t ld = 0, rows = 0, k = 0;
    void *dst = nullptr;
    const int *ids = nullptr;
    int pairs = 0;
    size_t expert_rows = 1;
    bool compact = false;
};
int launch_pad_rows16(tpt_cuda_ctx *ctx, const PadJob &a, const PadJob &b, const PadJob &c);

#ifdef __CUDACC__

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) {
    return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) {
    return __half2float(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
    return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
    return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
    return __float2half_rn(v);
}

// A sum over the values' upper parts and the one over their lower parts. An infinite
// weight makes the first what it is and the second an infinity of any sign, or 0 x inf.
__device__ __forceinline__ float add_low(float upper, float lower) { return isfinite(upper) ? upper + lower : upper; }

// x / (1 + e^-z). HARD takes the hardware's exponential and quotient: a relative error of
// (6 + 1.2 |z|) 2^-23, since the exponential's grows with its argument (under 2^-16 at
// z = -80), far under the rounding to 16 bits that follows; left of -87 the quotient may be
// -0, its limit. Otherwise, for f32 results, expf(-|z|), which left of zero is the numerator
// too, and the hardware's reciprocal with one Newton step: 5 * 2^-23 down to the smallest
// normal results.
template <bool HARD>
__device__ __forceinline__ float over_one_plus_exp(float x, float z) {
    if (HARD) return __fdividef(x, 1.0f + __expf(-z));
    const float e = expf(-fabsf(z)), d = 1.0f + e;
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
    r = fmaf(r, fmaf(-d, r, 1.0f), r);
    return x * (z < 0.0f ? e * r : r);
}

// The activations of the products' epilogues, C values in place, HARD as above; act is
// uniform, so the choice is one branch for all of them. silu has z = x, and gelu
// z = 2 sqrt(2 / pi) (x + 0.044715 x^3), since 0.5 (1 + tanh(z / 2)) = 1 / (1 + e^-z); z's
// own roundings add 2 |z| 2^-23 to the relative error. relu leaves NaN a NaN.
template <bool HARD, int C>
__device__ __forceinline__ void act16(float (&v)[C], int act) {
    if (act == TPT_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < C; i++) v[i] = v[i] < 0.0f ? 0.0f : v[i];
    } else if (act == TPT_ACT_GELU) {
#pragma unroll
        for (int i = 0; i < C; i++)
            v[i] = over_one_plus_exp<HARD>(v[i], v[i] * fmaf(0.0713548162726f * v[i], v[i], 1.5957691216057f));
    } else if (act == TPT_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < C; i++) v[i] = over_one_plus_exp<HARD>(v[i], v[i]);
    }
}

#endif
}  // namespace tpt
