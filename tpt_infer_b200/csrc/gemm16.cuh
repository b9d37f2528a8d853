// gemm16.cuh -- what the 16-bit matrix products (linear layers and the
// experts' products) share: the description of one product, the experts'
// schedule, and the element helpers of their epilogues.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "tc_common.cuh"

namespace tpt {

// One product Y[row, f] = act(sum_k X[row, k] W[f, k] + bias[f]) + R[row, f],
// or, gated, Y[row, f] = act(gate) * up with gate = W[f, :] x and
// up = W[n + f, :] x. Grouped: the rows of tile t go through the weight of
// tiles[t].expert; X's row of a slot is row_token[slot] (the slot itself
// without a list), Y's row is the slot.
struct Tile16 {
    int expert, row0, rows, pad;
};
struct Gemm16 {
    const void *x = nullptr;
    size_t ldx = 0;
    const void *w = nullptr;
    size_t ldw = 0, w_expert = 0;  // elements from one weight row, one expert, to the next
    int rows = 0, n = 0, k = 0;    // rows of X (dense) or slots (grouped); output features; products per output
    int x_rows = 0;                // rows that X has in memory
    int experts = 1;
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
};

// device enqueue; dtype TPT_DT_BF16 or TPT_DT_F16
int launch_gemm16(tpt_cuda_ctx *ctx, int dtype, const Gemm16 &g);
// the tensor-core kernels: whether TMA can read the operands, and the launch
bool gemm16_tc_ok(const Gemm16 &g);
int launch_gemm16_tc(tpt_cuda_ctx *ctx, int dtype, const Gemm16 &g);

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

// silu(x) = x / (1 + e^-x): for very negative x the quotient's denominator is
// +inf and the result -0, the limit
__device__ __forceinline__ float silu(float x) { return __fdividef(x, 1.0f + __expf(-x)); }

__device__ __forceinline__ float act16(float v, int act) {
    if (act == TPT_ACT_SILU) return silu(v);
    return apply_act(v, act);
}

#endif
}  // namespace tpt
