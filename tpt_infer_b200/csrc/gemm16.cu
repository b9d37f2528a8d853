// gemm16.cu -- the 16-bit linear layer y = act(x w^T + bias) + residual: its
// entry point, and the copies of operands whose rows TMA cannot read.
#include "gemm16.cuh"

namespace tpt {
namespace {

__global__ void __launch_bounds__(256)
    k_pad_rows16(const uint16_t *__restrict__ src, size_t ld, size_t rows, size_t k, uint16_t *dst, size_t k8) {
    pdl_wait();
    pdl_trigger();
    const size_t n = rows * k8;
    for (size_t i = blockIdx.x * (size_t)256 + threadIdx.x; i < n; i += (size_t)gridDim.x * 256) {
        const size_t r = i / k8, c = i - r * k8;
        dst[i] = c < k ? src[r * ld + c] : (uint16_t)0;
    }
}

}  // namespace

int launch_pad_rows16(tpt_cuda_ctx *ctx, const void *src, size_t ld, size_t rows, size_t k, void *dst) {
    const size_t k8 = k ? (k + 7) / 8 * 8 : 8;
    launch_pdl(k_pad_rows16, grid_1d(rows * k8, 256), 256, 0, ctx->stream, (const uint16_t *)src, ld, rows, k,
               (uint16_t *)dst, k8);
    return after_launch(ctx, "pad_rows16");
}

}  // namespace tpt

using namespace tpt;

extern "C" {

int tpt_cuda_linear_dev(tpt_cuda_ctx *ctx, int dtype, const void *x, size_t ldx, size_t m, size_t k, const void *w,
                        size_t ldw, size_t n, const void *bias, int act, const void *residual, size_t ldr, void *y,
                        size_t ldy, int y_dtype) {
    if (!ctx) return TPT_INVALID;
    cudaSetDevice(ctx->device);
    if (dtype != TPT_DT_BF16 && dtype != TPT_DT_F16) return TPT_UNSUPPORTED;
    if (y_dtype != dtype && y_dtype != TPT_DT_F32) return TPT_UNSUPPORTED;
    if (act < 0 || act > TPT_ACT_SILU) return TPT_INVALID;
    if (m > 0x7fffffff || n > 0x7fffffff || k > 0x7fffffff) return TPT_UNSUPPORTED;
    if (m == 0 || n == 0) return TPT_OK;
    if (!y || (k && (!x || !w))) return TPT_INVALID;
    if ((m > 1 && (ldx < k || ldy < n || (residual && ldr < n))) || (n > 1 && ldw < k)) return TPT_SHAPE_MISMATCH;
    const uintptr_t ya = y_dtype == TPT_DT_F32 ? 3 : 1;
    if ((((uintptr_t)x | (uintptr_t)w | (uintptr_t)bias) & 1) || (((uintptr_t)y | (uintptr_t)residual) & ya))
        return TPT_INVALID;
    Gemm16 g;
    g.x = x;
    g.ldx = ldx;
    g.w = w;
    g.ldw = ldw;
    g.rows = g.x_rows = (int)m;
    g.n = (int)n;
    g.k = (int)k;
    g.bias = bias;
    g.act = act;
    g.residual = residual;
    g.ldr = ldr;
    g.y = y;
    g.ldy = ldy;
    g.y_f32 = y_dtype == TPT_DT_F32;
    if (k > 0 && m <= STREAM_TOKENS && stream_x_bytes(m, k) <= STREAM_X_BYTES)
        return launch_gemm16_stream(ctx, dtype, g);
    // TMA reads rows that start on 16 bytes; others are copied to the workspace
    // first (k = 0 becomes eight zero products).
    const size_t k8 = k ? (k + 7) / 8 * 8 : 8;
    const bool px = k == 0 || !rows16_ok(x, ldx, m), pw = k == 0 || !rows16_ok(w, ldw, n);
    const size_t xb = px ? Staging::align_up(m * k8 * 2) : 0, wb = pw ? n * k8 * 2 : 0;
    if (px || pw) {
        int st = ensure_ws(ctx, xb + wb);
        if (st) return st;
        if (px) {
            st = launch_pad_rows16(ctx, x, ldx, m, k, ctx->ws);
            if (st) return st;
            g.x = ctx->ws;
            g.ldx = k8;
        }
        if (pw) {
            st = launch_pad_rows16(ctx, w, ldw, n, k, ctx->ws + xb);
            if (st) return st;
            g.w = ctx->ws + xb;
            g.ldw = k8;
        }
        if (k == 0) g.k = 8;
    }
    return launch_gemm16(ctx, dtype, g);
}

}  // extern "C"
