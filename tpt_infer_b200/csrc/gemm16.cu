// gemm16.cu -- the 16-bit linear layer y = act(x w^T + bias) + residual: its
// entry point, and the copies of operands whose rows TMA cannot read.
#include "gemm16.cuh"

namespace tpt {
namespace {

// A warp per row, 16 bytes a thread from eight 2-byte loads (a row starts on any
// value, so no wider load fits all of them; the loads of a warp share lines).
// 1537 x 1003 and 2051 x 1003 together: 3 us.
__global__ void __launch_bounds__(256) k_pad_rows16(PadJob a, PadJob b) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31;
    const size_t rows = a.rows + b.rows;
    for (size_t i = blockIdx.x * (size_t)8 + (threadIdx.x >> 5); i < rows; i += (size_t)gridDim.x * 8) {
        const bool second = i >= a.rows;
        const size_t r = second ? i - a.rows : i, k = second ? b.k : a.k;
        const size_t pieces = k ? (k + 7) / 8 : 1;
        const uint16_t *__restrict__ src = static_cast<const uint16_t *>(second ? b.src : a.src) + r * (second ? b.ld : a.ld);
        uint4 *__restrict__ dst = static_cast<uint4 *>(second ? b.dst : a.dst) + r * pieces;
        for (size_t p0 = lane; p0 < pieces; p0 += 128) {
            uint32_t e[4][8];
#pragma unroll
            for (int u = 0; u < 4; u++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const size_t c = (p0 + 32 * u) * 8 + j;
                    e[u][j] = c < k ? (uint32_t)__ldg(src + c) : 0u;
                }
#pragma unroll
            for (int u = 0; u < 4; u++)
                if (p0 + 32 * u < pieces)
                    dst[p0 + 32 * u] = make_uint4(e[u][0] | e[u][1] << 16, e[u][2] | e[u][3] << 16,
                                                  e[u][4] | e[u][5] << 16, e[u][6] | e[u][7] << 16);
        }
    }
}

}  // namespace

int launch_pad_rows16(tpt_cuda_ctx *ctx, const PadJob &a, const PadJob &b) {
    const size_t rows = a.rows + b.rows;
    if (rows == 0) return TPT_OK;
    launch_pdl(k_pad_rows16, grid_1d(rows, 8, (unsigned)ctx->sm_count * 8), 256, 0, ctx->stream, a, b);
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
        PadJob jx, jw;
        if (px) {
            jx = PadJob{x, ldx, m, k, ctx->ws};
            g.x = ctx->ws;
            g.ldx = k8;
        }
        if (pw) {
            jw = PadJob{w, ldw, n, k, ctx->ws + xb};
            g.w = ctx->ws + xb;
            g.ldw = k8;
        }
        st = launch_pad_rows16(ctx, jx, jw);
        if (st) return st;
        if (k == 0) g.k = 8;
    }
    return launch_gemm16(ctx, dtype, g);
}

}  // extern "C"
