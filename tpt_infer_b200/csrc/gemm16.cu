// gemm16.cu -- 16-bit matrix products with their epilogue: the linear layer
// y = act(x w^T + bias) + residual, and one of the experts' products over a
// schedule of (expert, rows) tiles.
#include "gemm16.cuh"

namespace tpt {
namespace {

constexpr int SB = 64, SK = 16;  // output tile, k step

// 64 x 64 outputs per block of 256 threads, 4 x 4 per thread, f32 sums.
// gridDim.x: feature tiles; gridDim.y: row tiles (dense) or schedule tiles.
template <typename T, typename TY, bool GATED>
__global__ void __launch_bounds__(256) k_gemm16_simple(Gemm16 g) {
    pdl_wait();
    pdl_trigger();
    __shared__ float xs[SK][SB + 4], ws[SK][SB + 4], us[GATED ? SK : 1][SB + 4];
    int row0, rows, expert = 0;
    if (g.tiles) {
        const int sub = (g.tile_rows + SB - 1) / SB;
        const int ti = blockIdx.y / sub, off = (blockIdx.y - ti * sub) * SB;
        if (ti >= *g.n_tiles) return;
        const Tile16 t = g.tiles[ti];
        if (off >= t.rows) return;
        row0 = t.row0 + off;
        rows = min(SB, t.rows - off);
        expert = t.expert;
    } else {
        row0 = blockIdx.y * SB;
        rows = min(SB, g.rows - row0);
    }
    const int f0 = blockIdx.x * SB;
    const T *x = static_cast<const T *>(g.x);
    const T *w = static_cast<const T *>(g.w) + (size_t)expert * g.w_expert;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {}, up[4][4] = {};
    for (int k0 = 0; k0 < g.k; k0 += SK) {
        for (int i = threadIdx.x; i < SB * SK; i += 256) {
            const int r = i / SK, c = i % SK;
            const bool kin = k0 + c < g.k;
            float v = 0.0f, a = 0.0f, u = 0.0f;
            if (kin && r < rows) {
                const size_t xr = g.row_token ? (size_t)g.row_token[row0 + r] : (size_t)(row0 + r);
                v = to_f32(x[xr * g.ldx + k0 + c]);
            }
            if (kin && f0 + r < g.n) {
                a = to_f32(w[(size_t)(f0 + r) * g.ldw + k0 + c]);
                if (GATED) u = to_f32(w[(size_t)(g.n + f0 + r) * g.ldw + k0 + c]);
            }
            xs[c][r] = v;
            ws[c][r] = a;
            if (GATED) us[c][r] = u;
        }
        __syncthreads();
#pragma unroll
        for (int c = 0; c < SK; c++) {
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    acc[i][j] = fmaf(xs[c][ty * 4 + i], ws[c][tx * 4 + j], acc[i][j]);
                    if (GATED) up[i][j] = fmaf(xs[c][ty * 4 + i], us[c][tx * 4 + j], up[i][j]);
                }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int r = ty * 4 + i;
        if (r >= rows) continue;
        if (g.bias) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (f0 + tx * 4 + j < g.n) acc[i][j] += to_f32(static_cast<const T *>(g.bias)[f0 + tx * 4 + j]);
        }
        act16(acc[i], g.act);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int f = f0 + tx * 4 + j;
            if (f >= g.n) continue;
            float v = acc[i][j];
            if (GATED) v *= up[i][j];
            if (g.residual) v += to_f32(static_cast<const TY *>(g.residual)[(size_t)(row0 + r) * g.ldr + f]);
            static_cast<TY *>(g.y)[(size_t)(row0 + r) * g.ldy + f] = from_f32<TY>(v);
        }
    }
}

template <typename T>
int launch_simple(tpt_cuda_ctx *ctx, const Gemm16 &g) {
    const dim3 grid((g.n + SB - 1) / SB, g.tiles ? g.max_tiles * ((g.tile_rows + SB - 1) / SB) : (g.rows + SB - 1) / SB);
    if (g.gated)
        launch_pdl(k_gemm16_simple<T, T, true>, grid, 256, 0, ctx->stream, g);
    else if (g.y_f32)
        launch_pdl(k_gemm16_simple<T, float, false>, grid, 256, 0, ctx->stream, g);
    else
        launch_pdl(k_gemm16_simple<T, T, false>, grid, 256, 0, ctx->stream, g);
    return after_launch(ctx, "gemm16_simple");
}

}  // namespace

int launch_gemm16(tpt_cuda_ctx *ctx, int dtype, const Gemm16 &g) {
    if (gemm16_tc_ok(g)) return launch_gemm16_tc(ctx, dtype, g);
    return dtype == TPT_DT_BF16 ? launch_simple<__nv_bfloat16>(ctx, g) : launch_simple<__half>(ctx, g);
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
    return launch_gemm16(ctx, dtype, g);
}

}  // extern "C"
