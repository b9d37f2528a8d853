// gemm16.cu -- the 16-bit linear layer y = act(x w^T + bias) + residual: its
// entry point, and the copies of operands whose rows TMA cannot read.
#include "gemm16.cuh"

namespace tpt {
namespace {

// A row starts on any value, so each lane loads the aligned 16 bytes that hold
// the start of its piece, takes the next 16 from its neighbour and shifts the
// piece out of the two: every byte is loaded once, in whole lines (eight 2-byte
// loads a piece touch every sector eight times). WHOLE: all those aligned words
// lie inside the operand; otherwise the ones that reach past its ends are put
// together from single values.
template <bool WHOLE>
__device__ __forceinline__ void pad_row(uintptr_t first, uintptr_t last, uintptr_t row, size_t k, size_t pieces,
                                        uint4 *dst, int lane) {
    const uintptr_t base = row & ~(uintptr_t)15;
    const int off = (int)(row & 15);  // even
    auto word = [&](size_t n) {
        const uintptr_t at = base + n * 16;
        if (WHOLE || (at >= first && at + 16 <= last)) return __ldg(reinterpret_cast<const uint4 *>(at));
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (at + 2 * j >= first && at + 2 * j + 2 <= last)
                w[j / 2] |= (uint32_t)__ldg(reinterpret_cast<const uint16_t *>(at + 2 * j)) << (16 * (j & 1));
        return make_uint4(w[0], w[1], w[2], w[3]);
    };
    constexpr int U = 6;  // loads in flight
    for (size_t p0 = 0; p0 < pieces; p0 += 31 * U) {  // 31 pieces a load: the last lane's word is its neighbour's next
        uint4 v[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const size_t c = p0 + 31 * u + lane;
            v[u] = c <= pieces ? word(c) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (p0 + 31 * u >= pieces) break;
            const size_t c = p0 + 31 * u + lane;
            uint32_t w[8] = {v[u].x, v[u].y, v[u].z, v[u].w,
                             __shfl_down_sync(0xffffffffu, v[u].x, 1), __shfl_down_sync(0xffffffffu, v[u].y, 1),
                             __shfl_down_sync(0xffffffffu, v[u].z, 1), __shfl_down_sync(0xffffffffu, v[u].w, 1)};
            if (off & 8) {
#pragma unroll
                for (int j = 0; j < 6; j++) w[j] = w[j + 2];
            }
            if (off & 4) {
#pragma unroll
                for (int j = 0; j < 5; j++) w[j] = w[j + 1];
            }
            const uint32_t sh = (uint32_t)(off & 2) * 8;
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; j++) {
                o[j] = __funnelshift_r(w[j], w[j + 1], sh);
                const size_t e = c * 8 + 2 * j;  // values past k are zero
                o[j] = e >= k ? 0u : e + 1 >= k ? o[j] & 0xffffu : o[j];
            }
            if (lane < 31 && c < pieces) dst[c] = make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

// blockIdx.y: the operand; a warp per row. Bound by the bytes read and written (1003 and
// 1537 rows of 2051: 21 MB, ~5 us, from L2 in part). COMPACT: the jobs with ids are compact
// (a template argument: chosen at run time it cost 8 registers and 0.2 us everywhere).
template <bool COMPACT>
__global__ void __launch_bounds__(256) k_pad_rows16(PadJob a, PadJob b, PadJob c) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, job = blockIdx.y;
    const void *src = job == 0 ? a.src : job == 1 ? b.src : c.src;
    void *dst = job == 0 ? a.dst : job == 1 ? b.dst : c.dst;
    const int *ids = job == 0 ? a.ids : job == 1 ? b.ids : c.ids;
    const size_t ld = job == 0 ? a.ld : job == 1 ? b.ld : c.ld, k = job == 0 ? a.k : job == 1 ? b.k : c.k;
    const size_t all = job == 0 ? a.rows : job == 1 ? b.rows : c.rows;
    const size_t er = job == 0 ? a.expert_rows : job == 1 ? b.expert_rows : c.expert_rows;
    const int pairs = job == 0 ? a.pairs : job == 1 ? b.pairs : c.pairs;
    size_t rows = all;
    int id = -1;
    unsigned firsts = 0;
    if (ids) {  // the named experts' rows, in the order of their first choice
        id = lane < pairs ? __ldcg(ids + lane) : -1;
        const bool valid = id >= 0 && (size_t)id < all / er;
        const unsigned same = __match_any_sync(0xffffffffu, valid ? id : -1 - lane);
        firsts = __ballot_sync(0xffffffffu, valid && __ffs(same) - 1 == lane);
        rows = __popc(firsts) * er;
    }
    const size_t pieces = k ? (k + 7) / 8 : 1;
    // an operand without values (k = 0) may be a null pointer with any stride: no word lies inside it
    const uintptr_t first = reinterpret_cast<uintptr_t>(src), last = first + (k ? ((all - 1) * ld + k) * 2 : 0);
    for (size_t i = blockIdx.x * (size_t)8 + (threadIdx.x >> 5); i < rows; i += (size_t)gridDim.x * 8) {
        size_t r = i;
        if (ids) {
            const int tile = (int)(i / er);
            r = (size_t)__shfl_sync(0xffffffffu, id, __fns(firsts, 0, tile + 1)) * er + (i - tile * er);
        }
        const uintptr_t row = first + r * ld * 2, base = row & ~(uintptr_t)15;
        uint4 *out = static_cast<uint4 *>(dst) + (COMPACT ? i : r) * pieces;
        if (base >= first && base + (pieces + 1) * 16 <= last)
            pad_row<true>(first, last, row, k, pieces, out, lane);
        else
            pad_row<false>(first, last, row, k, pieces, out, lane);
    }
}

}  // namespace

int launch_pad_rows16(tpt_cuda_ctx *ctx, const PadJob &a, const PadJob &b, const PadJob &c) {
    if (a.rows + b.rows + c.rows == 0) return TPT_OK;
    size_t most = 0;
    for (const PadJob *j : {&a, &b, &c}) {
        const size_t named = j->pairs * j->expert_rows, rows = j->ids && named < j->rows ? named : j->rows;
        if (rows > most) most = rows;
    }
    auto kern = a.compact || b.compact ? k_pad_rows16<true> : k_pad_rows16<false>;
    launch_pdl(kern, dim3(grid_1d(most, 8, (unsigned)ctx->sm_count * 8), c.rows ? 3 : b.rows ? 2 : 1), 256, 0,
               ctx->stream, a, b, c);
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
    if (m > TPT_LINEAR_MAX || n > TPT_LINEAR_MAX || k > TPT_LINEAR_MAX) return TPT_UNSUPPORTED;
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
            jx = PadJob{x, ldx, m, k, ctx->ws, nullptr, 0, 1};
            g.x = ctx->ws;
            g.ldx = k8;
        }
        if (pw) {
            jw = PadJob{w, ldw, n, k, ctx->ws + xb, nullptr, 0, 1};
            g.w = ctx->ws + xb;
            g.ldw = k8;
        }
        st = launch_pad_rows16(ctx, jx, jw, PadJob{});
        if (st) return st;
        if (k == 0) g.k = 8;
    }
    // The stream kernel reads weights eight at a time: past k the rows must hold the
    // copy's zeros, not what lies between strided rows or behind a single one (the
    // other kernels' maps end at k; 1 x 4096 x 4093 in rows of 4096: 9.8 us there, 18.4
    // copied first).
    const bool whole = k % 8 == 0 || pw;
    if (m <= STREAM_TOKENS && whole && stream_x_bytes(m, (size_t)g.k) <= STREAM_X_BYTES)
        return launch_gemm16_stream(ctx, dtype, g);
    return launch_gemm16(ctx, dtype, g);
}

}  // extern "C"
