// mx_gemv.cu -- the product of microscaled matrices for one or two tokens: decode's weight
// streaming.
//
// Its floor is memory: a weight is 0.53 bytes and used once per token. At the measured 6.45 TB/s an
// SM gets 23 bytes, 43 weights, a clock, so that about 3 lane instructions per weight is all that
// its 128 lanes have. mma.sync m16n8k16 (fp16 in, fp32 out) takes the multiplications; the codes'
// values are exact in fp16, and a block's sum is scaled by both scales in fp32. The tensor-core
// kernels' fixed costs (TMEM, tensor maps, a single issuing thread) are what this kernel avoids.
//
// A warp reads 16 weight rows x 128 columns as lane 4 g + t holding block t (16 bytes) of rows g
// and g + 8, and feeds that to the MMA as it stands: each MMA then sums over columns of all four
// blocks. The token side keeps the blocks apart. Its 8 columns are 2 tokens x 4 blocks, column
// 4 j + b having token j's values in the k slots of lanes t = b and zeros elsewhere, so that after
// the 8 MMAs of a piece D[row][4 j + b] is the sum over block b alone. Nothing is moved between
// lanes, and a piece is scaled once: 1.1 instructions per weight for 1 or 2 tokens. (With a block's
// 8 columns per MMA taken by 8 tokens, four words had to be exchanged among lanes and every block
// scaled by itself: 2.8 per weight.)
//
// A CTA is units x splits warps: a unit is 16 MT rows (in SwiGLU the CTA's units are 32 gate rows
// and the 32 up rows that go with them), shared by `splits` warps that take every splits'th 128
// columns and are added in order through shared memory.
//
// Measured: 1 x 49152 x 576 6.0 us (2.5 TB/s; its 15 MB are 2.4 us of memory), 1 x 2048 x 8192 4.6
// us, 1 x 576 x 576 2.0 us, SwiGLU of 1 x 16384 x 2048 7.4 us (2.8 for its bytes). At these sizes latency bounds it: launch, first loads, and one or two
// more rounds of loads by the 11 to 16 warps that fit an SM.
#include <algorithm>

#include "mx_gemm.cuh"

namespace opure {
namespace {

constexpr uint32_t kMaxTokens = 2;  // from 3 on mx_gemm.cu is as fast (4 x 2048 x 8192: 5.7 us both) or faster (4 x 49152 x 576: 12.5 and 8.6)
constexpr uint32_t kMaxWarps = 16;

struct GemvParams {
    const uint8_t *w, *ws, *x, *xs;
    uint32_t n, rows, cols, half, units, splits;
    uint32_t epilogue, y_type, out_format;
    void *y;
    size_t y_stride;
    const void *residual;
    uint8_t *out, *outs;
    bool vec;
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two scale bytes as fp32.
__device__ __forceinline__ void scale_pair(uint16_t bytes, float &s0, float &s1) {
    uint32_t b;
    asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;" : "=r"(b) : "h"(bytes));
    s0 = __uint_as_float(b << 16);
    s1 = __uint_as_float(b & 0xffff0000u);
}

// Weights of 16 MT rows x 128 columns: block t of rows g and g + 8 of each tile, and the scales of
// the two blocks whose sums this lane gets.
template <uint32_t MT>
struct Weights {
    uint4 w[2 * MT];
    uint16_t s[2 * MT];
};
// The tokens' 128 columns: this lane's block of its token (or zeros), and two blocks' scales.
template <uint32_t XF>
struct Tokens {
    uint4 x[XF / 4];
    uint16_t s;
};

// MT: tiles of 16 rows per warp.
template <uint32_t XF, uint32_t MT>
__global__ void __launch_bounds__(kMaxWarps * 32) mx_gemv_kernel(GemvParams p) {
    constexpr uint32_t kAhead = MT == 1 ? 4 : 3;  // pieces in flight
    constexpr uint32_t kRows = 16 * MT;
    __shared__ float part[kMaxWarps][kRows][kMaxTokens + 1];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t unit = warp / p.splits, split = warp % p.splits;
    const uint32_t pieces = mx_kp(p.cols) / 128;
    const bool swiglu = p.epilogue == OPURE_EPI_SWIGLU;
    // This warp's rows. In SwiGLU (two tiles a warp) unit 0 is 32 gate rows and unit 1 the up rows
    // that go with them.
    const uint32_t c0 = blockIdx.x * (swiglu ? 32 : p.units * kRows);  // first result column of the CTA
    const uint32_t local = c0 + (swiglu ? 0 : unit * kRows) + g;
    const uint32_t limit = swiglu ? p.half : p.rows, first = swiglu && unit ? p.half : 0;
    const size_t row_bytes = mx_row_bytes(OPURE_MX_FP4, p.cols);
    const uint8_t *w[2 * MT], *ws[2 * MT];
#pragma unroll
    for (uint32_t j = 0; j < 2 * MT; ++j) {
        const uint32_t r = min(local + 8 * j, limit - 1);  // rows past the end repeat the last one
        w[j] = p.w + (first + r) * row_bytes + t * 16;
        ws[j] = p.ws + mx_scale_offset(p.cols, first + r, 0) + t % 2 * 2;
    }
    // The weights may be asked for before the kernel that this one waits for has ended, into L2
    // only, where a late write of its would show.
    if (t == 0 && split < pieces)
#pragma unroll
        for (uint32_t j = 0; j < 2 * MT; ++j) asm volatile("prefetch.global.L2 [%0];" ::"l"(w[j] + size_t(split) * 64));
    grid_dependency_wait();
    grid_dependents_launch();

    // Column g of the MMA is block g % 4 of token g / 4: the lanes t = g % 4 hold it. D's columns
    // 2 t and 2 t + 1 are blocks 2 t % 4 and the next of token t / 2.
    const bool holds = t == g % 4 && g / 4 < p.n;
    const uint8_t *x = p.x + g / 4 * mx_row_bytes(XF, p.cols) + t * (4 * XF);
    const uint8_t *xs = p.xs + mx_scale_offset(p.cols, min(t / 2, p.n - 1), 0) + t % 2 * 2;
    auto load = [&](Weights<MT> &in, Tokens<XF> &tk, uint32_t k) {
#pragma unroll
        for (uint32_t j = 0; j < 2 * MT; ++j) {
            in.w[j] = ldg_stream(w[j] + size_t(k) * 64);
            in.s[j] = *reinterpret_cast<const uint16_t *>(ws[j] + size_t(k) * kMxTileBytes);
        }
#pragma unroll
        for (uint32_t j = 0; j < XF / 4; ++j) {
            tk.x[j] = make_uint4(0, 0, 0, 0);
            if (holds) tk.x[j] = *reinterpret_cast<const uint4 *>(x + size_t(k) * (16 * XF) + j * 16);
        }
        tk.s = *reinterpret_cast<const uint16_t *>(xs + size_t(k) * kMxTileBytes);
    };
    float sum_of[2 * MT] = {};
    auto compute = [&](const Weights<MT> &wt, const Tokens<XF> &tk) {
        // The tokens' 32 values per lane as fp16 pairs, in the order of the weights' codes.
        uint32_t b[16];
        const uint32_t *c = reinterpret_cast<const uint32_t *>(tk.x);
#pragma unroll
        for (uint32_t q = 0; q < 4; ++q) {
            uint32_t h[4];
            if constexpr (XF == OPURE_MX_FP4) {
                mx_unpack_fp4(c[q], h);
            } else {
                mx_unpack_fp8(c[2 * q], h[0], h[1]);
                mx_unpack_fp8(c[2 * q + 1], h[2], h[3]);
            }
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) b[4 * q + j] = h[j];
        }
        float x0, x1;
        scale_pair(tk.s, x0, x1);
#pragma unroll
        for (uint32_t m = 0; m < MT; ++m) {
            float d[4] = {};
            const uint32_t lo[4] = {wt.w[2 * m].x, wt.w[2 * m].y, wt.w[2 * m].z, wt.w[2 * m].w};
            const uint32_t hi[4] = {wt.w[2 * m + 1].x, wt.w[2 * m + 1].y, wt.w[2 * m + 1].z, wt.w[2 * m + 1].w};
#pragma unroll
            for (uint32_t q = 0; q < 4; ++q) {
                uint32_t a0[4], a1[4];
                mx_unpack_fp4(lo[q], a0);
                mx_unpack_fp4(hi[q], a1);
                mma_f16(d, a0[0], a1[0], a0[1], a1[1], b[4 * q], b[4 * q + 1]);
                mma_f16(d, a0[2], a1[2], a0[3], a1[3], b[4 * q + 2], b[4 * q + 3]);
            }
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j) {
                float s0, s1;
                scale_pair(wt.s[2 * m + j], s0, s1);
                // The scales first: d times one of them can pass fp32 where the other would bring it back.
                sum_of[2 * m + j] = fmaf(d[2 * j], x0 * s0, fmaf(d[2 * j + 1], x1 * s1, sum_of[2 * m + j]));
            }
        }
    };
    Weights<MT> in[kAhead];
    Tokens<XF> tk[kAhead];
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i)
        if (split + i * p.splits < pieces) load(in[i], tk[i], split + i * p.splits);
    for (uint32_t k0 = split; k0 < pieces; k0 += kAhead * p.splits) {
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) {
            const uint32_t k = k0 + i * p.splits, next = k + kAhead * p.splits;
            if (k >= pieces) break;
            compute(in[i], tk[i]);
            if (next < pieces) load(in[i], tk[i], next);
        }
    }
    // Lanes t and t ^ 1 hold two blocks each of one token.
#pragma unroll
    for (uint32_t j = 0; j < 2 * MT; ++j) {
        const float v = sum_of[j] + __shfl_xor_sync(0xffffffffu, sum_of[j], 1);
        if (t % 2 == 0) part[warp][g + 8 * j][t / 2] = v;
    }
    __syncthreads();

    // Results: a thread takes 4 neighbouring columns of a token.
    auto sum = [&](uint32_t column, uint32_t token) {
        float v = 0.f;
        for (uint32_t q = 0; q < p.splits; ++q) v += part[column / kRows * p.splits + q][column % kRows][token];
        return v;
    };
    const uint32_t quads = (swiglu ? 32 : p.units * kRows) / 4;
    const uint32_t all = (quads * p.n + 31) / 32 * 32;  // whole warps
    for (uint32_t u = threadIdx.x; u < all; u += blockDim.x) {
        const bool real = u / quads < p.n;
        const uint32_t token = min(u / quads, p.n - 1), c = u % quads * 4, col = c0 + c;
        float v[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) v[j] = sum(c + j, token);
        if (swiglu) {
#pragma unroll
            for (uint32_t j = 0; j < 4; j += 2) swiglu2(v[j], v[j + 1], sum(32 + c + j, token), sum(33 + c + j, token));
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
                if (col + j >= p.half) v[j] = 0.f;  // gate rows past the half repeat the last one
            uint8_t *scale = p.outs + mx_scale_offset(p.half, token, c0 / 32);
            if (p.out_format == OPURE_MX_FP4)
                store_block<OPURE_MX_FP4>(v, p.out + token * mx_row_bytes(OPURE_MX_FP4, p.half) + size_t(c0) / 2, scale, real);
            else
                store_block<OPURE_MX_FP8>(v, p.out + token * mx_row_bytes(OPURE_MX_FP8, p.half) + c0, scale, real);
        } else if (real) {
            const size_t at = token * p.y_stride + col;
            const uint32_t left = columns_left(p.rows, col);
            auto store = [&](auto type) {
                using T = decltype(type);
                T *y = static_cast<T *>(p.y) + at;
                const T *res = static_cast<const T *>(p.residual) + at;
                // One or two tokens: unaligned values one at a time cost nothing that shows.
                for (uint32_t j = 0; j < 4; j += p.vec ? 4 : 1) {
                    if (j >= left) break;
                    if (p.vec) {
                        p.epilogue == OPURE_EPI_ADD ? store_quad<OPURE_EPI_ADD>(v, y, res, left) : store_quad<OPURE_EPI_STORE>(v, y, res, left);
                    } else {
                        y[j] = from_f32<T>(p.epilogue == OPURE_EPI_ADD ? v[j] + to_f32(res[j]) : v[j]);
                    }
                }
            };
            if (p.y_type == OPURE_F32)
                store(float());
            else if (p.y_type == OPURE_F16)
                store(__half());
            else
                store(__nv_bfloat16());
        }
    }
}

// Units and splits per CTA: the least estimated time. 16 warps of this kernel's registers fit an
// SM. A wave of CTAs costs its fixed part (about 500 cycles) and a memory latency (700) for every
// round of pieces in flight; an SM takes about 120 cycles for a piece of two tiles and 75 for one.
void choose(GemvParams &p, uint32_t pieces, uint32_t units_all, uint32_t cta_units, bool two, uint32_t sms) {
    uint64_t best = ~uint64_t(0);
    for (uint32_t u = cta_units ? cta_units : 1; u <= (cta_units ? cta_units : kMaxWarps); ++u)
        for (uint32_t s = 1; u * s <= kMaxWarps && s <= pieces; ++s) {
            if (u * s < 4 && s < pieces && !cta_units) continue;  // CTAs of 4 warps at least
            const uint64_t ctas = ceil_div(units_all, u), resident = uint64_t(sms) * (kMaxWarps / (u * s));
            const uint64_t waves = (ctas + resident - 1) / resident;
            const uint64_t rounds = ceil_div(ceil_div(pieces, s), two ? 3 : 4);
            const uint64_t cost = waves * (500 + 700 * rounds) + (ctas + sms - 1) / sms * u * pieces * (two ? 120 : 75);
            if (cost < best) {
                best = cost;
                p.units = u;
                p.splits = s;
            }
        }
}

}  // namespace

bool mx_gemv_suits(const opure_mx_gemm_args *a) { return a->x.rows <= kMaxTokens; }

opure_status mx_gemv(opure_ctx *ctx, const opure_mx_gemm_args *a) {
    const bool swiglu = a->epilogue == OPURE_EPI_SWIGLU, fp8 = a->x.format == OPURE_MX_FP8;
    GemvParams p{};
    p.w = a->w.codes;
    p.ws = a->w.scales;
    p.x = a->x.codes;
    p.xs = a->x.scales;
    p.n = a->x.rows;
    p.rows = a->w.rows;
    p.cols = a->w.cols;
    p.half = a->w.rows / 2;
    p.epilogue = a->epilogue;
    p.y_type = a->y_type;
    p.out_format = a->out.format;
    p.y = a->y;
    p.y_stride = a->y_stride;
    p.residual = a->residual;
    p.out = a->out.codes;
    p.outs = a->out.scales;
    p.vec = rows_aligned16(a->y, a->y_type, a->y_stride) && rows_aligned16(a->residual, a->y_type, a->y_stride);
    const uint32_t pieces = mx_kp(p.cols) / 128, sms = uint32_t(ctx->sm_count);
    const uint32_t row_tiles = swiglu ? mx_kp(p.half) / 32 * 4 : ceil_div(p.rows, 16);
    // Two tiles per warp halve the work on the tokens' side; one where that would leave SMs empty.
    const bool two = swiglu || row_tiles >= 2 * sms;
    const uint32_t units_all = two ? (row_tiles + 1) / 2 : row_tiles;
    choose(p, pieces, units_all, swiglu ? 2 : 0, two, sms);
    const dim3 grid(ceil_div(units_all, p.units)), block(32 * p.units * p.splits);
    auto go = [&](auto kernel) { return launch(ctx, kernel, grid, block, 0, true, p); };
    if (two) return fp8 ? go(mx_gemv_kernel<OPURE_MX_FP8, 2>) : go(mx_gemv_kernel<OPURE_MX_FP4, 2>);
    return fp8 ? go(mx_gemv_kernel<OPURE_MX_FP8, 1>) : go(mx_gemv_kernel<OPURE_MX_FP4, 1>);
}

}  // namespace opure
