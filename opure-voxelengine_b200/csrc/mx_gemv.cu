// mx_gemv.cu -- the product of microscaled matrices for at most 8 tokens: decode's weight
// streaming.
//
// Bound by memory: a weight is 0.53 bytes and used once per token. At the measured 6.45 TB/s an SM
// gets 23 bytes, 43 weights, a clock, so that about 3 lane instructions per weight is all that its
// 128 lanes have. mma.sync m16n8k16 (fp16 in, fp32 out) takes the multiplications: 16 weight rows,
// up to 8 tokens, half a block of 32 columns. The codes' values are exact in fp16, and a block's
// sum is scaled by both scales in fp32. The tensor-core kernels' fixed costs (TMEM, tensor maps,
// a single issuing thread) are what this kernel avoids: there one token took 2 to 3 times as long.
//
// A warp reads 16 rows x 128 columns at once: lane 4 g + t holds block t (16 bytes) of rows g and
// g + 8. mma.sync wants a row's block spread over the four lanes t; which columns a lane holds
// does not matter as long as weights and tokens agree, so four words are exchanged among the four
// lanes and lane t takes columns 8 t .. 8 t + 7 of every block.
//
// A CTA is tiles x splits warps: `tiles` tiles of 16 rows (SwiGLU: 32 gate rows and the up rows that
// go with them), each shared by `splits` warps that take every splits'th 128 columns and are added
// in order through shared memory.
#include <algorithm>
#include <type_traits>

#include "mx_gemm.cuh"

namespace opure {
namespace {

constexpr uint32_t kMaxTokens = 8;
constexpr uint32_t kMaxWarps = 16;
constexpr uint32_t kAhead = 4;  // 128-column pieces that a warp has in flight

struct GemvParams {
    const uint8_t *w, *ws, *us, *x, *xs;
    uint32_t n, rows, cols, half, tiles, splits;
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
__device__ __forceinline__ void scale_pair(uint32_t bytes, float &s0, float &s1) {
    uint32_t b;
    asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;" : "=r"(b) : "h"(uint16_t(bytes)));
    s0 = __uint_as_float(b << 16);
    s1 = __uint_as_float(b & 0xffff0000u);
}

// Word j of lane t <-> word t of lane j, among four neighbouring lanes.
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
    const uint32_t t = threadIdx.x & 3u;
    {
        const bool up = t & 2u;
        const uint32_t r0 = __shfl_xor_sync(0xffffffffu, up ? w[0] : w[2], 2), r1 = __shfl_xor_sync(0xffffffffu, up ? w[1] : w[3], 2);
        if (up) {
            w[0] = r0;
            w[1] = r1;
        } else {
            w[2] = r0;
            w[3] = r1;
        }
    }
    {
        const bool up = t & 1u;
        const uint32_t r0 = __shfl_xor_sync(0xffffffffu, up ? w[0] : w[1], 1), r1 = __shfl_xor_sync(0xffffffffu, up ? w[2] : w[3], 1);
        if (up) {
            w[0] = r0;
            w[2] = r1;
        } else {
            w[1] = r0;
            w[3] = r1;
        }
    }
}

// What a warp reads of 128 columns.
template <uint32_t XF>
struct Piece {
    uint4 w[2];            // block t of rows g, g + 8
    uint32_t sw[2];        // four scales of each
    uint32_t x[4][XF / 4];  // columns 8 t .. of token g in each block
    uint32_t sx[2];        // four scales of tokens 2 t, 2 t + 1
};

// T: the type of y, or for SwiGLU uint8_t (E4M3) or uint32_t (E2M1).
template <uint32_t XF, int EPI, typename T>
__global__ void __launch_bounds__(kMaxWarps * 32) mx_gemv_kernel(GemvParams p) {
    constexpr bool kSwiglu = EPI == OPURE_EPI_SWIGLU;
    __shared__ float part[kMaxWarps][16][kMaxTokens];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, g = lane >> 2, t = lane & 3u;
    const uint32_t tile = warp / p.splits, split = warp % p.splits;
    const uint32_t pieces = mx_kp(p.cols) / 128;
    // This warp's rows. In SwiGLU tiles 0 and 1 are gate rows, 2 and 3 up rows, whose scale tiles
    // are counted from the first up row.
    const uint32_t c0 = blockIdx.x * (kSwiglu ? 32 : p.tiles * 16);  // first result column of the CTA
    const uint32_t local = c0 + (kSwiglu ? tile % 2 : tile) * 16 + g;
    const uint32_t limit = kSwiglu ? p.half : p.rows, first = kSwiglu && tile >= 2 ? p.half : 0;
    const uint8_t *scales = first ? p.us : p.ws;
    const uint8_t *w[2], *sw[2];
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) {
        const uint32_t r = min(local + 8 * j, limit - 1);  // rows past the end repeat the last one
        w[j] = p.w + size_t(first + r) * mx_row_bytes(OPURE_MX_FP4, p.cols) + t * 16;
        sw[j] = scales + mx_scale_offset(p.cols, r, 0);
    }
    // Weights may be asked for before the kernel that this one waits for has ended: into L2 only,
    // where a late write of theirs would show.
    if (t == 0)
#pragma unroll
        for (uint32_t i = 0; i < 2; ++i)
            if (split + i * p.splits < pieces)
#pragma unroll
                for (uint32_t j = 0; j < 2; ++j)
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(w[j] + size_t(split + i * p.splits) * 64));
    grid_dependency_wait();
    grid_dependents_launch();

    const uint8_t *x = p.x + size_t(min(g, p.n - 1)) * mx_row_bytes(XF, p.cols) + t * XF;
    const uint8_t *sx[2];
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j) sx[j] = p.xs + mx_scale_offset(p.cols, min(2 * t + j, p.n - 1), 0);
    float acc[4] = {};
    for (uint32_t k0 = split; k0 < pieces; k0 += kAhead * p.splits) {
        Piece<XF> in[kAhead];
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) {
            const uint32_t k = min(k0 + i * p.splits, pieces - 1);
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j) {
                in[i].w[j] = ldg_stream(w[j] + size_t(k) * 64);
                in[i].sw[j] = *reinterpret_cast<const uint32_t *>(sw[j] + size_t(k) * kMxTileBytes);
                in[i].sx[j] = *reinterpret_cast<const uint32_t *>(sx[j] + size_t(k) * kMxTileBytes);
            }
#pragma unroll
            for (uint32_t b = 0; b < 4; ++b) {
                const uint32_t *s = reinterpret_cast<const uint32_t *>(x + size_t(k) * (16 * XF) + b * (4 * XF));
#pragma unroll
                for (uint32_t j = 0; j < XF / 4; ++j) in[i].x[b][j] = s[j];
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < kAhead; ++i) {
            if (k0 + i * p.splits >= pieces) break;
            uint32_t lo[4] = {in[i].w[0].x, in[i].w[0].y, in[i].w[0].z, in[i].w[0].w};
            uint32_t hi[4] = {in[i].w[1].x, in[i].w[1].y, in[i].w[1].z, in[i].w[1].w};
            transpose4(lo);
            transpose4(hi);
            float fw[2][4], fx[2][4];
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j) {
                scale_pair(in[i].sw[j], fw[j][0], fw[j][1]);
                scale_pair(in[i].sw[j] >> 16, fw[j][2], fw[j][3]);
                scale_pair(in[i].sx[j], fx[j][0], fx[j][1]);
                scale_pair(in[i].sx[j] >> 16, fx[j][2], fx[j][3]);
            }
#pragma unroll
            for (uint32_t b = 0; b < 4; ++b) {
                uint32_t a0[4], a1[4], bx[4];
                mx_unpack_fp4(lo[b], a0);
                mx_unpack_fp4(hi[b], a1);
                if constexpr (XF == OPURE_MX_FP4) {
                    mx_unpack_fp4(in[i].x[b][0], bx);
                } else {
                    mx_unpack_fp8(in[i].x[b][0], bx[0], bx[1]);
                    mx_unpack_fp8(in[i].x[b][1], bx[2], bx[3]);
                }
                float d[4] = {};
                mma_f16(d, a0[0], a1[0], a0[1], a1[1], bx[0], bx[1]);
                mma_f16(d, a0[2], a1[2], a0[3], a1[3], bx[2], bx[3]);
#pragma unroll
                for (uint32_t j = 0; j < 4; ++j) acc[j] = fmaf(d[j] * fx[j & 1][b], fw[j >> 1][b], acc[j]);
            }
        }
    }
#pragma unroll
    for (uint32_t j = 0; j < 2; ++j)
        *reinterpret_cast<float2 *>(&part[warp][g + 8 * j][2 * t]) = make_float2(acc[2 * j], acc[2 * j + 1]);
    __syncthreads();

    // Results: a thread takes 4 neighbouring columns of a token.
    auto sum = [&](uint32_t column, uint32_t token) {
        float v = 0.f;
        for (uint32_t q = 0; q < p.splits; ++q) v += part[column / 16 * p.splits + q][column % 16][token];
        return v;
    };
    const uint32_t quads = kSwiglu ? 8 : p.tiles * 4;
    const uint32_t all = (quads * p.n + 31) / 32 * 32;  // whole warps
    for (uint32_t u = threadIdx.x; u < all; u += blockDim.x) {
        const uint32_t token = min(u / quads, p.n - 1), c = u % quads * 4, col = c0 + c;
        float v[4];
        if constexpr (kSwiglu) {
            constexpr uint32_t kF = sizeof(T) == 1 ? OPURE_MX_FP8 : OPURE_MX_FP4;
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) v[j] = col + j < p.half ? silu(sum(c + j, token)) * sum(32 + c + j, token) : 0.f;
            store_block<kF>(v, p.out + token * mx_row_bytes(kF, p.half) + size_t(c0) * kF / 8,
                            p.outs + mx_scale_offset(p.half, token, c0 / 32), u / quads < p.n);
        } else if (u / quads < p.n) {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) v[j] = sum(c + j, token);
            const size_t at = token * p.y_stride + col;
            store_quad<EPI>(v, static_cast<T *>(p.y) + at, static_cast<const T *>(p.residual) + at,
                            col < p.rows ? min(p.rows - col, 4u) : 0u, p.vec);
        }
    }
}

}  // namespace

bool mx_gemv_suits(const opure_mx_gemm_args *a) { return a->x.rows <= kMaxTokens; }

opure_status mx_gemv(opure_ctx *ctx, const opure_mx_gemm_args *a, const uint8_t *ws, const uint8_t *us) {
    const bool swiglu = a->epilogue == OPURE_EPI_SWIGLU, fp8 = a->x.format == OPURE_MX_FP8;
    GemvParams p{};
    p.w = a->w.codes;
    p.ws = ws;
    p.us = us;
    p.x = a->x.codes;
    p.xs = a->x.scales;
    p.n = a->x.rows;
    p.rows = a->w.rows;
    p.cols = a->w.cols;
    p.half = a->w.rows / 2;
    p.y = a->y;
    p.y_stride = a->y_stride;
    p.residual = a->residual;
    p.out = a->out.codes;
    p.outs = a->out.scales;
    p.vec = rows_aligned16(a->y, a->y_type, a->y_stride) && rows_aligned16(a->residual, a->y_type, a->y_stride);
    // About 16 warps per SM, each with 128 columns at least; CTAs of at least 4 warps.
    const uint32_t pieces = mx_kp(p.cols) / 128;
    const uint32_t row_tiles = swiglu ? mx_kp(p.half) / 32 * 4 : ceil_div(p.rows, 16);
    p.splits = 1;
    while (row_tiles * p.splits < uint32_t(ctx->sm_count) * 16 && p.splits * 2 <= pieces && p.splits * (swiglu ? 4 : 1) < kMaxWarps)
        p.splits *= 2;
    p.tiles = swiglu ? 4 : std::max(1u, 4 / p.splits);
    const dim3 grid(swiglu ? mx_kp(p.half) / 32 : ceil_div(row_tiles, p.tiles)), block(32 * p.tiles * p.splits);
    auto go = [&](auto t, auto epi) {
        using T = decltype(t);
        constexpr int kEpi = decltype(epi)::value;
        return fp8 ? launch(ctx, mx_gemv_kernel<OPURE_MX_FP8, kEpi, T>, grid, block, 0, true, p)
                   : launch(ctx, mx_gemv_kernel<OPURE_MX_FP4, kEpi, T>, grid, block, 0, true, p);
    };
    if (swiglu) {
        const std::integral_constant<int, OPURE_EPI_SWIGLU> epi;
        return a->out.format == OPURE_MX_FP4 ? go(uint32_t(), epi) : go(uint8_t(), epi);
    }
    return with_type(a->y_type, [&](auto t) {
        return a->epilogue == OPURE_EPI_ADD ? go(t, std::integral_constant<int, OPURE_EPI_ADD>())
                                            : go(t, std::integral_constant<int, OPURE_EPI_STORE>());
    });
}

}  // namespace opure
