// mx_gemm.cu -- the product of microscaled (MX) matrices: y[i][r] = sum_k x[i][k] w[r][k], with
// the linear layer's epilogues (store, residual add, SwiGLU with an MX result).
//
// With block b's scales sx and sw and its codes' values cx and cw,
//   y[i][r] = sum_b sx[i][b] sw[r][b] (sum_{k in b} cx[i][k] cw[r][k]).
// The products of codes are exact in fp16; sums are fp32.
#include <algorithm>
#include <type_traits>

#include "mx.cuh"

namespace opure {
namespace {

struct GemmParams {
    const uint8_t *w, *ws, *x, *xs;
    uint32_t n, rows, cols, x_format;
    void *y;
    size_t y_stride;
    const void *residual;
    uint8_t *out, *outs;  // OPURE_EPI_SWIGLU
};

// Dot product of token i and weight row r; every lane of the warp gets it. A lane takes every
// 32nd block.
__device__ __forceinline__ float dot(const GemmParams &p, uint32_t i, uint32_t r) {
    const uint32_t lane = threadIdx.x & 31u, blocks = (p.cols + kMxBlock - 1) / kMxBlock;
    float acc = 0.f;
    for (uint32_t b = lane; b < blocks; b += 32) {
        const uint4 w = *reinterpret_cast<const uint4 *>(p.w + r * mx_row_bytes(OPURE_MX_FP4, p.cols) + b * 16);
        const uint32_t wv[4] = {w.x, w.y, w.z, w.w};
        uint32_t xv[8];
        const uint8_t *xr = p.x + i * mx_row_bytes(p.x_format, p.cols) + b * (4 * p.x_format);
        for (uint32_t j = 0; j < p.x_format; ++j) xv[j] = reinterpret_cast<const uint32_t *>(xr)[j];
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            uint32_t hw[4], hx[4];
            mx_unpack_fp4(wv[j], hw);
            if (p.x_format == OPURE_MX_FP4) {
                mx_unpack_fp4(xv[j], hx);
            } else {
                mx_unpack_fp8(xv[2 * j], hx[0], hx[1]);
                mx_unpack_fp8(xv[2 * j + 1], hx[2], hx[3]);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float2 a = h2f2(hw[q]), c = h2f2(hx[q]);
                t = fmaf(a.x, c.x, t);
                t = fmaf(a.y, c.y, t);
            }
        }
        acc = fmaf(t * mx_scale_value(p.xs[mx_scale_offset(p.cols, i, b)]),
                   mx_scale_value(p.ws[mx_scale_offset(p.cols, r, b)]), acc);
    }
    return warp_sum(acc);
}

// One warp per (token, 32 result columns): lane j keeps column j.
template <int EPI, typename T>
__global__ void __launch_bounds__(256) mx_gemm_kernel(GemmParams p) {
    grid_dependency_wait();
    grid_dependents_launch();
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t out_rows = EPI == OPURE_EPI_SWIGLU ? p.rows / 2 : p.rows;
    const uint32_t units = EPI == OPURE_EPI_SWIGLU ? mx_kp(out_rows) / 32 : (out_rows + 31) / 32;
    const uint64_t unit = (uint64_t(blockIdx.x) * blockDim.x + threadIdx.x) / 32;
    const uint64_t i64 = unit / units;
    if (i64 >= p.n) return;
    const uint32_t i = uint32_t(i64), r0 = uint32_t(unit - i64 * units) * 32;
    float v = 0.f;
    for (uint32_t j = 0; j < 32 && r0 + j < out_rows; ++j) {
        float d = dot(p, i, r0 + j);
        if constexpr (EPI == OPURE_EPI_SWIGLU) {
            const float up = dot(p, i, out_rows + r0 + j);
            d = d * (1.0f / (1.0f + expf(-d))) * up;
        }
        if (lane == j) v = d;
    }
    if constexpr (EPI == OPURE_EPI_SWIGLU) {
        uint32_t m = __float_as_uint(v) & 0x7fffffffu;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        const bool fp4 = std::is_same_v<T, uint32_t>;
        const uint32_t byte = fp4 ? mx_scale_byte<OPURE_MX_FP4>(m) : mx_scale_byte<OPURE_MX_FP8>(m);
        v = byte == 255u ? 0.f : v * mx_inverse(byte);
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __shfl_sync(0xffffffffu, v, (lane % 4) * 8 + j);
        uint8_t *row = p.out + i * mx_row_bytes(fp4 ? OPURE_MX_FP4 : OPURE_MX_FP8, out_rows);
        if (lane < 4) {
            if (fp4)
                reinterpret_cast<uint32_t *>(row)[r0 / 8 + lane] = mx_pack_fp4(f);
            else
                reinterpret_cast<uint2 *>(row)[r0 / 8 + lane] =
                    make_uint2(mx_pack_fp8(f[0], f[1], f[2], f[3]), mx_pack_fp8(f[4], f[5], f[6], f[7]));
        }
        if (lane == 0) p.outs[mx_scale_offset(out_rows, i, r0 / kMxBlock)] = uint8_t(byte);
    } else if (r0 + lane < out_rows) {
        const size_t o = i * p.y_stride + r0 + lane;
        if constexpr (EPI == OPURE_EPI_ADD) v += to_f32(static_cast<const T *>(p.residual)[o]);
        static_cast<T *>(p.y)[o] = from_f32<T>(v);
    }
}

}  // namespace
}  // namespace opure

using namespace opure;

extern "C" {

opure_status opure_mx_gemm(opure_ctx *ctx, const opure_mx_gemm_args *a) {
    opure_status s = enter(ctx);
    if (s) return s;
    if (!a || !mx_valid(a->w) || !mx_valid(a->x) || a->w.cols != a->x.cols) return OPURE_ERR_INVALID_ARG;
    if (a->w.format != OPURE_MX_FP4) return OPURE_ERR_UNSUPPORTED;
    const bool swiglu = a->epilogue == OPURE_EPI_SWIGLU;
    if (swiglu) {
        if (a->w.rows % 2 || !mx_valid(a->out) || a->out.rows != a->x.rows || a->out.cols != a->w.rows / 2)
            return OPURE_ERR_INVALID_ARG;
    } else if (a->epilogue == OPURE_EPI_STORE || a->epilogue == OPURE_EPI_ADD) {
        if (!type_aligned(a->y, a->y_type) || a->y_stride < a->w.rows) return OPURE_ERR_INVALID_ARG;
        if (a->epilogue == OPURE_EPI_ADD && !type_aligned(a->residual, a->y_type)) return OPURE_ERR_INVALID_ARG;
    } else {
        return a->epilogue == OPURE_EPI_ARGMAX ? OPURE_ERR_UNSUPPORTED : OPURE_ERR_INVALID_ARG;
    }
    if (a->x.rows == 0 || a->w.rows == 0) return OPURE_OK;
    if (!swiglu && (!a->y || (a->epilogue == OPURE_EPI_ADD && !a->residual))) return OPURE_ERR_INVALID_ARG;
    GemmParams p{a->w.codes, a->w.scales, a->x.codes, a->x.scales, a->x.rows, a->w.rows, a->w.cols, a->x.format,
                 a->y, a->y_stride, a->residual, a->out.codes, a->out.scales};
    const uint64_t units = uint64_t(a->x.rows) * (swiglu ? mx_kp(a->w.rows / 2) / 32 : ceil_div(a->w.rows, 32));
    if ((units + 7) / 8 > 0x7fffffffu) return OPURE_ERR_UNSUPPORTED;
    auto go = [&](auto kernel) { return launch(ctx, kernel, dim3(ceil_div(units, 8)), dim3(256), 0, true, p); };
    if (swiglu)
        return a->out.format == OPURE_MX_FP4 ? go(mx_gemm_kernel<OPURE_EPI_SWIGLU, uint32_t>)
                                             : go(mx_gemm_kernel<OPURE_EPI_SWIGLU, uint8_t>);
    return with_type(a->y_type, [&](auto t) {
        using T = decltype(t);
        return a->epilogue == OPURE_EPI_ADD ? go(mx_gemm_kernel<OPURE_EPI_ADD, T>) : go(mx_gemm_kernel<OPURE_EPI_STORE, T>);
    });
}

}  // extern "C"
