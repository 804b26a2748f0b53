// mx_gemm.cuh -- what the product kernels (mx_gemv.cu, mx_gemm.cu, mx_gemm_pair.cu) share.
#pragma once

#include "mx.cuh"
#include "tcgen05.cuh"

namespace opure {

// Two floats in a register pair, for the instructions that work on both.
__device__ __forceinline__ uint64_t pair2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair2(uint64_t v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// g0, g1 <- silu(g0) u0, silu(g1) u1, silu(g) = g / (1 + exp(-g)), from t = exp(-|g|), which does not
// overflow: g t / (1 + t) for negative g. Within a few units of fp32's last place down to g = -88, and
// to 2^-16 below, as far as silu(g) is a normal number (-92). The same for any number of tokens. Without
// branches, so that a thread's results overlap, and two at a time: with expf and a division 4096 x 4096 x
// 576 in 4 bits took 27 us instead of 17. (exp2 of the rounded product and an approximate division are
// 1 to 5% faster still, 16 us there, but give 0 for g below -87 and lose a bit for every doubling of |g|.)
__device__ __forceinline__ void swiglu2(float &g0, float &g1, float u0, float u1) {
    constexpr float kLog2e = 1.44269502f, kLog2eRest = 1.92596299e-8f, kLn2 = 0.693147181f;
    // t = 2^-32 2^(p + q), p + q = 32 - |g| log2(e) to twice fp32's length, 2^q = 1 + q ln 2 for a q that
    // is a rounding error of p. The 32 keeps 2^p normal where t is not; from |g| = 110 on, where t is 0,
    // it no longer does, and 2^p is 0. (A NaN stays in g.)
    const uint64_t a = pair2(fminf(fabsf(g0), 110.f), fminf(fabsf(g1), 110.f));
    const uint64_t l = pair2(-kLog2e, -kLog2e), p = fma2(a, l, pair2(32.f, 32.f));
    const uint64_t q = fma2(a, pair2(-kLog2eRest, -kLog2eRest), fma2(a, l, fma2(p, pair2(-1.f, -1.f), pair2(32.f, 32.f))));
    float p0, p1, e0, e1, t0, t1, d0, d1, r0, r1;
    unpair2(p, p0, p1);
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e0) : "f"(p0));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e1) : "f"(p1));
    constexpr float kLow = 0x1p-32f;
    const uint64_t t = mul2(pair2(e0, e1), fma2(q, pair2(kLn2 * kLow, kLn2 * kLow), pair2(kLow, kLow)));
    unpair2(t, t0, t1);
    const uint64_t d = fma2(t, pair2(-1.f, -1.f), pair2(-1.f, -1.f));  // -(1 + t)
    unpair2(d, d0, d1);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r0) : "f"(-d0));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r1) : "f"(-d1));
    // n / (1 + t) = n r (1 + e) for the residue e = 1 - (1 + t) r of the hardware's reciprocal.
    const uint64_t r = pair2(r0, r1), e = fma2(d, r, pair2(1.f, 1.f));
    const uint64_t w = mul2(mul2(pair2(g0, g1), pair2(g0 < 0.f ? t0 : 1.f, g1 < 0.f ? t1 : 1.f)), r);
    unpair2(mul2(fma2(w, e, w), pair2(u0, u1)), g0, g1);
}

// Quantises a block held as 4 values in each of 8 neighbouring lanes; `codes` is the block's
// place in its row. All lanes of the warp call it; only those with `in` store.
template <uint32_t FMT>
__device__ __forceinline__ void store_block(const float (&v)[4], uint8_t *codes, uint8_t *scale, bool in) {
    const uint32_t lane = threadIdx.x & 7u;
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    const uint32_t byte = mx_scale_byte<FMT>(m), keep = byte == 255u ? 0u : ~0u;
    const float inv = mx_inverse(byte);
    if (!in) return;
    if constexpr (FMT == OPURE_MX_FP4) {
        const float f[8] = {v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv};
        reinterpret_cast<uint16_t *>(codes)[lane] = uint16_t(mx_pack_fp4(f) & keep);
    } else {
        reinterpret_cast<uint32_t *>(codes)[lane] = mx_pack_fp8(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv) & keep;
    }
    if (lane == 0) *scale = uint8_t(byte);
}

// Stores (EPI: adds the residual to) the first `left` of 4 neighbouring results; all four at once
// where there are as many (y and res aligned for that).
template <int EPI, typename T>
__device__ __forceinline__ void store_quad(float (&v)[4], T *y, const T *res, uint32_t left) {
    if (left >= 4) {
        struct alignas(4 * sizeof(T)) Quad {
            T v[4];
        } o;
        if constexpr (EPI == OPURE_EPI_ADD) {
            const Quad q = *reinterpret_cast<const Quad *>(res);
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) v[j] += to_f32(q.v[j]);
        }
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) o.v[j] = from_f32<T>(v[j]);
        *reinterpret_cast<Quad *>(y) = o;
    } else {
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            if (j >= left) break;
            if constexpr (EPI == OPURE_EPI_ADD) v[j] += to_f32(res[j]);
            y[j] = from_f32<T>(v[j]);
        }
    }
}

// A tensor map without gaps between elements: dims and box innermost first, strides (bytes) of
// all dimensions but the first.
bool make_map(CUtensorMap *m, CUtensorMapDataType type, uint32_t rank, const void *p, const uint64_t *dims, const uint64_t *strides,
              const uint32_t *box, CUtensorMapSwizzle swizzle);
// A row-major matrix.
inline bool make_map(CUtensorMap *m, CUtensorMapDataType type, const void *p, uint64_t cols, uint64_t rows, uint64_t row_bytes,
                     uint32_t box_cols, uint32_t box_rows, CUtensorMapSwizzle swizzle) {
    const uint64_t dims[2] = {cols, rows}, strides[1] = {row_bytes};
    const uint32_t box[2] = {box_cols, box_rows};
    return make_map(m, type, 2, p, dims, strides, box, swizzle);
}

// Codes as byte slots in shared memory: boxes of 128 columns x box_rows rows in 128-byte
// swizzled rows. E2M1 is spread by the copy: 16 codes (8 bytes) to 16 bytes.
inline bool make_slot_map(CUtensorMap *m, const opure_mx_matrix &a, uint32_t box_rows) {
    return make_map(m, a.format == OPURE_MX_FP4 ? CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B : CU_TENSOR_MAP_DATA_TYPE_UINT8, a.codes,
                    mx_kp(a.cols), a.rows, mx_row_bytes(a.format, a.cols), 128, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

// The product over pairs of SMs, for many tokens (a already validated; w_scales the scale tiles
// of w, in SwiGLU those of its gate half followed by those of its up half).
uint64_t mx_gemm_pair_ns(const opure_ctx *ctx, const opure_mx_gemm_args *a);  // estimated time
opure_status mx_gemm_pair(opure_ctx *ctx, const opure_mx_gemm_args *a, const uint8_t *w_scales);

// The product for one or two tokens, weights streamed through registers (a already validated).
bool mx_gemv_suits(const opure_mx_gemm_args *a);
opure_status mx_gemv(opure_ctx *ctx, const opure_mx_gemm_args *a);

}  // namespace opure
