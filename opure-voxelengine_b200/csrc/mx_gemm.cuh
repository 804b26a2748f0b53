// mx_gemm.cuh -- what the product kernels (mx_gemv.cu, mx_gemm.cu, mx_gemm_pair.cu) share.
#pragma once

#include "mx.cuh"
#include "tcgen05.cuh"

namespace opure {

// silu(g) with the float exp of the reference's CPU path (Opure_CpuReference.cpp:195).
__device__ __forceinline__ float silu(float g) { return g * (1.0f / (1.0f + expf(-g))); }

// silu(g) u with the hardware's exp2 and reciprocal, each within 2 units of fp32's last place
// (exp's argument times log2 e adds |g| 2^-24): far below a step of the 8-bit result, and a
// third of the instructions of expf and a rounded division (a prompt of 4096 x 16384 x 2048: 102
// us against 137).
__device__ __forceinline__ float swiglu(float g, float u) { return __fdividef(g, 1.0f + __expf(-g)) * u; }

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

// The product for one or two tokens, weights streamed through registers (a already validated; ws and us the
// scale tiles of w, or in SwiGLU of its gate and its up half).
bool mx_gemv_suits(const opure_mx_gemm_args *a);
opure_status mx_gemv(opure_ctx *ctx, const opure_mx_gemm_args *a, const uint8_t *ws, const uint8_t *us);

}  // namespace opure
