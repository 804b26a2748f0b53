// mx_gemm.cuh -- what the two product kernels (mx_gemm.cu, mx_gemm_pair.cu) share.
#pragma once

#include "mx.cuh"
#include "tcgen05.cuh"

namespace opure {

// silu(g) with the float exp of the reference's CPU path (Opure_CpuReference.cpp:195).
__device__ __forceinline__ float silu(float g) { return g * (1.0f / (1.0f + expf(-g))); }

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
bool mx_gemm_pair_suits(const opure_ctx *ctx, const opure_mx_gemm_args *a);
opure_status mx_gemm_pair(opure_ctx *ctx, const opure_mx_gemm_args *a, const uint8_t *w_scales);

}  // namespace opure
