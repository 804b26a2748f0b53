// mx.cuh -- microscaled (MX) matrices: layout, code conversions and typed row access shared by
// mx.cu (quantise, dequantise, norm) and mx_gemm.cu (product). Layout: opure_mx_matrix in
// opure_cuda.h.
#pragma once

#include <cuda_bf16.h>

#include "ctx.cuh"

namespace opure {

constexpr uint32_t kMxBlock = 32;      // values per scale
constexpr uint32_t kMxTileBytes = 512;  // scales of 128 rows x 128 columns

__host__ __device__ __forceinline__ uint32_t mx_kp(uint32_t cols) { return (cols + 127u) & ~127u; }
__host__ __device__ __forceinline__ size_t mx_row_bytes(uint32_t format, uint32_t cols) {
    return size_t(mx_kp(cols)) * format / 8;
}
// Byte offset of the scale of (row, block of 32 columns).
__host__ __device__ __forceinline__ size_t mx_scale_offset(uint32_t cols, uint32_t row, uint32_t block) {
    return (size_t(row / 128) * (mx_kp(cols) / 128) + block / 4) * kMxTileBytes + row % 32 * 16 + row / 32 % 4 * 4 +
           block % 4;
}
// The row of a warp in a grid with a warp per row: no larger than the rows are, where the index of
// the thread would pass 32 bits from 2^27 rows on.
__host__ __device__ __forceinline__ uint32_t mx_warp_row(uint32_t block, uint32_t thread, uint32_t threads) {
    return block * (threads / 32) + thread / 32;
}

__device__ __forceinline__ uint32_t columns_left(uint32_t cols, uint32_t first) { return first < cols ? cols - first : 0u; }

// The scale byte of a block from the largest magnitude's bits. Magnitudes compare as
// integers, so a NaN or infinity in the block is the largest and gives 255.
template <uint32_t FMT>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax_bits) {
    constexpr int kEmax = FMT == OPURE_MX_FP4 ? 2 : 8;
    if (amax_bits >= 0x7f800000u) return 255u;
    return uint32_t(max(int(amax_bits >> 23) - kEmax, 0));
}
// 2^(127 - byte): what a block's values are multiplied by. Exact for bytes up to 253 (those of finite
// blocks are at most 252); 0 for 255, whose codes are 0.
__device__ __forceinline__ float mx_inverse(uint32_t byte) {
    return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
}
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
    return byte == 0u ? __uint_as_float(0x00400000u) : byte == 255u ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
}

// 8 floats -> 8 E2M1 codes (4 bytes, the first value in the lowest half-byte).
__device__ __forceinline__ uint32_t mx_pack_fp4(const float (&v)[8]) {
    uint32_t r;
    asm("{\n .reg .b8 a, b, c, d;\n"
        " cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n"
        " cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n"
        " mov.b32 %0, {a, b, c, d};\n}"
        : "=r"(r)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return r;
}
// 4 floats -> 4 E4M3 codes.
__device__ __forceinline__ uint32_t mx_pack_fp8(float v0, float v1, float v2, float v3) {
    uint32_t r;
    asm("{\n .reg .b16 a, b;\n cvt.rn.satfinite.e4m3x2.f32 a, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 b, %4, %3;\n"
        " mov.b32 %0, {a, b};\n}"
        : "=r"(r)
        : "f"(v0), "f"(v1), "f"(v2), "f"(v3));
    return r;
}
// 8 E2M1 codes -> 4 fp16 pairs (exact).
__device__ __forceinline__ void mx_unpack_fp4(uint32_t w, uint32_t (&h)[4]) {
    asm("{\n .reg .b8 a, b, c, d;\n mov.b32 {a, b, c, d}, %4;\n"
        " cvt.rn.f16x2.e2m1x2 %0, a;\n cvt.rn.f16x2.e2m1x2 %1, b;\n"
        " cvt.rn.f16x2.e2m1x2 %2, c;\n cvt.rn.f16x2.e2m1x2 %3, d;\n}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
}
// 4 E4M3 codes -> 2 fp16 pairs (exact).
__device__ __forceinline__ void mx_unpack_fp8(uint32_t w, uint32_t &h0, uint32_t &h1) {
    asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.rn.f16x2.e4m3x2 %0, a;\n cvt.rn.f16x2.e4m3x2 %1, b;\n}"
        : "=r"(h0), "=r"(h1)
        : "r"(w));
}

// ---- values of an opure_type ---------------------------------------------------------
template <typename T>
__device__ __forceinline__ float to_f32(T v) {
    if constexpr (sizeof(T) == 4)
        return v;
    else if constexpr (std::is_same_v<T, __half>)
        return __half2float(v);
    else
        return __bfloat162float(v);
}
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    if constexpr (sizeof(T) == 4)
        return v;
    else if constexpr (std::is_same_v<T, __half>)
        return __float2half_rn(v);
    else
        return __float2bfloat16_rn(v);
}
// 8 neighbouring values in 16-byte loads (p 16-byte aligned).
template <typename T>
__device__ __forceinline__ void load8(const T *p, float (&f)[8]) {
    if constexpr (sizeof(T) == 4) {
        const float4 a = reinterpret_cast<const float4 *>(p)[0], b = reinterpret_cast<const float4 *>(p)[1];
        f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w;
        f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
        const uint4 u = *reinterpret_cast<const uint4 *>(p);
        const T *h = reinterpret_cast<const T *>(&u);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = to_f32(h[j]);
    }
}
template <typename T>
__device__ __forceinline__ void store8(T *p, const float (&f)[8]) {
    if constexpr (sizeof(T) == 4) {
        reinterpret_cast<float4 *>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4 *>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
        uint4 u;
        T *h = reinterpret_cast<T *>(&u);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = from_f32<T>(f[j]);
        *reinterpret_cast<uint4 *>(p) = u;
    }
}
// 16 neighbouring values in 32-byte loads and stores (p 32-byte aligned).
__device__ __forceinline__ void ldg256(const void *p, uint32_t (&r)[8]) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "l"(p)
                 : "memory");
}
__device__ __forceinline__ void stg256(void *p, const uint32_t (&r)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
template <typename T>
__device__ __forceinline__ void load16(const T *p, uint32_t (&raw)[4 * sizeof(T)]) {
#pragma unroll
    for (uint32_t j = 0; j < sizeof(T) / 2; ++j) ldg256(reinterpret_cast<const uint8_t *>(p) + 32 * j, *reinterpret_cast<uint32_t(*)[8]>(raw + 8 * j));
}
// The first `n` of 8 neighbouring values, zeros after them; any alignment.
template <typename T>
__device__ __forceinline__ void load8_part(const T *p, uint32_t n, float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = uint32_t(j) < n ? to_f32(p[j]) : 0.f;
}
template <typename T>
__device__ __forceinline__ void store8_part(T *p, uint32_t n, const float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (uint32_t(j) < n) p[j] = from_f32<T>(f[j]);
}

// The largest of three magnitudes; NaN if one is.
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// Quantises a block held as 8 values in each of 4 neighbouring lanes and stores this lane's
// codes at `codes` (the row's base), columns 8 oct .. 8 oct + 7. Returns the scale byte. All
// lanes of the warp call it; only those with `in` store.
template <uint32_t FMT>
__device__ __forceinline__ uint32_t mx_store_octet(float (&v)[8], uint8_t *codes, uint32_t oct, bool in) {
    const float f = max_abs3(max_abs3(v[0], v[1], v[2]), max_abs3(v[3], v[4], v[5]), max_abs3(v[6], v[7], 0.f));
    uint32_t m = __float_as_uint(f) & 0x7fffffffu;
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
    m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
    const uint32_t byte = mx_scale_byte<FMT>(m), keep = byte == 255u ? 0u : ~0u;
    const float inv = mx_inverse(byte);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= inv;
    if constexpr (FMT == OPURE_MX_FP4) {
        const uint32_t c = mx_pack_fp4(v) & keep;
        if (in) reinterpret_cast<uint32_t *>(codes)[oct] = c;
    } else {
        const uint2 c = make_uint2(mx_pack_fp8(v[0], v[1], v[2], v[3]) & keep, mx_pack_fp8(v[4], v[5], v[6], v[7]) & keep);
        if (in) reinterpret_cast<uint2 *>(codes)[oct] = c;
    }
    return byte;
}
// Gathers the scale bytes of 4 neighbouring blocks (16 lanes) into one word, the layout of a
// scale tile's row.
__device__ __forceinline__ uint32_t mx_scale_word(uint32_t byte) {
    uint32_t s = byte << (8u * ((threadIdx.x >> 2) & 3u));
    s |= __shfl_xor_sync(0xffffffffu, s, 4);
    s |= __shfl_xor_sync(0xffffffffu, s, 8);
    return s;
}

// The norm goes over a row longer than 16384 columns this many at a time, counted in 32 bits, which
// the last step must not pass; and over rows with a 31-bit grid.
constexpr uint32_t kMxNormStep = 8192;
inline bool mx_norm_takes(uint32_t rows, uint32_t cols) { return rows <= 0x7fffffffu && cols <= 0u - kMxNormStep; }

// ---- host checks -------------------------------------------------------------------------
inline bool mx_valid(const opure_mx_matrix &m) {
    return (m.format == OPURE_MX_FP4 || m.format == OPURE_MX_FP8) && m.cols != 0 && m.cols <= 0xffffff80u &&
           (m.rows == 0 || (m.codes && m.scales && reinterpret_cast<uintptr_t>(m.codes) % 32 == 0 &&
                            reinterpret_cast<uintptr_t>(m.scales) % 16 == 0));
}
inline uint32_t type_bytes(uint32_t type) { return type == OPURE_F32 ? 4 : type <= OPURE_BF16 ? 2 : 0; }
inline bool type_aligned(const void *p, uint32_t type) {
    return type_bytes(type) && reinterpret_cast<uintptr_t>(p) % type_bytes(type) == 0;
}
// Whether rows can be read and written 16 bytes at a time.
inline bool rows_aligned16(const void *p, uint32_t type, size_t stride) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && stride * type_bytes(type) % 16 == 0;
}

// f(T()) for the C++ type of an opure_type.
template <typename F>
opure_status with_type(uint32_t type, F &&f) {
    if (type == OPURE_F32) return f(float());
    if (type == OPURE_F16) return f(__half());
    return f(__nv_bfloat16());
}

}  // namespace opure
