// mx.cu -- to and from microscaled (MX) form: quantise, dequantise, and RMSNorm with the
// residual's addition and an MX result.
//
// All three are bound by memory: a value is read once and its code written once. A lane owns
// 8 neighbouring values (one 16-byte load of 16-bit values, two of fp32), 4 lanes a block of
// 32, 16 lanes the four blocks whose scales make one 4-byte word of a scale tile.
#include <algorithm>
#include <type_traits>

#include "mx.cuh"

namespace opure {
namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kUnitCols = 256;  // columns that a warp takes at once
constexpr uint32_t kUnits = 4;       // how many times: loads of all are in flight together

// A warp's units: pieces of 256 columns, row after row.
struct Units {
    uint32_t row, piece, per_row;
    __device__ __forceinline__ Units(uint32_t cols) {
        per_row = (mx_kp(cols) + kUnitCols - 1) / kUnitCols;
        const uint32_t unit = (blockIdx.x * (kThreads / 32) + threadIdx.x / 32) * kUnits;
        row = unit / per_row;
        piece = unit - row * per_row;
    }
    // This lane's first column in the current unit, then on to the next one.
    __device__ __forceinline__ uint32_t column() const { return piece * kUnitCols + (threadIdx.x & 31u) * 8; }
    __device__ __forceinline__ void next() {
        if (++piece == per_row) {
            piece = 0;
            ++row;
        }
    }
};

template <typename T, uint32_t FMT, bool VEC>
__global__ void __launch_bounds__(kThreads)
    mx_quantize_kernel(const T *x, size_t stride, uint8_t *codes, uint8_t *scales, uint32_t rows, uint32_t cols) {
    grid_dependency_wait();
    grid_dependents_launch();
    const uint32_t kp = mx_kp(cols);
    float v[kUnits][8];
    Units u(cols), w = u;
#pragma unroll
    for (uint32_t i = 0; i < kUnits; ++i, u.next()) {
        const uint32_t c = u.column(), n = u.row < rows && c < cols ? min(cols - c, 8u) : 0u;
        const T *p = x + size_t(u.row) * stride + c;
        if (VEC && n == 8)
            load8(p, v[i]);
        else
            load8_part(p, n, v[i]);
    }
#pragma unroll
    for (uint32_t i = 0; i < kUnits; ++i, w.next()) {
        const uint32_t c = w.column();
        const bool in = w.row < rows && c < kp;
        const uint32_t byte = mx_store_octet<FMT>(v[i], codes + size_t(w.row) * mx_row_bytes(FMT, cols), c / 8, in);
        const uint32_t word = mx_scale_word(byte);
        if (in && threadIdx.x % 16 == 0)
            *reinterpret_cast<uint32_t *>(scales + mx_scale_offset(cols, w.row, c / kMxBlock)) = word;
    }
}

template <typename T, uint32_t FMT, bool VEC>
__global__ void __launch_bounds__(kThreads)
    mx_dequantize_kernel(const uint8_t *codes, const uint8_t *scales, T *y, size_t stride, uint32_t rows, uint32_t cols) {
    using Word = std::conditional_t<FMT == OPURE_MX_FP4, uint32_t, uint2>;  // 8 codes
    grid_dependency_wait();
    grid_dependents_launch();
    Word code[kUnits];
    uint8_t scale[kUnits];
    Units u(cols), w = u;
#pragma unroll
    for (uint32_t i = 0; i < kUnits; ++i, u.next()) {
        const uint32_t c = u.column();
        code[i] = Word{};
        scale[i] = 0;
        if (u.row < rows && c < cols) {
            code[i] = reinterpret_cast<const Word *>(codes + size_t(u.row) * mx_row_bytes(FMT, cols))[c / 8];
            scale[i] = scales[mx_scale_offset(cols, u.row, c / kMxBlock)];
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < kUnits; ++i, w.next()) {
        const uint32_t c = w.column();
        if (w.row >= rows || c >= cols) continue;
        const float s = mx_scale_value(scale[i]);
        uint32_t h[4];
        if constexpr (FMT == OPURE_MX_FP4) {
            mx_unpack_fp4(code[i], h);
        } else {
            mx_unpack_fp8(code[i].x, h[0], h[1]);
            mx_unpack_fp8(code[i].y, h[2], h[3]);
        }
        float v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = h2f2(h[j]);
            v[2 * j] = f.x * s;
            v[2 * j + 1] = f.y * s;
        }
        T *p = y + size_t(w.row) * stride + c;
        if (VEC && cols - c >= 8)
            store8(p, v);
        else
            store8_part(p, min(cols - c, 8u), v);
    }
}

// ---- norm ---------------------------------------------------------------------------------
struct NormParams {
    const void *x, *residual;
    void *sum;
    size_t stride;
    const __half *gain;
    float eps;
    uint8_t *codes, *scales;
    uint32_t cols;
    bool vec, gain_vec;  // rows of x, residual and sum, and the gain, allow 16-byte accesses
};

// One CTA per row. With KEEP a thread holds its (up to KEEP) octets of s between the sum of
// squares and the codes, so that x and residual are read once; KEEP 0, for rows longer than
// 16384, reads them twice (the second time from L2).
template <typename T, uint32_t FMT, uint32_t KEEP>
__global__ void __launch_bounds__(1024) mx_rmsnorm_kernel(NormParams p) {
    __shared__ float part[32];
    grid_dependency_wait();
    grid_dependents_launch();
    const uint32_t row = blockIdx.x, cols = p.cols, kp = mx_kp(cols), step = blockDim.x * 8, c0 = threadIdx.x * 8;
    const T *x = static_cast<const T *>(p.x) + size_t(row) * p.stride;
    const T *r = p.residual ? static_cast<const T *>(p.residual) + size_t(row) * p.stride : nullptr;
    T *sum = p.sum ? static_cast<T *>(p.sum) + size_t(row) * p.stride : nullptr;
    auto load = [&](uint32_t c, float (&v)[8]) {
        const uint32_t n = c < cols ? min(cols - c, 8u) : 0u;
        if (p.vec && n == 8)
            load8(x + c, v);
        else
            load8_part(x + c, n, v);
        if (r) {
            float t[8];
            if (p.vec && n == 8)
                load8(r + c, t);
            else
                load8_part(r + c, n, t);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += t[j];
        }
    };
    float ss = 0.f;
    auto square = [&](const float (&v)[8]) {
#pragma unroll
        for (int j = 0; j < 8; ++j) ss = fmaf(v[j], v[j], ss);
    };
    float kept[KEEP ? KEEP : 1][8];
    if constexpr (KEEP > 0) {
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i) load(c0 + i * step, kept[i]);
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i) square(kept[i]);
    } else {
        for (uint32_t c = c0; c < cols; c += step) {
            load(c, kept[0]);
            square(kept[0]);
        }
    }
    ss = warp_sum(ss);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = ss;
    __syncthreads();
    ss = 0.f;
    for (uint32_t w = 0; w < blockDim.x / 32; ++w) ss += part[w];
    const float inv = 1.0f / sqrtf(ss / float(cols) + p.eps);
    uint8_t *codes = p.codes + size_t(row) * mx_row_bytes(FMT, cols);
    auto finish = [&](uint32_t c, float (&v)[8]) {
        const uint32_t n = c < cols ? min(cols - c, 8u) : 0u;
        // sum may be x or residual: this thread alone reads and writes these columns, and it
        // has read them for the last time.
        if (sum && n) {
            if (p.vec && n == 8)
                store8(sum + c, v);
            else
                store8_part(sum + c, n, v);
        }
        if (p.gain && n) {
            float g[8];
            if (p.gain_vec && n == 8)
                load8(p.gain + c, g);
            else
                load8_part(p.gain + c, n, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = v[j] * inv * g[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= inv;
        }
        const uint32_t byte = mx_store_octet<FMT>(v, codes, c / 8, c < kp);
        const uint32_t word = mx_scale_word(byte);
        if (c < kp && threadIdx.x % 16 == 0)
            *reinterpret_cast<uint32_t *>(p.scales + mx_scale_offset(cols, row, c / kMxBlock)) = word;
    };
    if constexpr (KEEP > 0) {
#pragma unroll
        for (uint32_t i = 0; i < KEEP; ++i) finish(c0 + i * step, kept[i]);
    } else {
        for (uint32_t b = 0; b < kp; b += step) {
            load(b + c0, kept[0]);
            finish(b + c0, kept[0]);
        }
    }
}

// Blocks of kThreads that cover a matrix; 0 when there would be too many units to count.
uint32_t unit_blocks(const opure_mx_matrix &m) {
    const uint64_t units = uint64_t(m.rows) * ceil_div(mx_kp(m.cols), kUnitCols);
    const uint64_t per_block = kThreads / 32 * kUnits;
    return units < 0xffffffffu - per_block ? uint32_t((units + per_block - 1) / per_block) : 0u;
}

}  // namespace
}  // namespace opure

using namespace opure;

extern "C" {

size_t opure_mx_code_bytes(uint32_t format, uint32_t rows, uint32_t cols) {
    if (format != OPURE_MX_FP4 && format != OPURE_MX_FP8) return 0;
    return rows * mx_row_bytes(format, cols);
}

size_t opure_mx_scale_bytes(uint32_t rows, uint32_t cols) {
    return (size_t(rows) + 127) / 128 * (mx_kp(cols) / 128) * kMxTileBytes;
}

opure_status opure_mx_quantize(opure_ctx *ctx, const void *x, uint32_t x_type, size_t x_stride,
                               const opure_mx_matrix *out) {
    opure_status s = enter(ctx);
    if (s) return s;
    if (!out || !mx_valid(*out) || !type_aligned(x, x_type) || x_stride < out->cols) return OPURE_ERR_INVALID_ARG;
    if (out->rows == 0) return OPURE_OK;
    if (!x) return OPURE_ERR_INVALID_ARG;
    const uint32_t blocks = unit_blocks(*out);
    if (!blocks) return OPURE_ERR_UNSUPPORTED;
    const bool vec = rows_aligned16(x, x_type, x_stride);
    return with_type(x_type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto kernel) {
            return launch(ctx, kernel, dim3(blocks), dim3(kThreads), 0, true, static_cast<const T *>(x), x_stride,
                          out->codes, out->scales, out->rows, out->cols);
        };
        if (out->format == OPURE_MX_FP4)
            return vec ? go(mx_quantize_kernel<T, OPURE_MX_FP4, true>) : go(mx_quantize_kernel<T, OPURE_MX_FP4, false>);
        return vec ? go(mx_quantize_kernel<T, OPURE_MX_FP8, true>) : go(mx_quantize_kernel<T, OPURE_MX_FP8, false>);
    });
}

opure_status opure_mx_dequantize(opure_ctx *ctx, const opure_mx_matrix *x, void *y, uint32_t y_type, size_t y_stride) {
    opure_status s = enter(ctx);
    if (s) return s;
    if (!x || !mx_valid(*x) || !type_aligned(y, y_type) || y_stride < x->cols) return OPURE_ERR_INVALID_ARG;
    if (x->rows == 0) return OPURE_OK;
    if (!y) return OPURE_ERR_INVALID_ARG;
    const uint32_t blocks = unit_blocks(*x);
    if (!blocks) return OPURE_ERR_UNSUPPORTED;
    const bool vec = rows_aligned16(y, y_type, y_stride);
    return with_type(y_type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto kernel) {
            return launch(ctx, kernel, dim3(blocks), dim3(kThreads), 0, true, static_cast<const uint8_t *>(x->codes),
                          static_cast<const uint8_t *>(x->scales), static_cast<T *>(y), y_stride, x->rows, x->cols);
        };
        if (x->format == OPURE_MX_FP4)
            return vec ? go(mx_dequantize_kernel<T, OPURE_MX_FP4, true>) : go(mx_dequantize_kernel<T, OPURE_MX_FP4, false>);
        return vec ? go(mx_dequantize_kernel<T, OPURE_MX_FP8, true>) : go(mx_dequantize_kernel<T, OPURE_MX_FP8, false>);
    });
}

opure_status opure_mx_rmsnorm(opure_ctx *ctx, const opure_mx_norm_args *a) {
    opure_status s = enter(ctx);
    if (s) return s;
    if (!a || !mx_valid(a->out) || !type_aligned(a->x, a->x_type) || !type_aligned(a->residual, a->x_type) ||
        !type_aligned(a->sum, a->x_type) || reinterpret_cast<uintptr_t>(a->gain) % 2 || a->x_stride < a->out.cols)
        return OPURE_ERR_INVALID_ARG;
    if (a->out.rows == 0) return OPURE_OK;
    if (!a->x) return OPURE_ERR_INVALID_ARG;
    if (a->out.rows > 0x7fffffffu) return OPURE_ERR_UNSUPPORTED;
    NormParams p{a->x, a->residual, a->sum, a->x_stride, reinterpret_cast<const __half *>(a->gain), a->eps,
                 a->out.codes, a->out.scales, a->out.cols,
                 rows_aligned16(a->x, a->x_type, a->x_stride) && rows_aligned16(a->residual, a->x_type, a->x_stride) &&
                     rows_aligned16(a->sum, a->x_type, a->x_stride),
                 reinterpret_cast<uintptr_t>(a->gain) % 16 == 0};
    // A thread per 8 values up to 1024 threads, then two octets each.
    const uint32_t octets = mx_kp(a->out.cols) / 8, keep = octets <= 1024 ? 1 : octets <= 2048 ? 2 : 0;
    const uint32_t threads = keep ? (ceil_div(octets, keep) + 31) / 32 * 32 : 1024;
    return with_type(a->x_type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto kernel) { return launch(ctx, kernel, dim3(a->out.rows), dim3(threads), 0, true, p); };
        auto pick = [&](auto format) {
            constexpr uint32_t F = decltype(format)::value;
            return keep == 1 ? go(mx_rmsnorm_kernel<T, F, 1>) : keep == 2 ? go(mx_rmsnorm_kernel<T, F, 2>) : go(mx_rmsnorm_kernel<T, F, 0>);
        };
        return a->out.format == OPURE_MX_FP4 ? pick(std::integral_constant<uint32_t, OPURE_MX_FP4>())
                                             : pick(std::integral_constant<uint32_t, OPURE_MX_FP8>());
    });
}

}  // extern "C"
