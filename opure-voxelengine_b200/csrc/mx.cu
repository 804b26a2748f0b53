// mx.cu -- to and from microscaled (MX) form: quantise, dequantise, and RMSNorm with the
// residual's addition and an MX result.
//
// All three are bound by memory: a value is read once and its code written once. Measured: 49152 x
// 2048 fp16 to 4 bits and back 81.5 us (6,250 GB/s), the norm of 8192 x 2048 fp32 with residual and
// sum 34.3 us (6,370 GB/s); copies run at 6,451 GB/s. The norm of 2-byte types is bound by instructions
// (8192 x 2048 fp16 26.5 us, bf16 28.3 us, 18.3 us for the bytes): 8 values a lane share a scale's work.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "mx.cuh"

namespace opure {
namespace {

constexpr uint32_t kThreads = 256;

// To and from MX, a lane owns 16 neighbouring values, 8 lanes the 128 columns whose four scales
// make one word of a scale tile: a group. Groups are counted row after row, so that no lane idles
// at a row's end. At 8 values a lane the same kernels were bound by instructions (half of them
// for the scale and the addresses): 65 us for 49152 x 2048 fp16, against 40 us for the bytes.
struct Groups {
    uint32_t rows, per_row, magic;  // magic: per_row's reciprocal
    __device__ __forceinline__ bool at(uint32_t group, uint32_t &row, uint32_t &c) const {
        // floor(group / per_row) or one more (group < 2^31, magic rounded up), then corrected.
        row = per_row == 1 ? group : __umulhi(group, magic);
        if (row * per_row > group) --row;
        c = (group - row * per_row) * 128 + (threadIdx.x & 7u) * 16;
        return row < rows;
    }
};

// Rows that 32-byte accesses cannot serve (odd strides, unaligned pointers) are read and written
// in the aligned 16-byte words that hold a lane's values, and the values shifted into their places
// in registers. 10432 x 3109 fp16 to 4 bits and back: 39 us; with a warp per group and a lane per
// column of each block, whose shuffles and small accesses the SMs cannot issue fast enough, 92 us.
template <typename T, uint32_t V>
constexpr uint32_t kRegs = V * sizeof(T) / 4;  // of V values

// V values of w, from `bytes` (whole values, at most 15 bytes) on.
template <typename T, uint32_t V>
__device__ __forceinline__ void shift_words(const uint32_t (&w)[kRegs<T, V> + 4], uint32_t bytes, uint32_t (&out)[kRegs<T, V>]) {
    constexpr uint32_t N = kRegs<T, V>;
    uint32_t t[N + 2], u[N + 1];
#pragma unroll
    for (uint32_t i = 0; i < N + 2; ++i) t[i] = bytes & 8u ? w[i + 2] : w[i];
#pragma unroll
    for (uint32_t i = 0; i < N + 1; ++i) u[i] = bytes & 4u ? t[i + 1] : t[i];
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) out[i] = sizeof(T) == 4 ? u[i] : __funnelshift_r(u[i], u[i + 1], (bytes & 3u) * 8u);
}

// The words that hold the V values at p, of a matrix in [begin, end); returns how many bytes of
// them come before p.
template <typename T, uint32_t V>
__device__ __forceinline__ uint32_t load_any(const T *p, const T *begin, const T *end, uint32_t (&w)[kRegs<T, V> + 4]) {
    constexpr uint32_t kWords = kRegs<T, V> / 4;  // of 16 bytes
    const uint32_t before = uint32_t(reinterpret_cast<uintptr_t>(p)) & 15u;
    const uintptr_t first = reinterpret_cast<uintptr_t>(p) - before;
    if (first < reinterpret_cast<uintptr_t>(begin) || first + 16 * (kWords + (before != 0)) > reinterpret_cast<uintptr_t>(end)) {
        T *r = reinterpret_cast<T *>(w);
#pragma unroll
        for (uint32_t j = 0; j < V; ++j) r[j] = p[j];
        return 0;
    }
    const uint4 *words = reinterpret_cast<const uint4 *>(first);
    uint4 q[kWords + 1];
#pragma unroll
    for (uint32_t k = 0; k < kWords; ++k) q[k] = words[k];
    q[kWords] = before ? words[kWords] : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (uint32_t k = 0; k <= kWords; ++k) {
        w[4 * k] = q[k].x;
        w[4 * k + 1] = q[k].y;
        w[4 * k + 2] = q[k].z;
        w[4 * k + 3] = q[k].w;
    }
    return before;
}

// V values to any address: words across two lanes are written by the later lane, if it holds all
// of its values (full) and the lane before it the same row's (follows). All lanes of the warp call.
template <typename T, uint32_t V>
__device__ __forceinline__ void store_any(T *p, bool full, bool follows, const uint32_t (&raw)[kRegs<T, V>]) {
    constexpr uint32_t kWords = kRegs<T, V> / 4;
    const uint32_t lane = threadIdx.x & 31u, before = uint32_t(reinterpret_cast<uintptr_t>(p)) & 15u;
    const bool joins = full && follows && lane != 0;
    const bool joined = __shfl_down_sync(0xffffffffu, joins, 1) && lane != 31;
    uint32_t w[4 * kWords + 4], out[4 * kWords];
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) w[i] = __shfl_up_sync(0xffffffffu, raw[4 * kWords - 4 + i], 1);
#pragma unroll
    for (uint32_t i = 0; i < 4 * kWords; ++i) w[4 + i] = raw[i];
    if (!full) return;
    const T *r = reinterpret_cast<const T *>(raw);
    uint4 *words = reinterpret_cast<uint4 *>(reinterpret_cast<uintptr_t>(p) - before);
    if (before == 0) {
#pragma unroll
        for (uint32_t k = 0; k < kWords; ++k) words[k] = make_uint4(raw[4 * k], raw[4 * k + 1], raw[4 * k + 2], raw[4 * k + 3]);
        return;
    }
    shift_words<T, V>(w, 16 - before, out);
#pragma unroll
    for (uint32_t k = 0; k < kWords; ++k)
        if (k || joins) words[k] = make_uint4(out[4 * k], out[4 * k + 1], out[4 * k + 2], out[4 * k + 3]);
    constexpr uint32_t kPer = 16 / sizeof(T);  // values per word
    const uint32_t later = before / sizeof(T);  // of them after a word's beginning
    if (!joins)
#pragma unroll
        for (uint32_t j = 0; j < kPer - 1; ++j)
            if (j + later < kPer) p[j] = r[j];
    if (!joined)
#pragma unroll
        for (uint32_t j = V + 1 - kPer; j < V; ++j)
            if (j + later >= V) p[j] = r[j];
}

template <typename T, uint32_t FMT, uint32_t U, bool ANY>
__global__ void __launch_bounds__(kThreads)
    mx_quantize_kernel(const T *x, size_t stride, uint8_t *codes, uint8_t *scales, Groups groups, uint32_t cols) {
    grid_dependency_wait();
    grid_dependents_launch();
    const uint32_t first = (blockIdx.x * U * kThreads + threadIdx.x) / 8;
    uint32_t raw[U][4 * sizeof(T) + (ANY ? 4 : 0)];
    uint32_t row[U], c[U], before[U];
    bool in[U];
#pragma unroll
    for (uint32_t i = 0; i < U; ++i) {
        in[i] = groups.at(first + i * (kThreads / 8), row[i], c[i]);
        const T *p = x + size_t(row[i]) * stride + c[i];
        before[i] = 0;
        if (in[i] && c[i] + 16 <= cols) {
            if constexpr (ANY)
                before[i] = load_any<T, 16>(p, x, x + size_t(groups.rows - 1) * stride + cols, raw[i]);
            else
                load16(p, raw[i]);
        } else {
            T *r = reinterpret_cast<T *>(raw[i]);
#pragma unroll
            for (uint32_t j = 0; j < 16; ++j) r[j] = in[i] && c[i] + j < cols ? p[j] : from_f32<T>(0.f);
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < U; ++i) {
        float v[16];
        if constexpr (ANY) {
            uint32_t place[4 * sizeof(T)];
            shift_words<T, 16>(raw[i], before[i], place);
#pragma unroll
            for (uint32_t j = 0; j < 16; ++j) v[j] = to_f32(reinterpret_cast<const T *>(place)[j]);
        } else {
#pragma unroll
            for (uint32_t j = 0; j < 16; ++j) v[j] = to_f32(reinterpret_cast<const T *>(raw[i])[j]);
        }
        float f = max_abs3(v[0], v[1], 0.f);
#pragma unroll
        for (uint32_t j = 2; j < 16; j += 2) f = max_abs3(f, v[j], v[j + 1]);
        uint32_t m = __float_as_uint(f) & 0x7fffffffu;
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        const uint32_t byte = mx_scale_byte<FMT>(m), keep = byte == 255u ? 0u : ~0u;
        const float inv = mx_inverse(byte);
        uint32_t s = byte << (4u * (threadIdx.x & 6u));
        s |= __shfl_xor_sync(0xffffffffu, s, 2);
        s |= __shfl_xor_sync(0xffffffffu, s, 4);
        if (!in[i]) continue;
#pragma unroll
        for (uint32_t j = 0; j < 16; ++j) v[j] *= inv;
        uint8_t *dst = codes + size_t(row[i]) * mx_row_bytes(FMT, cols) + size_t(c[i]) * FMT / 8;
        if constexpr (FMT == OPURE_MX_FP4) {
            const float lo[8] = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
            const float hi[8] = {v[8], v[9], v[10], v[11], v[12], v[13], v[14], v[15]};
            *reinterpret_cast<uint2 *>(dst) = make_uint2(mx_pack_fp4(lo) & keep, mx_pack_fp4(hi) & keep);
        } else {
            *reinterpret_cast<uint4 *>(dst) =
                make_uint4(mx_pack_fp8(v[0], v[1], v[2], v[3]) & keep, mx_pack_fp8(v[4], v[5], v[6], v[7]) & keep,
                           mx_pack_fp8(v[8], v[9], v[10], v[11]) & keep, mx_pack_fp8(v[12], v[13], v[14], v[15]) & keep);
        }
        if (threadIdx.x % 8 == 0) *reinterpret_cast<uint32_t *>(scales + mx_scale_offset(cols, row[i], c[i] / kMxBlock)) = s;
    }
}

template <typename T, uint32_t FMT, uint32_t U, bool ANY>
__global__ void __launch_bounds__(kThreads)
    mx_dequantize_kernel(const uint8_t *codes, const uint8_t *scales, T *y, size_t stride, Groups groups, uint32_t cols) {
    grid_dependency_wait();
    grid_dependents_launch();
    const uint32_t first = (blockIdx.x * U * kThreads + threadIdx.x) / 8;
    using Word = std::conditional_t<FMT == OPURE_MX_FP4, uint2, uint4>;  // 16 codes
    Word code[U];
    uint8_t scale[U];
    uint32_t row[U], c[U];
    bool in[U];
#pragma unroll
    for (uint32_t i = 0; i < U; ++i) {
        in[i] = groups.at(first + i * (kThreads / 8), row[i], c[i]) && c[i] < cols;
        if (in[i]) {
            code[i] = *reinterpret_cast<const Word *>(codes + size_t(row[i]) * mx_row_bytes(FMT, cols) + size_t(c[i]) * FMT / 8);
            scale[i] = scales[mx_scale_offset(cols, row[i], c[i] / kMxBlock)];
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < U; ++i) {
        if constexpr (ANY) {
            if (!__any_sync(0xffffffffu, in[i])) continue;
            if (!in[i]) code[i] = Word{}, scale[i] = 0;
        } else if (!in[i]) {
            continue;
        }
        const float s = mx_scale_value(scale[i]);
        uint32_t h[8];
        const uint32_t *w = reinterpret_cast<const uint32_t *>(&code[i]);
#pragma unroll
        for (uint32_t q = 0; q < 2; ++q) {
            uint32_t f[4];
            if constexpr (FMT == OPURE_MX_FP4) {
                mx_unpack_fp4(w[q], f);
            } else {
                mx_unpack_fp8(w[2 * q], f[0], f[1]);
                mx_unpack_fp8(w[2 * q + 1], f[2], f[3]);
            }
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) h[4 * q + j] = f[j];
        }
        uint32_t raw[4 * sizeof(T)];
        T *r = reinterpret_cast<T *>(raw);
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j) {
            const float2 f = h2f2(h[j]);
            r[2 * j] = from_f32<T>(f.x * s);
            r[2 * j + 1] = from_f32<T>(f.y * s);
        }
        T *p = y + size_t(row[i]) * stride + c[i];
        const bool full = c[i] + 16 <= cols;
        if constexpr (ANY) {
            // The lane before holds the columns before, unless a row begins here.
            store_any<T, 16>(p, in[i] && full, c[i] != 0, raw);
        } else if (full) {
#pragma unroll
            for (uint32_t j = 0; j < sizeof(T) / 2; ++j)
                stg256(reinterpret_cast<uint8_t *>(p) + 32 * j, *reinterpret_cast<const uint32_t(*)[8]>(raw + 8 * j));
        }
        if (in[i] && !full) {
#pragma unroll
            for (uint32_t j = 0; j < 16; ++j)
                if (c[i] + j < cols) p[j] = r[j];
        }
    }
}


// ---- norm ---------------------------------------------------------------------------------
struct NormParams {
    const void *x, *residual;
    void *sum;
    size_t stride;
    const __half *gain;
    double per_col, eps;  // per_col: 1 / cols
    uint8_t *codes, *scales;
    uint32_t rows, cols;
    bool gain_vec;  // the gain allows 16-byte accesses
};

// Sum over a row's threads: a warp's, or a CTA's (part: 32 values).
template <bool WARP>
__device__ __forceinline__ double row_sum(double v, double *part) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if constexpr (!WARP) {
        if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
        __syncthreads();
        v = (threadIdx.x & 31) < blockDim.x / 32 ? part[threadIdx.x & 31] : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    }
    return v;
}

// A result that lies on the other side of a rounding boundary of its code is a whole step off, so
// the norm's own rounding is kept out of the way: a lane's 8 squares are added in fp32, whose
// errors even out over a row, and those sums in 64 bits; the inverse root is a pair of floats (one
// Newton step from rsqrt, with the products' rest by fma), and so is its product with the gain, so
// that a result is rounded once. Each square in 64 bits
// cost 1831 x 7528 fp16 37 us instead of 31.
//
// Where the mean square m leaves the middle of fp32's range, values are first multiplied by a power
// of two (`pre`) that brings it back, and the root is taken of m pre^2: every finite row has a norm,
// from subnormals to the largest values (8192 x 2048 bf16 28.3 us; without the test 27.9).
struct Inverse {
    float hi, lo, pre;
};
// WIDE: T has such values (fp16 has not).
template <bool WIDE>
__device__ __forceinline__ Inverse inverse_rms(double sum_of_squares, const NormParams &p) {
    double m = fma(sum_of_squares, p.per_col, p.eps);
    float mh = float(m), pre = 1.f;
    if (WIDE && __builtin_expect(!(mh >= 0x1p-100f && mh <= 0x1p100f), 0)) {
        const int e = int(uint32_t(__double2hiint(m)) >> 20 & 0x7ffu) - 1023;  // |m| is 2^e or more, 0 2^-1023
        const int half = min(max(e / 2, -120), 120);
        pre = __uint_as_float(uint32_t(127 - half) << 23);
        m *= __hiloint2double((1023 - 2 * half) << 20, 0);
        mh = float(m);
        asm volatile("");  // a branch, not predicated instructions for every row
    }
    const float ml = float(m - double(mh)), y = rsqrtf(mh);
    const float q = mh * y, rest = fmaf(-q, y, 1.0f) - fmaf(mh, y, -q) * y - ml * y * y;  // 1 - m y^2
    const float lo = 0.5f * y * rest;
    return {y, isfinite(lo) ? lo : 0.f, pre};  // m of 0, infinity or NaN: the root alone
}
// Inf and NaN may come out as NaN: either makes the block's scale NaN.
__device__ __forceinline__ float normed(float v, Inverse inv) { return fmaf(v, inv.hi, v * inv.lo); }
__device__ __forceinline__ Inverse gained(Inverse inv, float gain) {
    const float hi = inv.hi * gain;
    return {hi, fmaf(inv.lo, gain, fmaf(inv.hi, gain, -hi)), 1.f};
}

// One CTA per row, or (WARP) one warp per row where there are many short ones: 15007 rows of 75
// took 16 us as that many CTAs. With KEEP a thread holds its (up to KEEP) octets of s between the
// sum of squares and the codes, so that x and residual are read once; KEEP 0, for rows longer
// than 16384, reads them twice (the second time from L2). ANY: rows that 16-byte accesses cannot
// serve.
template <typename T, uint32_t FMT, uint32_t KEEP, bool WARP, bool ANY>
__global__ void __launch_bounds__(WARP ? kThreads : KEEP == 4 ? 512 : 1024) mx_rmsnorm_kernel(NormParams p) {
    __shared__ double part[32];
    grid_dependency_wait();
    grid_dependents_launch();
    const uint32_t width = WARP ? 32 : blockDim.x, place = WARP ? threadIdx.x & 31u : threadIdx.x;
    const uint32_t row = WARP ? mx_warp_row(blockIdx.x, threadIdx.x, kThreads) : blockIdx.x;
    if (WARP && row >= p.rows) return;
    const uint32_t cols = p.cols, kp = mx_kp(cols), step = width * 8, c0 = place * 8;  // no sum of these passes 2^32
    const T *x = static_cast<const T *>(p.x) + size_t(row) * p.stride;
    const T *r = p.residual ? static_cast<const T *>(p.residual) + size_t(row) * p.stride : nullptr;
    T *sum = p.sum ? static_cast<T *>(p.sum) + size_t(row) * p.stride : nullptr;
    auto load = [&](uint32_t c, float (&v)[8]) {
        const uint32_t n = c < cols ? min(cols - c, 8u) : 0u;
        float t[8];
        if (n < 8) {
            load8_part(x + c, n, v);
            if (r) load8_part(r + c, n, t);
        } else if constexpr (ANY) {
            const size_t size = size_t(p.rows - 1) * p.stride + cols;
            const T *px = static_cast<const T *>(p.x), *pr = static_cast<const T *>(p.residual);
            uint32_t wx[kRegs<T, 8> + 4], wr[kRegs<T, 8> + 4], place[kRegs<T, 8>];
            const uint32_t bx = load_any<T, 8>(x + c, px, px + size, wx), br = r ? load_any<T, 8>(r + c, pr, pr + size, wr) : 0u;
            shift_words<T, 8>(wx, bx, place);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = to_f32(reinterpret_cast<const T *>(place)[j]);
            if (r) {
                shift_words<T, 8>(wr, br, place);
#pragma unroll
                for (int j = 0; j < 8; ++j) t[j] = to_f32(reinterpret_cast<const T *>(place)[j]);
            }
        } else {
            load8(x + c, v);
            if (r) load8(r + c, t);
        }
        if (r) {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] += t[j];
        }
    };
    double ss = 0.0;
    auto square = [&](const float (&v)[8]) {
        float q = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) q = fmaf(v[j], v[j], q);
        if (q >= 0x1p-100f && q <= FLT_MAX) {
            ss += double(q);
        } else {  // squares that fp32 has no room for, zeros, NaN
            for (int j = 0; j < 8; ++j) ss = fma(double(v[j]), double(v[j]), ss);
        }
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
    ss = row_sum<WARP>(ss, part);
    constexpr bool kWide = !std::is_same_v<T, __half>;
    const Inverse inv = inverse_rms<kWide>(ss, p);
    uint8_t *codes = p.codes + size_t(row) * mx_row_bytes(FMT, cols);
    auto finish = [&](uint32_t c, float (&v)[8]) {
        const uint32_t n = c < cols ? min(cols - c, 8u) : 0u;
        // sum may be x or residual: this thread alone uses these columns' values and has read them
        // for the last time; what the next lane writes of them comes from this one.
        if (sum) {
            if constexpr (ANY) {
                uint32_t raw[kRegs<T, 8>];
#pragma unroll
                for (int j = 0; j < 8; ++j) reinterpret_cast<T *>(raw)[j] = from_f32<T>(v[j]);
                store_any<T, 8>(sum + c, n == 8, c != 0, raw);
            } else if (n == 8) {
                store8(sum + c, v);
            }
            if (n < 8) store8_part(sum + c, n, v);
        }
        if (kWide && inv.pre != 1.f)
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] *= inv.pre;
        if (p.gain && n) {
            float g[8];
            if (p.gain_vec && n == 8)
                load8(p.gain + c, g);
            else
                load8_part(p.gain + c, n, g);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = normed(v[j], gained(inv, g[j]));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = normed(v[j], inv);
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

// The groups of a matrix, and how many each lane of its kernels takes: two where that still
// fills every SM, so that more loads are in flight; one in smaller calls, where latency counts.
bool make_groups(const opure_ctx *ctx, const opure_mx_matrix &m, Groups &g, uint32_t &per_lane, uint32_t &blocks) {
    g.rows = m.rows;
    g.per_row = mx_kp(m.cols) / 128;
    g.magic = g.per_row == 1 ? 0 : uint32_t(0xffffffffu / g.per_row + 1);
    const uint64_t groups = uint64_t(m.rows) * g.per_row;
    if (groups >= (uint64_t(1) << 31) - kThreads) return false;
    per_lane = groups >= uint64_t(ctx->sm_count) * 8 * kThreads / 8 ? 2 : 1;
    const uint64_t grid = (groups * 8 + kThreads * per_lane - 1) / (kThreads * per_lane);
    blocks = uint32_t(grid);
    return grid <= 0x7fffffffu / kThreads;  // thread indices are 32-bit
}
bool rows_aligned32(const void *p, uint32_t type, size_t stride) {
    return reinterpret_cast<uintptr_t>(p) % 32 == 0 && stride * type_bytes(type) % 32 == 0;
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
    Groups groups;
    uint32_t per_lane, blocks;
    const bool wide = rows_aligned32(x, x_type, x_stride);
    if (!make_groups(ctx, *out, groups, per_lane, blocks)) return OPURE_ERR_UNSUPPORTED;
    return with_type(x_type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto kernel) {
            return launch(ctx, kernel, dim3(blocks), dim3(kThreads), 0, true, static_cast<const T *>(x), x_stride,
                          out->codes, out->scales, groups, out->cols);
        };
        auto pick = [&](auto format) {
            constexpr uint32_t F = decltype(format)::value;
            if (!wide) return per_lane == 1 ? go(mx_quantize_kernel<T, F, 1, true>) : go(mx_quantize_kernel<T, F, 2, true>);
            return per_lane == 1 ? go(mx_quantize_kernel<T, F, 1, false>) : go(mx_quantize_kernel<T, F, 2, false>);
        };
        return out->format == OPURE_MX_FP4 ? pick(std::integral_constant<uint32_t, OPURE_MX_FP4>())
                                           : pick(std::integral_constant<uint32_t, OPURE_MX_FP8>());
    });
}

opure_status opure_mx_dequantize(opure_ctx *ctx, const opure_mx_matrix *x, void *y, uint32_t y_type, size_t y_stride) {
    opure_status s = enter(ctx);
    if (s) return s;
    if (!x || !mx_valid(*x) || !type_aligned(y, y_type) || y_stride < x->cols) return OPURE_ERR_INVALID_ARG;
    if (x->rows == 0) return OPURE_OK;
    if (!y) return OPURE_ERR_INVALID_ARG;
    Groups groups;
    uint32_t per_lane, blocks;
    const bool wide = rows_aligned32(y, y_type, y_stride);
    if (!make_groups(ctx, *x, groups, per_lane, blocks)) return OPURE_ERR_UNSUPPORTED;
    return with_type(y_type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto kernel) {
            return launch(ctx, kernel, dim3(blocks), dim3(kThreads), 0, true, static_cast<const uint8_t *>(x->codes),
                          static_cast<const uint8_t *>(x->scales), static_cast<T *>(y), y_stride, groups, x->cols);
        };
        auto pick = [&](auto format) {
            constexpr uint32_t F = decltype(format)::value;
            if (!wide) return per_lane == 1 ? go(mx_dequantize_kernel<T, F, 1, true>) : go(mx_dequantize_kernel<T, F, 2, true>);
            return per_lane == 1 ? go(mx_dequantize_kernel<T, F, 1, false>) : go(mx_dequantize_kernel<T, F, 2, false>);
        };
        return x->format == OPURE_MX_FP4 ? pick(std::integral_constant<uint32_t, OPURE_MX_FP4>())
                                         : pick(std::integral_constant<uint32_t, OPURE_MX_FP8>());
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
    if (!mx_norm_takes(a->out.rows, a->out.cols)) return OPURE_ERR_UNSUPPORTED;
    const NormParams p{a->x, a->residual, a->sum, a->x_stride, reinterpret_cast<const __half *>(a->gain), 1.0 / a->out.cols, a->eps,
                       a->out.codes, a->out.scales, a->out.rows, a->out.cols, reinterpret_cast<uintptr_t>(a->gain) % 16 == 0};
    const bool wide = rows_aligned16(a->x, a->x_type, a->x_stride) && rows_aligned16(a->residual, a->x_type, a->x_stride) &&
                      rows_aligned16(a->sum, a->x_type, a->x_stride);
    // A thread per octet up to 1024 threads, then two octets each. Where that is more threads than
    // the SMs hold at once, octets of 2-byte types, whose loads are half as long, go two (four) to a
    // thread for more bytes in flight: 1831 x 7524 fp16 36 us instead of 51, 512 x 16384 bf16 18 us
    // instead of 22; but fp32 39 us instead of 37 and, with fewer rows, 600 x 577 bf16 3.9 us
    // instead of 3.2. Rows of up to 512 values go one to a warp where that gives every SM 8 or more;
    // fewer or longer ones have a CTA each.
    const uint32_t octets = mx_kp(a->out.cols) / 8;
    const bool twice = type_bytes(a->x_type) == 2 && uint64_t(a->out.rows) * octets > uint64_t(ctx->sm_count) * 2048;
    const uint32_t keep = octets > 2048 ? 0 : (octets <= 1024 ? 1 : 2) * (twice ? 2 : 1);
    const uint32_t threads = keep ? (ceil_div(octets, keep) + 31) / 32 * 32 : kMxNormStep / 8;
    const bool warps = octets <= 64 && a->out.rows >= uint32_t(ctx->sm_count) * 8;
    return with_type(a->x_type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto kernel) {
            return warps ? launch(ctx, kernel, dim3(ceil_div(a->out.rows, kThreads / 32)), dim3(kThreads), 0, true, p)
                         : launch(ctx, kernel, dim3(a->out.rows), dim3(threads), 0, true, p);
        };
        auto pick = [&](auto format, auto any) {
            constexpr uint32_t F = decltype(format)::value;
            constexpr bool A = decltype(any)::value;
            if (warps) return octets <= 32 ? go(mx_rmsnorm_kernel<T, F, 1, true, A>) : go(mx_rmsnorm_kernel<T, F, 2, true, A>);
            if constexpr (sizeof(T) == 2)
                if (keep == 4) return go(mx_rmsnorm_kernel<T, F, 4, false, A>);
            return keep == 1   ? go(mx_rmsnorm_kernel<T, F, 1, false, A>)
                   : keep == 2 ? go(mx_rmsnorm_kernel<T, F, 2, false, A>)
                               : go(mx_rmsnorm_kernel<T, F, 0, false, A>);
        };
        auto pick_format = [&](auto any) {
            return a->out.format == OPURE_MX_FP4 ? pick(std::integral_constant<uint32_t, OPURE_MX_FP4>(), any)
                                                 : pick(std::integral_constant<uint32_t, OPURE_MX_FP8>(), any);
        };
        return wide ? pick_format(std::false_type()) : pick_format(std::true_type());
    });
}

}  // extern "C"
