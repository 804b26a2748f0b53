// kv4.cu -- appending to the 4-bit paged KV cache with RoPE on the way, and reading rows back.
//
// A block of 16 columns of a key or value row becomes E2M1 codes and one E4M3 scale (opure_cuda.h).
// A thread takes a whole block: it rotates the 8 pairs, finds the largest magnitude, and writes 8
// bytes of codes and the scale, without talking to other lanes. Codes and scales are those of the
// definition exactly: a rotated value comes out of double as an fp32 number with its last bit set
// where bits were cut off (so that it lies on the same side of every rounding boundary), and
// quotients that land on a boundary are moved to the side that their remainder is on.
//
// 8192 tokens of 32 + 64 heads of 64, fp16: 52 us the append and 30 the read, 239 MB or 37 us of memory at the copy
// rate together. The append issues 60% of the time, the conversions between fp32 and fp64 fill 45% of their
// unit's slots, DRAM is at 28%: its stores of 1 to 8 bytes make 5.5 million sectors of 1.6 million's data. The
// read waits for loads of 1 to 8 bytes (issue 28%, DRAM 11%). A block a thread is kept for its independence of
// other lanes: 64 tokens take 6.3 us, two launches' time.
#include "kv4.cuh"

namespace opure {
namespace {

constexpr uint32_t kThreads = 128;

struct AppendParams {
    const void *qkv;
    size_t stride;
    void *q_out;
    size_t q_stride;
    const int32_t *seq, *pos;
    uint32_t n, n_heads;
    double log2_theta;
    bool rotate;
    float k_inv, v_inv;      // 1 / tensor scales
    uint32_t first;          // first head that there is work for (queries are skipped without q_out)
    opure_kv4_layout kv;
    DeviceStatus *st;
};

// d in fp32 with the last bit set where it is not exact.
__device__ __forceinline__ float to_odd(double d) {
    const float f = __double2float_rz(d);
    return double(f) != d ? __uint_as_float(__float_as_uint(f) | 1u) : f;
}
// A quotient q of x / s rounded to fp32: where it is a number of at most 3 (codes) or 5 (scales)
// bits, one step towards the true quotient, so that a later rounding to fewer bits sees the side.
__device__ __forceinline__ float towards(float q, float s, float x, uint32_t low_bits) {
    const uint32_t b = __float_as_uint(q);
    if ((b & low_bits) == 0u) {
        const float r = fmaf(-q, s, x);
        if (r != 0.f) return __uint_as_float(((__float_as_uint(r) ^ b) >> 31) ? b - 1u : b + 1u);
    }
    return q;
}

// 16 values (times inv, a power of two) -> codes and the scale byte.
__device__ __forceinline__ uint32_t quantise16(float (&v)[16], float inv, uint2 &codes) {
    float m = max_abs3(v[0], v[1], v[2]);
#pragma unroll
    for (int j = 3; j < 15; j += 2) m = max_abs3(m, v[j], v[j + 1]);
    m = max_abs3(m, v[15], 0.f);
    codes = make_uint2(0u, 0u);
    if (!(m < __uint_as_float(0x7f800000u))) return 0x7fu;
    if (m * inv > 1e30f) {  // as good as infinite after the tensor scale: these blocks saturate anyway
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = fminf(fmaxf(v[j], -1e30f / inv), 1e30f / inv);
    }
    m = fminf(m * inv, 1e30f);
    const float quotient = m == 0.f ? 0.f : towards(__fdiv_rn(m, 6.f), 6.f, m, 0x7ffffu);
    const uint32_t byte = mx_pack_fp8(quotient, 0.f, 0.f, 0.f) & 0xffu;
    if (byte == 0u) return 0u;
    const uint32_t pair = kv4_scale_pair(byte);
    const float s = __low2float(*reinterpret_cast<const __half2 *>(&pair));
    // 1 / s as a sum of two floats: x times it is the quotient correctly rounded, but for what
    // `towards` settles.
    const float rh = __frcp_rn(s), rl = fmaf(-s, rh, 1.f) * rh;
    float lo[8], hi[8];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const float x = v[j] * inv;
        const float q = towards(fmaf(x, rh, x * rl), s, x, 0x1fffffu);
        (j < 8 ? lo[j & 7] : hi[j & 7]) = q;
    }
    codes = make_uint2(mx_pack_fp4(lo), mx_pack_fp4(hi));
    return byte;
}

template <typename T, bool VEC>
__device__ __forceinline__ void load_block(const T *p, float (&v)[16]) {
    if constexpr (VEC) {
        load8(p, *reinterpret_cast<float(*)[8]>(v));
        load8(p + 8, *reinterpret_cast<float(*)[8]>(v + 8));
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = to_f32(p[j]);
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_block(T *p, const float (&v)[16]) {
    if constexpr (VEC) {
        store8(p, *reinterpret_cast<const float(*)[8]>(v));
        store8(p + 8, *reinterpret_cast<const float(*)[8]>(v + 8));
    } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) p[j] = from_f32<T>(v[j]);
    }
}

// One CTA per token vector and part of its heads (grid.y): the angles' sines and cosines once per CTA.
template <typename T, int HD, bool VEC>
__global__ void __launch_bounds__(kThreads) append_kernel(AppendParams p) {
    constexpr uint32_t kBlocks = HD / 16;
    __shared__ double2 turn[kBlocks * 9];  // 8 pairs a block and a gap, so that blocks start in other banks
    grid_dependency_wait();
    grid_dependents_launch();
    const uint32_t i = blockIdx.x;
    const int32_t seq = p.seq[i], pos = p.pos[i];
    if (seq < 0) return;
    if (p.rotate) {
        for (uint32_t k = threadIdx.x; k < HD / 2; k += kThreads) {
            // Half turns: pos * theta^(-2 k / HD) / pi, reduced exactly by sincospi.
            const double f = exp2(-(2.0 / HD) * double(k) * p.log2_theta) * 0.31830988618379067154;
            double s, c;
            sincospi(double(pos) * f, &s, &c);
            turn[k / 8 * 9 + k % 8] = make_double2(c, s);
        }
        __syncthreads();
    }
    const uint32_t n_kv = p.kv.n_kv, items = (p.n_heads + 2 * n_kv) * kBlocks;
    const T *row = static_cast<const T *>(p.qkv) + size_t(i) * p.stride;
    for (uint32_t it = p.first * kBlocks + blockIdx.y * kThreads + threadIdx.x; it < items; it += gridDim.y * kThreads) {
        const uint32_t head = it / kBlocks, b = it % kBlocks;
        float v[16];
        load_block<T, VEC>(row + size_t(it) * 16, v);
        const bool is_q = head < p.n_heads, is_v = head >= p.n_heads + n_kv;
        if (!is_v && p.rotate) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const double2 t = turn[b * 9 + j];
                const double a = v[2 * j], e = v[2 * j + 1];
                const double r0 = a * t.x - e * t.y, r1 = a * t.y + e * t.x;
                v[2 * j] = is_q ? float(r0) : to_odd(r0);
                v[2 * j + 1] = is_q ? float(r1) : to_odd(r1);
            }
        }
        if (is_q) {
            store_block<T, VEC>(static_cast<T *>(p.q_out) + size_t(i) * p.q_stride + size_t(it) * 16, v);
            continue;
        }
        const uint32_t kvh = head - p.n_heads - (is_v ? n_kv : 0u);
        uint8_t *group = kv4_group(p.kv, seq, pos, kvh, p.st, 90);
        if (!group) continue;
        const uint32_t t = uint32_t(pos) % kKv4Group;
        uint2 codes;
        const uint32_t scale = quantise16(v, is_v ? p.v_inv : p.k_inv, codes);
        if (is_v) {
            *reinterpret_cast<uint32_t *>(group + kv4_value_at(HD, t, 2 * b)) = codes.x;
            *reinterpret_cast<uint32_t *>(group + kv4_value_at(HD, t, 2 * b + 1)) = codes.y;
            group[kv4_value_scale_at(HD, t, b)] = uint8_t(scale);
        } else {
            *reinterpret_cast<uint2 *>(group + kv4_key_at(t, b)) = codes;
            group[kv4_key_scale_at(HD, t, b)] = uint8_t(scale);
        }
    }
}

struct ReadParams {
    void *k, *v;
    size_t stride;
    const int32_t *seq, *pos;
    float k_scale, v_scale;
    opure_kv4_layout kv;
    DeviceStatus *st;
};

__device__ __forceinline__ void dequantise16(uint2 codes, uint32_t scale, float tensor, float (&v)[16]) {
    const uint32_t pair = kv4_scale_pair(scale);
    const float s = __low2float(*reinterpret_cast<const __half2 *>(&pair)) * tensor;
    uint32_t h[8];
    mx_unpack_fp4(codes.x, *reinterpret_cast<uint32_t(*)[4]>(h));
    mx_unpack_fp4(codes.y, *reinterpret_cast<uint32_t(*)[4]>(h + 4));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float2 f = h2f2(h[j]);
        v[2 * j] = f.x * s;
        v[2 * j + 1] = f.y * s;
    }
}

template <typename T, int HD, bool VEC>
__global__ void __launch_bounds__(kThreads) read_kernel(ReadParams p) {
    constexpr uint32_t kBlocks = HD / 16;
    grid_dependency_wait();
    grid_dependents_launch();
    const uint32_t i = blockIdx.x;
    const int32_t seq = p.seq[i], pos = p.pos[i];
    if (seq < 0) return;
    for (uint32_t it = blockIdx.y * kThreads + threadIdx.x; it < p.kv.n_kv * kBlocks; it += gridDim.y * kThreads) {
        const uint32_t b = it % kBlocks, t = uint32_t(pos) % kKv4Group;
        const uint8_t *group = kv4_group(p.kv, seq, pos, it / kBlocks, p.st, 91);
        if (!group) continue;
        float v[16];
        if (p.k) {
            dequantise16(*reinterpret_cast<const uint2 *>(group + kv4_key_at(t, b)), group[kv4_key_scale_at(HD, t, b)], p.k_scale, v);
            store_block<T, VEC>(static_cast<T *>(p.k) + size_t(i) * p.stride + size_t(it) * 16, v);
        }
        if (p.v) {
            const uint2 codes = make_uint2(*reinterpret_cast<const uint32_t *>(group + kv4_value_at(HD, t, 2 * b)),
                                           *reinterpret_cast<const uint32_t *>(group + kv4_value_at(HD, t, 2 * b + 1)));
            dequantise16(codes, group[kv4_value_scale_at(HD, t, b)], p.v_scale, v);
            store_block<T, VEC>(static_cast<T *>(p.v) + size_t(i) * p.stride + size_t(it) * 16, v);
        }
    }
}

float or_one(float s) { return s == 0.f ? 1.f : s; }

// Parts of a vector's heads on different CTAs: as many as keep every SM busy, down to one block of
// 16 columns a thread.
uint32_t parts(uint32_t n, uint32_t items, int sms) {
    const uint32_t most = ceil_div(items, kThreads), want = ceil_div(uint64_t(sms) * 4, n);
    return most < want ? most : want;
}

}  // namespace
}  // namespace opure

using namespace opure;

extern "C" size_t opure_kv4_page_bytes(uint32_t n_kv, uint32_t hd, uint32_t page_size) {
    return kv4_shape(n_kv, hd, page_size) ? size_t(n_kv) * (page_size / kKv4Group) * kv4_group_bytes(hd) : 0;
}

extern "C" opure_status opure_kv4_append(opure_ctx *ctx, const opure_kv4_append_args *a) {
    opure_status s = enter(ctx);
    if (s) return s;
    if (!a || type_bytes(a->type) == 0 || !(a->theta >= 0.0) || std::isinf(a->theta)) return OPURE_ERR_INVALID_ARG;
    if ((s = kv4_check(a->kv))) return s;
    const uint64_t hd = a->kv.head_dim, q_cols = a->n_heads * hd, cols = q_cols + 2 * a->kv.n_kv * hd;
    if (a->n_heads % a->kv.n_kv || a->stride < cols || (a->q_out && a->q_stride < q_cols)) return OPURE_ERR_INVALID_ARG;
    if (cols > 0x7fffffffu || a->n > 0x7fffffffu) return OPURE_ERR_UNSUPPORTED;
    if (a->n == 0) return OPURE_OK;
    if (!a->qkv || !a->seq || !a->pos || !type_aligned(a->qkv, a->type) || !type_aligned(a->q_out, a->type)) return OPURE_ERR_INVALID_ARG;
    AppendParams p{};
    p.qkv = a->qkv;
    p.stride = a->stride;
    p.q_out = a->q_out;
    p.q_stride = a->q_stride;
    p.seq = a->seq;
    p.pos = a->pos;
    p.n = a->n;
    p.n_heads = a->n_heads;
    p.rotate = a->theta > 0.0;
    p.log2_theta = p.rotate ? std::log2(a->theta) : 0.0;
    p.k_inv = 1.f / or_one(a->kv.k_scale);
    p.v_inv = 1.f / or_one(a->kv.v_scale);
    p.first = a->q_out ? 0 : a->n_heads;
    p.kv = a->kv;
    p.st = ctx->status;
    const bool vec = rows_aligned16(a->qkv, a->type, a->stride) && (!a->q_out || rows_aligned16(a->q_out, a->type, a->q_stride));
    const uint32_t items = uint32_t((cols - p.first * hd) / 16);
    const dim3 grid(a->n, parts(a->n, items, ctx->sm_count));
    return with_type(a->type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto k) { return launch(ctx, k, grid, dim3(kThreads), 0, true, p); };
        if (hd == 64) return vec ? go(append_kernel<T, 64, true>) : go(append_kernel<T, 64, false>);
        return vec ? go(append_kernel<T, 128, true>) : go(append_kernel<T, 128, false>);
    });
}

extern "C" opure_status opure_kv4_read(opure_ctx *ctx, const opure_kv4_read_args *a) {
    opure_status s = enter(ctx);
    if (s) return s;
    if (!a || type_bytes(a->type) == 0) return OPURE_ERR_INVALID_ARG;
    if ((s = kv4_check(a->kv))) return s;
    const uint64_t cols = uint64_t(a->kv.n_kv) * a->kv.head_dim;
    if (a->stride < cols || (!a->k && !a->v)) return OPURE_ERR_INVALID_ARG;
    if (a->n > 0x7fffffffu) return OPURE_ERR_UNSUPPORTED;
    if (a->n == 0) return OPURE_OK;
    if (!a->seq || !a->pos || !type_aligned(a->k, a->type) || !type_aligned(a->v, a->type)) return OPURE_ERR_INVALID_ARG;
    ReadParams p{a->k, a->v, a->stride, a->seq, a->pos, or_one(a->kv.k_scale), or_one(a->kv.v_scale), a->kv, ctx->status};
    const bool vec = rows_aligned16(a->k, a->type, a->stride) && rows_aligned16(a->v, a->type, a->stride);
    const dim3 grid(a->n, parts(a->n, uint32_t(cols / 16), ctx->sm_count));
    return with_type(a->type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto k) { return launch(ctx, k, grid, dim3(kThreads), 0, true, p); };
        if (a->kv.head_dim == 64) return vec ? go(read_kernel<T, 64, true>) : go(read_kernel<T, 64, false>);
        return vec ? go(read_kernel<T, 128, true>) : go(read_kernel<T, 128, false>);
    });
}
