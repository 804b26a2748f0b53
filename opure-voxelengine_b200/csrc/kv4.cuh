// kv4.cuh -- the 4-bit paged KV cache: layout, conversions and host checks shared by kv4.cu (append,
// read) and kv4_attention.cu. Layout: opure_kv4_layout in opure_cuda.h.
#pragma once

#include <cmath>

#include "mx.cuh"

namespace opure {

constexpr uint32_t kKv4Group = 16;  // positions in a group
__host__ __device__ constexpr uint32_t kv4_group_bytes(uint32_t hd) { return 18u * hd; }

// Offsets within a group: the 8 bytes of key codes of (position t, block b of 16 columns), the 4 bytes
// of value codes of (t, octet of columns), and the scale bytes.
__host__ __device__ __forceinline__ uint32_t kv4_key_at(uint32_t t, uint32_t b) {
    return b / 4 * 512 + t % 8 * 64 + b % 4 * 16 + t / 8 * 8;
}
__host__ __device__ __forceinline__ uint32_t kv4_value_lane(uint32_t t) { return t % 8 / 2; }            // c
__host__ __device__ __forceinline__ uint32_t kv4_value_slot(uint32_t t) { return t % 2 + 2 * (t / 8); }  // t of the layout
__host__ __device__ __forceinline__ uint32_t kv4_value_at(uint32_t hd, uint32_t t, uint32_t octet) {
    return 8 * hd + octet / 8 * 512 + octet % 8 * 64 + kv4_value_lane(t) * 16 + kv4_value_slot(t) * 4;
}
__host__ __device__ __forceinline__ uint32_t kv4_key_scale_at(uint32_t hd, uint32_t t, uint32_t b) {
    return 16 * hd + b / 4 * 64 + t % 8 * 8 + b % 4 * 2 + t / 8;
}
__host__ __device__ __forceinline__ uint32_t kv4_value_scale_at(uint32_t hd, uint32_t t, uint32_t b) {
    return 17 * hd + b / 4 * 64 + b % 4 * 16 + kv4_value_lane(t) * 4 + kv4_value_slot(t);
}

// The group of position `pos` of a sequence for one kv head, or null (reported) where the table has no
// page of the pool for it.
__device__ __forceinline__ uint8_t *kv4_group(const opure_kv4_layout &kv, int32_t seq, int32_t pos, uint32_t head, DeviceStatus *st,
                                              uint32_t where) {
    const uint32_t lp = ring_slot(uint32_t(pos) / kv.page_size, kv.ring);
    const int32_t page = pos >= 0 && lp < kv.max_pages ? kv.page_table[size_t(seq) * kv.max_pages + lp] : -1;
    if (page < 0 || uint32_t(page) >= kv.n_pages) {
        report(st, OPURE_ERR_DEVICE_BOUNDS, where, pos < 0 ? uint32_t(pos) : uint32_t(page));
        return nullptr;
    }
    const uint32_t groups = kv.page_size / kKv4Group;
    return kv.pool + ((size_t(page) * kv.n_kv + head) * groups + uint32_t(pos) % kv.page_size / kKv4Group) * kv4_group_bytes(kv.head_dim);
}

// Two E4M3 bytes -> their values as an fp16 pair (exact; 0x7f and 0xff are NaN).
__device__ __forceinline__ uint32_t kv4_scale_pair(uint32_t bytes) {
    uint32_t r;
    asm("{\n .reg .b16 a, b;\n mov.b32 {a, b}, %1;\n cvt.rn.f16x2.e4m3x2 %0, a;\n}" : "=r"(r) : "r"(bytes));
    return r;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// ---- host checks -------------------------------------------------------------------------
inline bool kv4_power_of_two(float s) {
    int e = 0;
    return s == 0.f || (std::isfinite(s) && std::frexp(s, &e) == 0.5f && e >= -59 && e <= 61);
}
inline bool kv4_shape(uint32_t n_kv, uint32_t hd, uint32_t page) {
    return n_kv != 0 && n_kv <= 65535 && (hd == 64 || hd == 128) && (page == 16 || page == 32 || page == 64 || page == 128);
}
inline opure_status kv4_check(const opure_kv4_layout &kv) {
    if (!kv.pool || !kv.page_table || !kv.n_pages || !kv.max_pages || !kv.n_kv || !kv.head_dim || !kv.page_size ||
        kv.ring > kv.max_pages || reinterpret_cast<uintptr_t>(kv.pool) % 16 || !kv4_power_of_two(kv.k_scale) ||
        !kv4_power_of_two(kv.v_scale))
        return OPURE_ERR_INVALID_ARG;
    return kv4_shape(kv.n_kv, kv.head_dim, kv.page_size) ? OPURE_OK : OPURE_ERR_UNSUPPORTED;
}

}  // namespace opure
