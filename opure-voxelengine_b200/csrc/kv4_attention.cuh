// kv4_attention.cuh -- what the two attention kernels over the 4-bit cache share: kv4_attention.cu (a few
// rows per sequence, mma.sync) and kv4_prompt.cu (many rows, tcgen05).
#pragma once

#include "attn_core.cuh"
#include "kv4.cuh"
#include "tma.cuh"

namespace opure {

struct Kv4AttnParams {
    const void *q;
    void *out;
    size_t q_stride, out_stride;
    const int32_t *seq, *seq_len, *q_begin;
    uint32_t n, n_rows, n_q, n_heads, group;
    uint32_t row_tiles;
    float factor;            // scale * log2(e) * k_scale
    float v_scale;
    uint32_t split_tokens, n_splits;
    uint32_t *counters;      // [unit], at the scratch's start
    float *partials;         // [unit][split][row of the tile][HD + 2]
    opure_kv4_layout kv;
    DeviceStatus *st;
    __half *out_packed;
    uint32_t pk_npad;
};

template <typename T>
__device__ __forceinline__ void kv4_store(const Kv4AttnParams &p, uint32_t row, uint32_t i, float v) {
    static_cast<T *>(p.out)[size_t(row) * p.out_stride + i] = from_f32<T>(v);
    if (p.out_packed) store_packed(p.out_packed, p.pk_npad, p.n_heads * p.kv.head_dim, row, i, v, p.st, 95);
}

// kv4_prompt.cu: keys in multiples of this per split, rows of a unit, and the launch.
constexpr uint32_t kKv4PromptKeys = 128, kKv4PromptRows = 256;
opure_status kv4_prompt_launch(opure_ctx *ctx, const Kv4AttnParams &p, uint32_t type, uint32_t units);

}  // namespace opure
