// kv4_prompt.cu -- attention over the 4-bit paged KV cache for many queries per sequence (prompts), on
// tcgen05.
//
// One CTA owns (entry, 256 rows, kv head, key split); a row is a (query, query head of the group)
// pair, so all rows share the kv head's keys and values. Per tile of 64 keys:
//   warps 8-11   convert the tile's codes from memory to fp16 operands in shared memory (scales
//                included, exact): K rows as they are, V transposed, both in 128-byte swizzled rows; the
//                codes of the next tile are loaded meanwhile
//   warps 12, 13 issue S = Q K^T for the two halves of 128 rows, two tiles ahead of P V
//   warps 0-3,   a thread per row: maximum, exponentials, row sum; P goes back to tensor memory over S, and
//   warps 4-7    every few tiles their P V is added to the row's sums in registers (left to run on in the
//                tensor cores, whose additions cut off, the sums drift)
// S has two buffers a half, so a row's thread finds the next scores ready when it is done with a tile, and
// the other half's thread keeps the exponentials going while it adds. With fp32 queries Q and P are
// pairs of fp16 (hi, lo), two MMAs each, so that products keep 22 bits; with 16-bit types Q is a single fp16
// (exact down to 2^-28 of the row's largest) and P is rounded to it once. A row's queries are scaled by a power
// of two to [2^14, 2^15) first, so that they are held to 2^-39 of the largest at least. The maximum is raised
// only when a score passes it by 2^4.
//
// What bounds it: 16,384 exponentials a tile of 64 keys and 256 rows at 16 a clock, 1,024 clocks; the
// tensor cores need as long for fp32 (two MMAs for one), half for 16-bit types. A tile takes 2,200-2,600 clocks
// (fp32: issue 49%, exponentials and conversions 32%, tensor cores 31% of the time):
// 4096 causal queries of 32 heads of 64 214 us with fp32, 171 with fp16; of 128 318 with fp32, 241 with bf16.
// (mma.sync took 980 us for the first of these, tiles of 128 keys with one score buffer a half 341.)
#include <type_traits>

#include "kv4_attention.cuh"
#include "tcgen05.cuh"

namespace opure {
namespace {

constexpr uint32_t kSoftmaxWarps = 8, kThreads = 512, kHalf = 128;
constexpr uint32_t kMmaWarp = 12;
constexpr uint32_t kTmemCols = 512;
// Log2 units by which a score may pass the running maximum, and by which probabilities are larger than
// relative to it: together 2^15, what fp16 has. So a probability has all its bits down to 2^-25 of the
// maximum's, and is off by 2^-36 at most below (2^-25 if the maximum's were 1: keys of 2^-24.5 and less, thousands
// of them beside one of weight 1, counted 1.4 times, or not at all).
constexpr float kRaise = 4.f, kLift = 11.f;
constexpr uint32_t KT = 64;          // keys of a tile
constexpr uint32_t kGroups = KT / kKv4Group;  // of 16 positions, one to each converting warp

template <typename T, int HD>
struct Shape {
    static constexpr bool kPair = sizeof(T) == 4;       // queries and probabilities as fp16 pairs
    static constexpr uint32_t kPanels = HD / 64;
    // Q as the A operand: with head_dim 64 in tensor memory (from shared memory, an MMA of 64 columns
    // would read three bytes of operands for two that the tensor cores can take), else in shared.
    static constexpr bool kQTmem = HD == 64;
    static constexpr uint32_t kQPart = kHalf * HD * 2;  // bytes of one half's Q, hi or lo
    static constexpr uint32_t kQBytes = kQTmem ? 0 : 2 * kQPart * (kPair ? 2 : 1);
    static constexpr uint32_t kTile = KT * HD * 2;      // bytes of K, or of V
    static constexpr uint32_t kStages = HD == 128 && kPair ? 3 : 4;
    static constexpr uint32_t kSmem = kQBytes + kStages * 2 * kTile + 1024;
    // Registers of a row's thread, and 256 less these for the others (65536 in all). With head_dim 64
    // they hold a tile's scores between the maximum and the exponentials; with 128 these are read twice.
    static constexpr int kSoftmaxRegs = HD == 64 ? 200 : 192;
    static constexpr uint32_t kChunk = HD == 64 ? 64 : 16;  // scores that a thread holds
    // Tiles whose products add up in tensor memory: a sum of 8 steps of 16 keys is cut off by 2^-22 of
    // itself at most, of 32 steps by 2^-20, less than one of fp16's roundings of P.
    static constexpr uint32_t kRun = kPair ? 2 : 8;
    // Tensor memory: S [half][buffer], O [half], Q [half][hi, lo].
    static constexpr uint32_t kOCol = 4 * KT, kQCol = kOCol + 2 * HD;
    static_assert(kOCol + 2 * HD + (kQTmem ? 2 * HD : 0) <= kTmemCols, "tensor memory");
};

__device__ __forceinline__ void mma_ss(bool one, uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 e, %5, 0;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(da), "l"(db), "r"(idesc), "r"(accumulate), "r"(uint32_t(one))
        : "memory");
}
// A from tensor memory: row i in lane i, two fp16 of neighbouring k in a column.
__device__ __forceinline__ void mma_ts(bool one, uint32_t d, uint32_t a, uint64_t db, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n .reg .pred p, e;\n setp.ne.b32 p, %4, 0;\n setp.ne.b32 e, %5, 0;\n"
        " @e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
        "r"(a), "l"(db), "r"(idesc), "r"(accumulate), "r"(uint32_t(one))
        : "memory");
}
__device__ __forceinline__ void ld_cols(uint32_t taddr, uint32_t (&r)[64]) {
    tc::ld32(taddr, *reinterpret_cast<uint32_t(*)[32]>(r));
    tc::ld32(taddr + 32, *reinterpret_cast<uint32_t(*)[32]>(r + 32));
}
__device__ __forceinline__ void ld_cols(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void st_cols(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void st_cols(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Column of P V that holds dimension d (counted within a panel of 64): V's rows are ordered so that the
// lanes that write them do not meet in a bank.
__host__ __device__ constexpr uint32_t column_of(uint32_t d) { return d / 64 * 64 + d % 8 * 8 + d % 64 / 8; }

template <typename T, int HD>
__global__ void __launch_bounds__(kThreads, 1) prompt_kernel(Kv4AttnParams p) {
    using S = Shape<T, HD>;
    constexpr uint32_t kPanels = S::kPanels, kStages = S::kStages;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages], s_full[2][2], p_full[2][2], o_full[2][2], done;
    __shared__ uint32_t tmem_base;
    __shared__ __align__(16) uint16_t bad_values[kStages][HD / 16][kGroups];  // positions whose block is NaN, 16 to a group
    __shared__ uint32_t ticket;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;

    grid_dependency_wait();
    grid_dependents_launch();

    // The unit: later rows, which see more keys, first.
    const uint32_t head = blockIdx.x % p.kv.n_kv, entry = blockIdx.x / p.kv.n_kv % p.n;
    const uint32_t tile = p.row_tiles - 1 - blockIdx.x / p.kv.n_kv / p.n;
    const uint32_t unit = (entry * p.row_tiles + tile) * p.kv.n_kv + head;
    const uint32_t row0 = p.q_begin ? uint32_t(p.q_begin[entry]) : entry * p.n_q;
    uint32_t queries = p.q_begin ? uint32_t(p.q_begin[entry + 1]) - row0 : p.n_q;
    if (queries > p.n_q || row0 > p.n_rows || queries > p.n_rows - row0) {
        if (tile == 0 && head == 0 && blockIdx.y == 0 && threadIdx.x == 0) report(p.st, OPURE_ERR_DEVICE_BOUNDS, 92, queries);
        queries = int32_t(queries) < 0 || row0 > p.n_rows ? 0u : min(queries, min(p.n_q, p.n_rows - row0));
    }
    const uint32_t first = tile * kKv4PromptRows, total = queries * p.group;
    if (first >= total) return;
    const int32_t seq = p.seq[entry], len0 = p.seq_len[entry];
    const uint32_t P = p.kv.page_size;
    const uint32_t half_rows[2] = {min(kHalf, total - first), total - first > kHalf ? min(kHalf, total - first - kHalf) : 0u};
    auto query_of = [&](uint32_t r) { return (first + r) / p.group; };  // r counts the unit's rows
    auto keys_end = [&](uint32_t j) { return seq < 0 ? 0u : uint32_t(max(len0 + int32_t(j), 0)); };
    auto keys_begin = [&](uint32_t j) { return window_begin(len0 + int32_t(j) - 1, P, p.kv.ring); };
    const uint32_t last_row = half_rows[0] + half_rows[1] - 1;
    const uint32_t end = keys_end(query_of(last_row)), begin = keys_begin(query_of(0));
    const uint32_t s_first = begin / p.split_tokens;
    uint32_t s_last = end ? (end - 1) / p.split_tokens : 0u;
    if (s_last >= p.n_splits) {
        if (blockIdx.y == 0 && threadIdx.x == 0) report(p.st, OPURE_ERR_DEVICE_BOUNDS, 93, end);
        s_last = p.n_splits - 1;
    }
    const uint32_t split = blockIdx.y;
    if (end > begin ? split < s_first || split > s_last : split != 0u) return;
    const uint32_t splits = end > begin ? s_last - s_first + 1 : 1u;
    // Keys of this CTA, in tiles of KT from tile0 on; each half takes part in tiles [from, upto).
    const uint32_t k_begin = max(begin, split * p.split_tokens), k_end = min(end, (split + 1) * p.split_tokens);
    const uint32_t tile0 = k_begin / KT, n_tiles = k_end > k_begin ? (k_end + KT - 1) / KT - tile0 : 0u;
    uint32_t from[2], upto[2], all_begin[2], all_end[2];  // all_*: keys that every row of the half sees
#pragma unroll
    for (uint32_t t = 0; t < 2; ++t) {
        from[t] = upto[t] = 0;
        all_begin[t] = 0;
        all_end[t] = ~0u;
        if (half_rows[t]) {
            const uint32_t ja = query_of(t * kHalf), jb = query_of(t * kHalf + half_rows[t] - 1);
            const uint32_t a = max(keys_begin(ja), k_begin), b = min(keys_end(jb), k_end);
            all_begin[t] = keys_begin(jb);
            all_end[t] = keys_end(ja);
            if (b > a) {
                from[t] = a / KT - tile0;
                upto[t] = (b + KT - 1) / KT - tile0;
            }
        }
    }
    // Whether every row that works on tile i sees all of it, in one half or in both.
    auto half_sees = [&](uint32_t t, uint32_t i) {
        const uint32_t t0 = (tile0 + i) * KT;
        return t0 >= max(t ? all_begin[1] : all_begin[0], k_begin) && t0 + KT <= min(t ? all_end[1] : all_end[0], k_end);
    };
    auto all_see = [&](uint32_t i) {
        return (i < from[0] || i >= upto[0] || half_sees(0, i)) && (i < from[1] || i >= upto[1] || half_sees(1, i));
    };

    uint8_t *smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    uint8_t *q_smem = smem;                    // [half][part][panel][128 rows][128 bytes]
    uint8_t *kv_smem = smem + S::kQBytes;      // [stage][K | V]: K [panel][KT rows], V [KT / 64][HD rows]
    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < kStages; ++s) {
            mbar_init(&k_full[s], 128);
            mbar_init(&k_empty[s], 2);
            mbar_init(&v_full[s], 128);
            mbar_init(&v_empty[s], 2);
        }
        for (uint32_t t = 0; t < 2; ++t) {
            mbar_init(&s_full[t][0], 1);
            mbar_init(&s_full[t][1], 1);
            mbar_init(&o_full[t][0], 1);
            mbar_init(&o_full[t][1], 1);
            mbar_init(&p_full[t][0], kHalf);
            mbar_init(&p_full[t][1], kHalf);
        }
        mbar_init(&done, 2);
    }
    if (warp == kMmaWarp) tc::alloc(&tmem_base, kTmemCols);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_base;

    // Queries to tensor or shared memory: a thread per row.
    float factor = 0.f;
    if (warp < kSoftmaxWarps) {
        const uint32_t half = warp / 4, r = threadIdx.x % kHalf;
        const bool live = r < (half ? half_rows[1] : half_rows[0]);
        const uint32_t q = first + half * kHalf + (live ? r : 0u);
        const T *qp = static_cast<const T *>(p.q) + size_t(row0 + q / p.group) * p.q_stride + (size_t(head) * p.group + q % p.group) * HD;
        const bool aligned = reinterpret_cast<uintptr_t>(qp) % 16 == 0;
        auto load = [&](uint32_t d, float (&v)[8]) {
            if (live && aligned)
                load8(qp + d, v);
            else
                load8_part(qp + d, live ? 8u : 0u, v);
        };
        float m = 0.f;
#pragma unroll 4
        for (uint32_t d = 0; d < HD; d += 8) {
            float v[8];
            load(d, v);
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) m = fmaxf(m, fabsf(v[k]));
        }
        // To [2^14, 2^15), times 2^(d - 127), and back in the factor (rows whose largest is below 2^-112 come
        // out smaller, an infinity or NaN stays one). The factor is not negative: a negative scale goes to the
        // queries.
        const uint32_t e = __float_as_uint(m) >> 23, d = min(268u - e, 253u);
        const float down = __uint_as_float(d << 23) * (p.factor < 0.f ? -1.f : 1.f);
        factor = __uint_as_float((254u - d) << 23) * fabsf(p.factor);
        uint8_t *dst = q_smem + half * (S::kQBytes / 2) + r * 128;
        const uint32_t q_col = tmem + ((warp % 4 * 32) << 16) + S::kQCol + half * HD;
#pragma unroll 2
        for (uint32_t d = 0; d < HD; d += 16) {
            uint32_t hi[8], lo[8];
            float v[16];
            load(d, *reinterpret_cast<float(*)[8]>(v));
            load(d + 8, *reinterpret_cast<float(*)[8]>(v + 8));
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) {
                const float a = v[2 * j] * down, b = v[2 * j + 1] * down;
                hi[j] = pack_half2(a, b);
                const float2 h = h2f2(hi[j]);
                lo[j] = pack_half2(a - h.x, b - h.y);
            }
            if constexpr (S::kQTmem) {
                st_cols(q_col + d / 2, hi);
                if (S::kPair) st_cols(q_col + HD / 2 + d / 2, lo);
            } else {
#pragma unroll
                for (uint32_t j = 0; j < 2; ++j) {
                    uint8_t *at = dst + d / 64 * (kHalf * 128) + ((d % 64 / 8 + j) ^ (r & 7u)) * 16;
                    *reinterpret_cast<uint4 *>(at) = make_uint4(hi[4 * j], hi[4 * j + 1], hi[4 * j + 2], hi[4 * j + 3]);
                    if (S::kPair) *reinterpret_cast<uint4 *>(at + S::kQPart) = make_uint4(lo[4 * j], lo[4 * j + 1], lo[4 * j + 2], lo[4 * j + 3]);
                }
            }
        }
        if constexpr (S::kQTmem)
            wait_st();
        else
            tc::fence_async_shared();
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();

    if (warp < kSoftmaxWarps) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(S::kSoftmaxRegs));
        const uint32_t half = warp / 4, r = threadIdx.x % kHalf;
        const uint32_t lanes = (warp % 4 * 32) << 16;
        const uint32_t s_base = tmem + lanes + half * 2 * KT, o_col = tmem + lanes + S::kOCol + half * HD;
        const bool live = r < (half ? half_rows[1] : half_rows[0]);
        const uint32_t j = query_of(half * kHalf + (live ? r : 0u));
        const uint32_t see0 = max(keys_begin(j), k_begin), see1 = live ? min(keys_end(j), k_end) : 0u;
        float acc[HD];
#pragma unroll
        for (uint32_t d = 0; d < HD; ++d) acc[d] = 0.f;
        float m = -INFINITY, l = 0.f;
        uint32_t nan_blocks = 0;  // blocks of 16 dimensions with a NaN among the values that this row sees
        bool ok = true;
        auto add_products = [&](float by) {
            constexpr uint32_t kOut = HD == 64 ? 64 : 16;
#pragma unroll
            for (uint32_t d = 0; d < HD; d += kOut) {
                uint32_t o[kOut];
                ld_cols(o_col + d, o);
                tc::wait_ld();
#pragma unroll
                for (uint32_t q = 0; q < kOut; q += 2) {
                    const float2 a = __ffma2_rn(make_float2(__uint_as_float(o[q]), __uint_as_float(o[q + 1])), make_float2(by, by),
                                                make_float2(acc[d + q], acc[d + q + 1]));
                    acc[d + q] = a.x;
                    acc[d + q + 1] = a.y;
                }
            }
        };
        auto rescale_products = [&](float by) {
#pragma unroll 1
            for (uint32_t d = 0; d < HD; d += 16) {
                uint32_t o[16];
                ld_cols(o_col + d, o);
                tc::wait_ld();
#pragma unroll
                for (uint32_t q = 0; q < 16; ++q) o[q] = __float_as_uint(__uint_as_float(o[q]) * by);
                st_cols(o_col + d, o);
            }
            wait_st();
        };
        const uint32_t from_mine = half ? from[1] : from[0], n_mine = (half ? upto[1] : upto[0]) - from_mine;
        for (uint32_t n = 0; n < n_mine; ++n) {
            const uint32_t i = from_mine + n, t0 = (tile0 + i) * KT, st = i % kStages;
            const uint32_t s_col = s_base + (n & 1u) * KT;
            if (!mbar_wait(&s_full[half][n & 1u], n / 2 & 1u)) {
                if (lane == 0) report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 100, blockIdx.x);
                ok = false;
                break;
            }
            tc::fence_after();
            float raised = 1.f;  // what the sums so far are multiplied by
            bool rescale = false;  // those in tensor memory too
            auto step = [&](auto masked) {
                constexpr bool kMasked = decltype(masked)::value;
                constexpr uint32_t CH = S::kChunk, PC = CH < 32 ? CH : 32;  // scores held; of one store of P
                auto seen = [&](uint32_t k) { return t0 + k >= see0 && t0 + k < see1; };
                uint32_t s[CH];
                float top = -INFINITY;
#pragma unroll 1
                for (uint32_t c = 0; c < KT; c += CH) {
                    ld_cols(s_col + c, s);
                    tc::wait_ld();
                    if (kMasked) {
#pragma unroll
                        for (uint32_t q = 0; q < CH; ++q) s[q] = seen(c + q) ? s[q] : 0xff800000u;
                    }
                    float high[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (uint32_t q = 0; q < CH; q += 2)
                        asm("max.f32 %0, %0, %1, %2;" : "+f"(high[q / 2 % 4]) : "f"(__uint_as_float(s[q])), "f"(__uint_as_float(s[q + 1])));
                    top = fmaxf(fmaxf(top, high[0]), fmaxf(fmaxf(high[1], high[2]), high[3]));
                }
                top = top == -INFINITY ? top : top * factor;
                if (__any_sync(0xffffffffu, top > m + kRaise)) {
                    const float up = fmaxf(m, top);
                    raised = up == -INFINITY ? 1.f : fast_exp2(m - up);
                    m = up;
                    l *= raised;
#pragma unroll
                    for (uint32_t d = 0; d < HD; ++d) acc[d] *= raised;
                    rescale = true;
                }
                const float base = m == -INFINITY ? 0.f : m - kLift;
#pragma unroll 1
                for (uint32_t c = 0; c < KT; c += CH) {
                    if (CH < KT) {
                        ld_cols(s_col + c, s);
                        tc::wait_ld();
                        if (kMasked) {
#pragma unroll
                            for (uint32_t q = 0; q < CH; ++q) s[q] = seen(c + q) ? s[q] : 0xff800000u;
                        }
                    }
                    float2 sum = make_float2(0.f, 0.f);
#pragma unroll
                    for (uint32_t c2 = 0; c2 < CH; c2 += PC) {
                        uint32_t hi[PC / 2], lo[PC / 2];
#pragma unroll
                        for (uint32_t q = 0; q < PC; q += 2) {
                            float2 x = __ffma2_rn(make_float2(__uint_as_float(s[c2 + q]), __uint_as_float(s[c2 + q + 1])), make_float2(factor, factor),
                                                  make_float2(-base, -base));
                            if (kMasked) {  // a factor of 0 has made NaN of -inf
                                x.x = s[c2 + q] == 0xff800000u ? -INFINITY : x.x;
                                x.y = s[c2 + q + 1] == 0xff800000u ? -INFINITY : x.y;
                            }
                            const float2 e = make_float2(fast_exp2(x.x), fast_exp2(x.y));
                            sum = __fadd2_rn(sum, e);
                            hi[q / 2] = pack_half2(e.x, e.y);
                            if (S::kPair) {
                                const float2 h = h2f2(hi[q / 2]);
                                const float2 d = __fadd2_rn(e, make_float2(-h.x, -h.y));
                                lo[q / 2] = pack_half2(d.x, d.y);
                            }
                        }
                        // Over the scores that were read: of each PC columns the first half hi, then lo.
                        st_cols(s_col + c + c2, hi);
                        if (S::kPair) st_cols(s_col + c + c2 + PC / 2, lo);
                    }
                    l += sum.x + sum.y;
                }
            };
            if (half_sees(half, i))
                step(std::false_type());
            else
                step(std::true_type());
            wait_st();
            if (!all_see(i)) {
                // NaN values were left out of V where not all rows see them.
                if (!mbar_wait(&v_full[st], i / kStages & 1u)) {
                    if (lane == 0) report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 101, blockIdx.x);
                    ok = false;
                    break;
                }
                const uint4 *w = reinterpret_cast<const uint4 *>(bad_values[st]);
                uint32_t any = 0;
                for (uint32_t q = 0; q < sizeof(bad_values[0]) / 16; ++q) any |= w[q].x | w[q].y | w[q].z | w[q].w;
                if (any)
                    for (uint32_t b = 0; b < HD / 16; ++b)
                        for (uint32_t k = 0; k < KT; ++k)
                            if (bad_values[st][b][k / 16] >> (k % 16) & 1u && t0 + k >= see0 && t0 + k < see1) nan_blocks |= 1u << b;
            }
            // The products so far are needed where a run of tiles ends, or the maximum was raised. (Two
            // barriers in turn: the products of tile n - 3 are done, as the scores of tile n - 1 came after them, so
            // that a wait for tile n - 1 cannot take another of its barrier's phases for it.)
            const bool run_ends = n % S::kRun == 0;
            if (n && (run_ends || rescale)) {
                if (!mbar_wait(&o_full[half][(n - 1) & 1u], (n - 1) / 2 & 1u)) {
                    if (lane == 0) report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 105, blockIdx.x);
                    ok = false;
                    break;
                }
                tc::fence_after();
                if (run_ends)
                    add_products(raised);
                else
                    rescale_products(raised);
            }
            tc::fence_before();
            arrive(&p_full[half][n & 1u]);
        }
        if (ok && n_mine) {
            if (mbar_wait(&o_full[half][(n_mine - 1) & 1u], (n_mine - 1) / 2 & 1u)) {
                tc::fence_after();
                add_products(1.f);
            } else if (lane == 0) {
                report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 102, blockIdx.x);
            }
        }
        if (live) {
            const uint32_t q = first + half * kHalf + r;
            const uint32_t out_row = row0 + q / p.group, out_col = (head * p.group + q % p.group) * HD;
            if (splits == 1) {
                const float inv = p.v_scale / fmaxf(l, 1e-30f);
                T *out = static_cast<T *>(p.out) + size_t(out_row) * p.out_stride + out_col;
                const bool aligned = reinterpret_cast<uintptr_t>(out) % 16 == 0;
#pragma unroll
                for (uint32_t d = 0; d < HD; d += 8) {
                    float v[8];
#pragma unroll
                    for (uint32_t k = 0; k < 8; ++k) v[k] = nan_blocks >> (d / 16) & 1u ? NAN : acc[column_of(d + k)] * inv;
                    if (aligned)
                        store8(out + d, v);
                    else
                        store8_part(out + d, 8, v);
                    if (p.out_packed)
#pragma unroll
                        for (uint32_t k = 0; k < 8; ++k)
                            store_packed(p.out_packed, p.pk_npad, p.n_heads * HD, out_row, out_col + d + k, v[k], p.st, 95);
                }
            } else {
                float *part = p.partials + ((size_t(unit) * p.n_splits + split) * kKv4PromptRows + half * kHalf + r) * (HD + 2);
#pragma unroll
                for (uint32_t d = 0; d < HD; d += 2)
                    *reinterpret_cast<float2 *>(part + d) = nan_blocks >> (d / 16) & 1u ? make_float2(NAN, NAN)
                                                                                         : make_float2(acc[column_of(d)], acc[column_of(d + 1)]);
                *reinterpret_cast<float2 *>(part + HD) = make_float2(m, l);
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(256 - S::kSoftmaxRegs));
        if (warp < kMmaWarp) {
            // Codes to operands, 16 positions a warp and tile.
            const uint32_t w = warp - kSoftmaxWarps, c = lane & 3u, g = lane >> 2;
            const int32_t *table = p.kv.page_table + size_t(max(seq, 0)) * p.kv.max_pages;
            const uint32_t groups_per_page = P / kKv4Group;
            struct Raw {
                uint4 k[kPanels], v[kPanels];
                uint32_t ks[kPanels], vs[kPanels];
            };
            auto position = [&](uint32_t i) { return (tile0 + i) * KT + w * kKv4Group; };
            auto page_of = [&](uint32_t i) -> int32_t {
                const uint32_t t = position(i);
                if (i >= n_tiles || t >= k_end || t + kKv4Group <= k_begin) return -2;
                const uint32_t lp = ring_slot(t / P, p.kv.ring);
                return lp < p.kv.max_pages ? table[lp] : -1;
            };
            auto load = [&](uint32_t i, int32_t page, Raw &raw) {
                const bool good = page >= 0 && uint32_t(page) < p.kv.n_pages;
                if (!good && page != -2 && lane == 0) report(p.st, OPURE_ERR_DEVICE_BOUNDS, 94, uint32_t(page));
                const uint8_t *group = p.kv.pool + ((size_t(good ? page : 0) * p.kv.n_kv + head) * groups_per_page + position(i) % P / kKv4Group) * kv4_group_bytes(HD);
#pragma unroll
                for (uint32_t pn = 0; pn < kPanels; ++pn) {
                    raw.k[pn] = raw.v[pn] = make_uint4(0, 0, 0, 0);
                    raw.ks[pn] = raw.vs[pn] = 0;
                    if (good) {
                        raw.k[pn] = __ldg(reinterpret_cast<const uint4 *>(group + pn * 512) + lane);
                        raw.v[pn] = __ldg(reinterpret_cast<const uint4 *>(group + 8 * HD + pn * 512) + lane);
                        raw.ks[pn] = __ldg(reinterpret_cast<const uint16_t *>(group + 16 * HD + pn * 64) + lane);
                        raw.vs[pn] = __ldg(reinterpret_cast<const uint32_t *>(group + 17 * HD + pn * 64) + g / 2 * 4 + c);
                    }
                }
            };
            Raw raw;
            load(0, page_of(0), raw);
            int32_t page_next = page_of(1);
            bool ok = true;
            for (uint32_t i = 0; i < n_tiles; ++i) {
                const uint32_t st = i % kStages;
                const bool whole = all_see(i);
                uint8_t *ktile = kv_smem + st * 2 * S::kTile, *vtile = ktile + S::kTile;
                if (i >= kStages && !mbar_wait(&k_empty[st], (i / kStages - 1) & 1u)) ok = false;
                if (ok) {
#pragma unroll
                        for (uint32_t pn = 0; pn < kPanels; ++pn) {
                            const uint32_t sp = kv4_scale_pair(raw.ks[pn]);
#pragma unroll
                            for (uint32_t u = 0; u < 2; ++u) {
                                const uint32_t s = u ? __byte_perm(sp, sp, 0x3232) : __byte_perm(sp, sp, 0x1010);
                                uint32_t h[8];
                                mx_unpack_fp4(u ? raw.k[pn].z : raw.k[pn].x, *reinterpret_cast<uint32_t(*)[4]>(h));
                                mx_unpack_fp4(u ? raw.k[pn].w : raw.k[pn].y, *reinterpret_cast<uint32_t(*)[4]>(h + 4));
#pragma unroll
                                for (uint32_t q = 0; q < 8; ++q) h[q] = hmul2(h[q], s);
                                uint8_t *row = ktile + pn * (KT * 128) + (w * 16 + u * 8 + g) * 128;
                                *reinterpret_cast<uint4 *>(row + ((2 * c) ^ g) * 16) = make_uint4(h[0], h[1], h[2], h[3]);
                                *reinterpret_cast<uint4 *>(row + ((2 * c + 1) ^ g) * 16) = make_uint4(h[4], h[5], h[6], h[7]);
                            }
                        }
                    tc::fence_async_shared();
                    arrive(&k_full[st]);
                    if (i >= kStages && !mbar_wait(&v_empty[st], (i / kStages - 1) & 1u)) ok = false;
                }
                if (!ok) {
                    if (lane == 0) report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 103, blockIdx.x);
                    break;
                }
#pragma unroll
                    for (uint32_t pn = 0; pn < kPanels; ++pn) {
                        uint32_t sv = raw.vs[pn];
                        if (!whole) {
                            // Positions that no row sees may hold anything; NaN blocks are named to the rows.
                            const uint32_t t = position(i) + 2 * c;
                            uint32_t bad = 0;
#pragma unroll
                            for (uint32_t b = 0; b < 4; ++b) {
                                const uint32_t at = b % 2 + 8 * (b / 2);
                                const bool in = t + at >= k_begin && t + at < k_end;
                                const bool nan = (sv >> (8 * b) & 0x7fu) == 0x7fu;
                                if (in && nan) bad |= 1u << (2 * c + at);
                                if (!in || nan) sv &= ~(0xffu << (8 * b));
                            }
                            bad |= __shfl_xor_sync(0xffffffffu, bad, 1);
                            bad |= __shfl_xor_sync(0xffffffffu, bad, 2);
                            if (c == 0 && g % 2 == 0) bad_values[st][pn * 4 + g / 2][w] = uint16_t(bad);
                        }
                        const uint32_t s01 = kv4_scale_pair(sv), s23 = kv4_scale_pair(sv >> 16), low = 0x0f0f0f0fu;
                        const uint4 v = raw.v[pn];
                        // A row per dimension, 8 (d % 8) + d / 8; two positions a word.
                        const uint32_t chunk = w * 2;
                        uint8_t *base = vtile + (pn * 64 + g) * 128 + c * 4;
                        auto put = [&](uint32_t word, uint32_t odd, uint32_t s, uint32_t ch) {
                            uint32_t h[4];
                            mx_unpack_fp4(word, h);
#pragma unroll
                            for (uint32_t q = 0; q < 4; ++q)
                                *reinterpret_cast<uint32_t *>(base + (2 * q + odd) * 8 * 128 + (ch ^ g) * 16) = hmul2(h[q], s);
                        };
                        put((v.x & low) | (v.y << 4 & ~low), 0, s01, chunk);
                        put((v.x >> 4 & low) | (v.y & ~low), 1, s01, chunk);
                        put((v.z & low) | (v.w << 4 & ~low), 0, s23, chunk + 1);
                        put((v.z >> 4 & low) | (v.w & ~low), 1, s23, chunk + 1);
                    }
                tc::fence_async_shared();
                arrive(&v_full[st]);
                load(i + 1, page_next, raw);
                page_next = page_of(i + 2);
            }
        } else if (warp < kMmaWarp + 2) {
            const uint32_t t = warp - kMmaWarp;  // the half
            const uint32_t from_t = t ? from[1] : from[0], upto_t = t ? upto[1] : upto[0];
            const bool one = tc::elect();
            constexpr uint32_t idesc_s = (1u << 4) | ((KT >> 3) << 17) | ((kHalf >> 4) << 24);
            constexpr uint32_t idesc_o = (1u << 4) | ((uint32_t(HD) >> 3) << 17) | ((kHalf >> 4) << 24);
            bool ok = true;
            auto wait = [&](uint64_t *bar, uint32_t phase) {
                if (ok && !mbar_wait(bar, phase)) {
                    if (lane == 0) report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 104, blockIdx.x);
                    ok = false;
                }
            };
            // Tile i's scores, and the products of tile i - 2, over whose P the scores go. A stage is free after one
            // arrival of each half's warp, so a warp whose half has no part in a tile (rows that are not there, keys
            // that they do not see) waits for the tile all the same: its arrivals for two tiles would else fill
            // one phase, and the stage be written again under the other half.
            for (uint32_t i = 0; i < n_tiles + 2; ++i) {
                const uint32_t n = i - from_t;
                const uint32_t s_col = tmem + (t * 2 + (n & 1u)) * KT;
                if (i >= 2) wait(&v_full[(i - 2) % kStages], (i - 2) / kStages & 1u);
                if (i >= from_t + 2 && i < upto_t + 2 && upto_t > from_t) {
                    const uint32_t st = (i - 2) % kStages, v = smem_addr(kv_smem + st * 2 * S::kTile + S::kTile);
                    wait(&p_full[t][n & 1u], (n - 2) / 2 & 1u);
                    if (!ok) break;
                    tc::fence_after();
                    constexpr uint32_t PC = S::kChunk < 32 ? S::kChunk : 32;
                    // lo first: its sums are too small to cut much off.
#pragma unroll
                    for (uint32_t part = S::kPair ? 0 : 1; part < 2; ++part)
#pragma unroll
                        for (uint32_t k = 0; k < KT / 16; ++k) {
                            const uint32_t col = k * 16 / PC * PC + k * 16 % PC / 2 + (part == 0 ? PC / 2 : 0u);
                            mma_ts(one, tmem + S::kOCol + t * HD, s_col + col, tc::desc_sw128(v + k * 32), idesc_o,
                                   part != (S::kPair ? 0 : 1) || k != 0 || (n - 2) % S::kRun != 0);
                        }
                    tc::commit(one, &o_full[t][n & 1u]);
                }
                if (!ok) break;
                if (i >= 2) tc::commit(one, &v_empty[(i - 2) % kStages]);
                if (i < n_tiles) wait(&k_full[i % kStages], i / kStages & 1u);
                if (!ok) break;
                if (i >= from_t && i < upto_t) {
                    const uint32_t st = i % kStages, kt = smem_addr(kv_smem + st * 2 * S::kTile);
                    tc::fence_after();
#pragma unroll
                    for (uint32_t part = 0; part < (S::kPair ? 2 : 1); ++part) {
                        const uint32_t which = S::kPair ? 1 - part : 0;
#pragma unroll
                        for (uint32_t k = 0; k < HD / 16; ++k) {
                            const uint64_t db = tc::desc_sw128(kt + k / 4 * (KT * 128) + k % 4 * 32);
                            if constexpr (S::kQTmem)
                                mma_ts(one, s_col, tmem + S::kQCol + t * HD + which * (HD / 2) + k * 8, db, idesc_s, part != 0 || k != 0);
                            else
                                mma_ss(one, s_col, tc::desc_sw128(smem_addr(q_smem) + t * (S::kQBytes / 2) + which * S::kQPart + k / 4 * (kHalf * 128) + k % 4 * 32),
                                       db, idesc_s, part != 0 || k != 0);
                        }
                    }
                    tc::commit(one, &s_full[t][n & 1u]);
                }
                if (i < n_tiles) tc::commit(one, &k_empty[i % kStages]);
            }
            // Nothing may be in flight when the tensor memory is given back.
            tc::commit(one, &done);
            (void)mbar_wait(&done, 0);
        }
    }
    tc::fence_before();
    __syncthreads();
    if (warp == kMmaWarp) tc::dealloc(tmem, kTmemCols);
    if (splits == 1) {
        if (p.out_packed) asm volatile("fence.proxy.async.global;" ::: "memory");  // read by TMA next
        return;
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) ticket = atomicAdd(p.counters + unit, 1u);
    __syncthreads();
    if (ticket != splits - 1) return;
    __threadfence();
    const float *parts = p.partials + (size_t(unit) * p.n_splits + s_first) * kKv4PromptRows * (HD + 2);
    for (uint32_t x = threadIdx.x; x < (last_row + 1) * HD; x += kThreads) {
        const uint32_t r = x / HD, d = x % HD;
        float m = -INFINITY;
#pragma unroll 4
        for (uint32_t sp = 0; sp < splits; ++sp) m = fmaxf(m, __ldcg(parts + (size_t(sp) * kKv4PromptRows + r) * (HD + 2) + HD));
        float a = 0.f, l = 0.f;
#pragma unroll 4
        for (uint32_t sp = 0; sp < splits; ++sp) {
            const float *pp = parts + (size_t(sp) * kKv4PromptRows + r) * (HD + 2);
            const float ms = __ldcg(pp + HD), f = ms == -INFINITY ? 1.f : fast_exp2(ms - m);
            a += __ldcg(pp + d) * f;
            l += __ldcg(pp + HD + 1) * f;
        }
        const uint32_t q = first + r;
        kv4_store<T>(p, row0 + q / p.group, (head * p.group + q % p.group) * HD + d, a / fmaxf(l, 1e-30f) * p.v_scale);
    }
    if (p.out_packed) asm volatile("fence.proxy.async.global;" ::: "memory");
    if (threadIdx.x == 0) p.counters[unit] = 0u;
}

}  // namespace

opure_status kv4_prompt_launch(opure_ctx *ctx, const Kv4AttnParams &p, uint32_t type, uint32_t units) {
    return with_type(type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto k, uint32_t smem) -> opure_status {
            OPURE_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
            return launch(ctx, k, dim3(units, p.n_splits), dim3(kThreads), smem, true, p);
        };
        return p.kv.head_dim == 64 ? go(prompt_kernel<T, 64>, Shape<T, 64>::kSmem) : go(prompt_kernel<T, 128>, Shape<T, 128>::kSmem);
    });
}

}  // namespace opure
