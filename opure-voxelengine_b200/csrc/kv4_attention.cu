// kv4_attention.cu -- attention over the 4-bit paged KV cache for a few queries per sequence: one
// token (decode), or the drafted tokens of a verify step.
//
// One CTA owns (entry, tile of rows, kv head, key split); a row is a (query, query head of the group)
// pair, and all rows of the tile share one read of the keys and values. The products run on
// mma.m16n8k16 with the cache on the 16-row side, as S^T = K Q^T and O^T = V^T P^T: four rows fill
// the 8 columns, since a row takes two, the fp16 pair (hi, lo) of its query or probability, and
// products so keep 22 bits. Groups of 16 positions are stored in the order in which lanes hold these
// operands, so a lane reads 16 bytes of key codes and 16 of value codes per panel of 64 columns and
// converts them in registers: cvt of two codes, and one multiplication by the blocks' scales
// (exact in fp16). Score tiles come out with positions across lanes; movmatrix turns the
// probabilities into the second product's operand.
//
// Four warps take chunks of 64 positions in turn from rings of shared-memory stages, one for each,
// that a fifth fills by bulk copies: no barrier between warps until they merge their states. The running
// maximum is raised only when a score passes it by 2^8 (probabilities stay below 2^8, the sums in fp32).
//
// What bounds it: neither issue nor memory alone. Some 366 instructions a warp for 32 positions, most of them
// conversions, take 67% of the issue slots with DRAM at 47%; the rest is waiting, with 16 working warps an SM.
// 64 sequences of 32768 keys over 3 kv heads 125 us (3.6 TB/s), of 4096 over 32 heads 152 us (4.0 TB/s); one
// sequence of 4000 8 us, which is the latency of a split and of joining the splits.
#include <algorithm>

#include "kv4_attention.cuh"

namespace opure {
namespace {

constexpr uint32_t kWarps = 4;
constexpr uint32_t kChunk = 64;      // positions per stage
constexpr uint32_t kChunkGroups = kChunk / kKv4Group;
constexpr uint32_t kThreads = (kWarps + 1) * 32;
// Stages of a warp's ring and CTAs of an SM: as many of these as registers allow, the rest of shared
// memory in stages (about 200 KB of copies under way in an SM).
template <int HD, int NT>
constexpr int kCtasPerSm = HD == 64 && NT == 1 ? 4 : 2;
template <int HD, int NT>
constexpr uint32_t kStages = HD == 64 && NT == 2 ? 6 : 3;
template <int HD>
constexpr uint32_t kStageBytes = kChunkGroups * kv4_group_bytes(HD);
template <int HD, int NT>
constexpr uint32_t kRowsSmem = kWarps * kStages<HD, NT> * kStageBytes<HD>;
constexpr uint32_t kMaxSplits = 64;
constexpr float kRaise = 8.f;        // log2 units by which a score may pass the running maximum

__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16816_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {  // from 0
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// v as fp16 pair: hi in the low half, (v - hi) 2^11 in the high half.
__device__ __forceinline__ uint32_t split_pair(float v) {
    const __half hi = __float2half_rn(v);
    const __half lo = __float2half_rn((v - __half2float(hi)) * 2048.f);
    return uint32_t(__half_as_ushort(hi)) | uint32_t(__half_as_ushort(lo)) << 16;
}
__device__ __forceinline__ uint4 lds128_at(uint32_t a) {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "r"(a));
    return r;
}
__device__ __forceinline__ uint32_t lds32_at(uint32_t a) {
    uint32_t r;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(r) : "r"(a));
    return r;
}
__device__ __forceinline__ uint32_t lds16_at(uint32_t a) {
    unsigned short r;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(r) : "r"(a));
    return r;
}

template <typename T, int HD, int NT>
__global__ void __launch_bounds__(kThreads, kCtasPerSm<HD, NT>) rows_kernel(Kv4AttnParams p) {
    constexpr uint32_t kRows = 4 * NT, kPanels = HD / 64, S = kStages<HD, NT>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ __align__(8) uint64_t full[kWarps][S], empty[kWarps][S];
    __shared__ uint32_t have[kWarps][S];  // groups of the stage that hold positions of this split
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u, c = lane & 3u, g = lane >> 2;
    const uint32_t unit = blockIdx.x, head = unit % p.kv.n_kv, tile = unit / p.kv.n_kv % p.row_tiles,
                   entry = unit / p.kv.n_kv / p.row_tiles;
    if (warp < kWarps && lane < S) {
        mbar_init(&full[warp][lane], 1);
        mbar_init(&empty[warp][lane], 1);
    }
    __syncthreads();
    grid_dependency_wait();
    grid_dependents_launch();

    // This tile's rows: row r is query (first + r) / group of the entry, query head (first + r) % group.
    const uint32_t row0 = p.q_begin ? uint32_t(p.q_begin[entry]) : entry * p.n_q;
    uint32_t queries = p.q_begin ? uint32_t(p.q_begin[entry + 1]) - row0 : p.n_q;
    if (queries > p.n_q || row0 > p.n_rows || queries > p.n_rows - row0) {
        if (tile == 0 && head == 0 && blockIdx.y == 0 && threadIdx.x == 0) report(p.st, OPURE_ERR_DEVICE_BOUNDS, 92, queries);
        queries = min(int32_t(queries) < 0 || row0 > p.n_rows ? 0u : queries, min(p.n_q, row0 > p.n_rows ? 0u : p.n_rows - row0));
    }
    const uint32_t first = tile * kRows, total = queries * p.group;
    if (first >= total) return;
    const uint32_t rows = min(kRows, total - first), j0 = first / p.group, j1 = (first + rows - 1) / p.group;
    const int32_t seq = p.seq[entry], len0 = p.seq_len[entry];
    const uint32_t P = p.kv.page_size;
    // Keys that any row sees: [begin, end); that all rows see: [all_begin, all_end).
    const uint32_t end = seq < 0 ? 0u : uint32_t(max(len0 + int32_t(j1), 0)), all_end = uint32_t(max(len0 + int32_t(j0), 0));
    const uint32_t begin = window_begin(len0 + int32_t(j0) - 1, P, p.kv.ring), all_begin = window_begin(len0 + int32_t(j1) - 1, P, p.kv.ring);
    const uint32_t s_first = begin / p.split_tokens;
    uint32_t s_last = end ? (end - 1) / p.split_tokens : 0u;
    if (s_last >= p.n_splits) {  // a caller that understated max_ctx
        if (blockIdx.y == 0 && threadIdx.x == 0) report(p.st, OPURE_ERR_DEVICE_BOUNDS, 93, end);
        s_last = p.n_splits - 1;
    }
    const uint32_t split = blockIdx.y;
    if (end > begin ? split < s_first || split > s_last : split != 0u) return;
    const uint32_t t_begin = max(begin, split * p.split_tokens), t_end = min(end, (split + 1) * p.split_tokens);
    const uint32_t chunk0 = t_begin / kChunk * kChunk, n_chunks = t_end > t_begin ? (t_end - chunk0 + kChunk - 1) / kChunk : 0u;
    auto share = [&](uint32_t w) { return n_chunks > w ? (n_chunks - w + kWarps - 1) / kWarps : 0u; };  // chunks w, w + kWarps, ..

    if (warp == kWarps) {
        // Copies: four lanes fill a warp's stage, each the groups of its part of the chunk (a page, or as
        // much of one as the chunk covers); `k` counts each warp's chunks.
        const uint32_t w = lane / 4 % kWarps, part = lane & 3u, span = min(P, kChunk), parts = kChunk / span, mine = share(w);
        const bool active = lane < 4 * kWarps && part < parts;
        const int32_t *table = p.kv.page_table + size_t(max(seq, 0)) * p.kv.max_pages;
        auto page_of = [&](uint32_t k) -> int32_t {
            const uint32_t t = chunk0 + (w + k * kWarps) * kChunk + part * span;
            if (!active || k >= mine || t >= t_end || t + span <= t_begin) return -2;  // nothing to copy
            const uint32_t lp = ring_slot(t / P, p.kv.ring);
            return lp < p.kv.max_pages ? table[lp] : -1;
        };
        int32_t page = page_of(0);
        const uint32_t rounds = share(0);
        bool ok = true;
        for (uint32_t k = 0; k < rounds && ok; ++k) {
            const int32_t next_page = page_of(k + 1);
            const uint32_t stage = k % S, t = chunk0 + (w + k * kWarps) * kChunk + part * span;
            uint32_t g0 = 0, g1 = 0;
            if (page != -2) {
                if (page < 0 || uint32_t(page) >= p.kv.n_pages) {
                    report(p.st, OPURE_ERR_DEVICE_BOUNDS, 94, uint32_t(page));
                } else {
                    g0 = t < t_begin ? (t_begin - t) / kKv4Group : 0u;
                    g1 = min(span, t_end - t + kKv4Group - 1) / kKv4Group;
                }
            }
            const uint32_t bytes = (g1 - g0) * kv4_group_bytes(HD);
            uint32_t sum = bytes, bits = ((1u << g1) - (1u << g0)) << (part * (span / kKv4Group));
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            bits |= __shfl_xor_sync(0xffffffffu, bits, 1);
            bits |= __shfl_xor_sync(0xffffffffu, bits, 2);
            const bool there = lane < 4 * kWarps && k < mine;
            if (k >= S) ok = __all_sync(0xffffffffu, !there || mbar_wait(&empty[w][stage], (k / S - 1) & 1u));
            if (!ok) {
                if (lane == 0) report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 106, blockIdx.x);
                break;
            }
            if (there && part == 0) {
                have[w][stage] = bits;
                mbar_expect_tx(&full[w][stage], sum);
            }
            __syncwarp();
            if (there && bytes) {
                const uint8_t *src = p.kv.pool + ((size_t(page) * p.kv.n_kv + head) * (P / kKv4Group) + t % P / kKv4Group + g0) * kv4_group_bytes(HD);
                bulk_load_keep(smem + (w * S + stage) * kStageBytes<HD> + (part * (span / kKv4Group) + g0) * kv4_group_bytes(HD), src, bytes, &full[w][stage]);
            }
            page = next_page;
        }
    }
    const uint32_t mine = warp < kWarps ? share(warp) : 0u;
    uint8_t *ring = smem + size_t(warp) * S * kStageBytes<HD>;

    if (warp < kWarps) {
        // Queries: row r of this lane's column. Each row is scaled by a power of two to [2, 4).
        uint32_t qf[HD / 16][NT][2];
        float factor[NT];
        uint32_t row_end[NT], row_begin[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint32_t col_row = 4 * nt + g / 2;  // the row whose hi (g even) or lo this lane's B column holds
            const bool live = col_row < rows;
            const uint32_t q = first + (live ? col_row : 0u);
            const T *qp = static_cast<const T *>(p.q) + size_t(row0 + q / p.group) * p.q_stride + (size_t(head) * p.group + q % p.group) * HD;
            float v[HD / 4], m = 0.f;
#pragma unroll
            for (uint32_t k = 0; k < HD / 4; ++k) {  // columns 64 panel + 16 c + ..
                v[k] = live ? to_f32(qp[k / 16 * 64 + 16 * c + k % 16]) : 0.f;
                m = fmaxf(m, fabsf(v[k]));
            }
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
            // Times 2^(d - 127), and back in the factor (rows whose largest is below 2^-125 come out smaller,
            // one with an infinity or NaN is NaN).
            const uint32_t e = __float_as_uint(m) >> 23, d = min(255u - e, 253u);
            const float down = __uint_as_float(d << 23), up = __uint_as_float((254u - d) << 23);
#pragma unroll
            for (uint32_t k = 0; k < HD / 4; k += 2) {
                uint32_t pair[2];
#pragma unroll
                for (int u = 0; u < 2; ++u) pair[u] = split_pair(v[k + u] * down);
                qf[k / 4][nt][k / 2 % 2] = __byte_perm(pair[0], pair[1], g & 1u ? 0x7632 : 0x5410);
            }
            // Scores of this lane's accumulators belong to row 4 nt + c, whose columns lanes 8 c .. hold.
            factor[nt] = __shfl_sync(0xffffffffu, up, 8 * c) * p.factor;
            const uint32_t r = first + min(4u * nt + c, rows - 1), j = r / p.group;
            row_end[nt] = uint32_t(max(len0 + int32_t(j), 0));
            row_begin[nt] = window_begin(len0 + int32_t(j) - 1, P, p.kv.ring);
        }

        float acc[HD / 16][NT][2] = {};
        float m_run[NT], l_run[NT];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            m_run[nt] = -INFINITY;
            l_run[nt] = 0.f;
        }
        const uint32_t ring_addr = smem_addr(ring);
        bool ok = true;
        uint32_t k = 0;
        for (; k < mine; ++k) {
            const uint32_t stage = k % S;
            if (!mbar_wait(&full[warp][stage], k / S & 1u)) {
                if (lane == 0) report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 96, blockIdx.x);
                ok = false;
                break;
            }
            const uint32_t groups = have[warp][stage], tok0 = chunk0 + (warp + k * kWarps) * kChunk;
            const bool whole = groups == (1u << kChunkGroups) - 1 && tok0 >= max(all_begin, t_begin) && tok0 + kChunk <= min(all_end, t_end);
            // The tensor cores cut sums off where fp32 would round them: a chunk's sums start from 0 and join
            // the others at its end (left to run on, their bias was 3 times all other errors).
            float part[HD / 16][NT][4];
            bool started = false;
#pragma unroll 1
            for (uint32_t h = 0; h < kChunkGroups / 2; ++h) {
                if (!(groups >> (2 * h) & 3u)) continue;
                const uint32_t base = ring_addr + stage * kStageBytes<HD> + 2 * h * kv4_group_bytes(HD);
                float s[2][NT][4];
#pragma unroll
                for (uint32_t u = 0; u < 2; ++u)
#pragma unroll
                    for (uint32_t pn = 0; pn < kPanels; ++pn) {
                        const uint32_t at = base + u * kv4_group_bytes(HD);
                        const uint4 w = lds128_at(at + pn * 512 + lane * 16);
                        const uint32_t sp = kv4_scale_pair(lds16_at(at + 16 * HD + pn * 64 + lane * 2));
                        const uint32_t s0 = __byte_perm(sp, sp, 0x1010), s1 = __byte_perm(sp, sp, 0x3232);
                        uint32_t k0[8], k1[8];
                        mx_unpack_fp4(w.x, *reinterpret_cast<uint32_t(*)[4]>(k0));
                        mx_unpack_fp4(w.y, *reinterpret_cast<uint32_t(*)[4]>(k0 + 4));
                        mx_unpack_fp4(w.z, *reinterpret_cast<uint32_t(*)[4]>(k1));
                        mx_unpack_fp4(w.w, *reinterpret_cast<uint32_t(*)[4]>(k1 + 4));
#pragma unroll
                        for (uint32_t st = 0; st < 4; ++st) {
                            const uint32_t a[4] = {hmul2(k0[2 * st], s0), hmul2(k1[2 * st], s1), hmul2(k0[2 * st + 1], s0), hmul2(k1[2 * st + 1], s1)};
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                if (pn == 0 && st == 0)
                                    mma16816_first(s[u][nt], a, qf[0][nt][0], qf[0][nt][1]);
                                else
                                    mma16816(s[u][nt], a, qf[pn * 4 + st][nt][0], qf[pn * 4 + st][nt][1]);
                            }
                        }
                    }
                // Scores in log2 units: [u][position g, g + 8].
                float x[2][NT][2], top[NT];
                bool raise = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                    for (uint32_t u = 0; u < 2; ++u)
#pragma unroll
                        for (uint32_t v = 0; v < 2; ++v) {
                            x[u][nt][v] = fmaf(s[u][nt][2 * v + 1], 0x1p-11f, s[u][nt][2 * v]) * factor[nt];
                            if (!whole) {
                                const uint32_t t = tok0 + (2 * h + u) * kKv4Group + v * 8 + g;
                                const bool seen = t >= max(row_begin[nt], t_begin) && t < min(row_end[nt], t_end) && (groups >> (2 * h + u) & 1u);
                                x[u][nt][v] = seen ? x[u][nt][v] : -INFINITY;
                            }
                        }
                    top[nt] = fmaxf(fmaxf(x[0][nt][0], x[0][nt][1]), fmaxf(x[1][nt][0], x[1][nt][1]));
                    raise = raise || top[nt] > m_run[nt] + kRaise;
                }
                if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float m = top[nt];  // over the 8 lanes that share this lane's row
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                        m = fmaxf(m, m_run[nt]);
                        const float f = m == -INFINITY ? 1.f : fast_exp2(m_run[nt] - m);
                        m_run[nt] = m;
                        l_run[nt] *= f;
#pragma unroll
                        for (uint32_t i = 0; i < HD / 16; ++i)
#pragma unroll
                            for (int v = 0; v < 2; ++v) acc[i][nt][v] *= f;
                        if (started)
#pragma unroll
                            for (uint32_t i = 0; i < HD / 16; ++i)
#pragma unroll
                                for (int v = 0; v < 4; ++v) part[i][nt][v] *= f;
                    }
                }
                if (!started)
#pragma unroll
                    for (uint32_t i = 0; i < HD / 16; ++i)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int v = 0; v < 4; ++v) part[i][nt][v] = 0.f;
                started = true;
                uint32_t pf[2][NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    const float m = m_run[nt] == -INFINITY ? 0.f : m_run[nt];
#pragma unroll
                    for (uint32_t u = 0; u < 2; ++u)
#pragma unroll
                        for (uint32_t v = 0; v < 2; ++v) {
                            const float e = fast_exp2(x[u][nt][v] - m);
                            l_run[nt] += e;
                            pf[u][nt][v] = transpose8x8(split_pair(e));
                        }
                }
#pragma unroll
                for (uint32_t u = 0; u < 2; ++u)
#pragma unroll
                    for (uint32_t pn = 0; pn < kPanels; ++pn) {
                        const uint32_t at = base + u * kv4_group_bytes(HD);
                        uint4 w = lds128_at(at + 8 * HD + pn * 512 + lane * 16);
                        uint32_t sv = lds32_at(at + 17 * HD + pn * 64 + (g / 2 * 4 + c) * 4);
                        if (!whole) {
                            // Positions outside the split, of which anything may lie here: scale 0.
                            const uint32_t t = tok0 + (2 * h + u) * kKv4Group + 2 * c;
                            uint32_t keep = 0;
#pragma unroll
                            for (uint32_t b = 0; b < 4; ++b) {
                                const uint32_t tt = t + b % 2 + 8 * (b / 2);
                                keep |= (tt >= t_begin && tt < t_end ? 0xffu : 0u) << (8 * b);
                            }
                            sv &= groups >> (2 * h + u) & 1u ? keep : 0u;
                            // A value that is NaN reaches the rows that see its position only: its scale
                            // becomes 0, and those rows' sums NaN (0 times NaN would reach the others).
                            uint32_t bad = 0;
#pragma unroll
                            for (uint32_t b = 0; b < 4; ++b)
                                if ((sv >> (8 * b) & 0x7fu) == 0x7fu) {
                                    bad |= 1u << (2 * c + b % 2 + 8 * (b / 2));
                                    sv &= ~(0xffu << (8 * b));
                                }
                            bad |= __shfl_xor_sync(0xffffffffu, bad, 1);
                            bad |= __shfl_xor_sync(0xffffffffu, bad, 2);
                            if (bad) {
                                const uint32_t t0 = tok0 + (2 * h + u) * kKv4Group;
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    bool sees = false;
                                    for (uint32_t b = 0; b < kKv4Group; ++b) sees = sees || (bad >> b & 1u && t0 + b >= row_begin[nt] && t0 + b < row_end[nt]);
                                    if (sees)
#pragma unroll
                                        for (uint32_t i = 0; i < 4; ++i) acc[pn * 4 + i][nt][0] = acc[pn * 4 + i][nt][1] = NAN;
                                }
                            }
                        }
                        const uint32_t s01 = kv4_scale_pair(sv), s23 = kv4_scale_pair(sv >> 16);
                        // Bytes of one column of two positions each, even and odd columns.
                        const uint32_t lo = 0x0f0f0f0fu;
                        uint32_t e01[4], o01[4], e23[4], o23[4];
                        mx_unpack_fp4((w.x & lo) | (w.y << 4 & ~lo), e01);
                        mx_unpack_fp4((w.x >> 4 & lo) | (w.y & ~lo), o01);
                        mx_unpack_fp4((w.z & lo) | (w.w << 4 & ~lo), e23);
                        mx_unpack_fp4((w.z >> 4 & lo) | (w.w & ~lo), o23);
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i) {
                            const uint32_t a[4] = {hmul2(e01[i], s01), hmul2(o01[i], s01), hmul2(e23[i], s23), hmul2(o23[i], s23)};
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) mma16816(part[pn * 4 + i][nt], a, pf[u][nt][0], pf[u][nt][1]);
                        }
                    }
            }
            if (started)
#pragma unroll
                for (uint32_t i = 0; i < HD / 16; ++i)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int v = 0; v < 2; ++v) acc[i][nt][v] += fmaf(part[i][nt][2 * v + 1], 0x1p-11f, part[i][nt][2 * v]);
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(&empty[warp][stage])) : "memory");
        }
        // No copy may still be landing when the stages are used again below: after a wait that gave up,
        // the later ones are waited for too (bounded).
        if (!ok)
            for (uint32_t r = k; r < min(mine, k + S); ++r) (void)mbar_wait(&full[warp][r % S], r / S & 1u);

        // This warp's state to its own stages: [rows][HD] sums, then maxima and denominators.
        float *state = reinterpret_cast<float *>(ring);
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float l = l_run[nt];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            const uint32_t r = 4 * nt + c;
            __syncwarp();
#pragma unroll
            for (uint32_t i = 0; i < HD / 16; ++i) {
                float *o = state + r * HD + i / 4 * 64 + 8 * g + i % 4 * 2;
                o[0] = acc[i][nt][0];
                o[1] = acc[i][nt][1];
            }
            if (g == 0) {
                state[kRows * HD + r] = m_run[nt];
                state[kRows * HD + kRows + r] = l;
            }
        }
    }
    __syncthreads();
    auto warp_state = [&](uint32_t w) { return reinterpret_cast<const float *>(smem + size_t(w) * S * kStageBytes<HD>); };
    const uint32_t splits = end > begin ? s_last - s_first + 1 : 1u;
    float *parts_out = p.partials + (size_t(unit) * p.n_splits + split) * kRows * (HD + 2);
    auto finish = [&](uint32_t r, uint32_t d, float a, float l) {
        const uint32_t q = first + r;
        kv4_store<T>(p, row0 + q / p.group, (head * p.group + q % p.group) * HD + d, a / fmaxf(l, 1e-30f) * p.v_scale);
    };
    for (uint32_t i = threadIdx.x; i < rows * HD; i += kThreads) {
        const uint32_t r = i / HD, d = i % HD;
        float m = -INFINITY;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) m = fmaxf(m, warp_state(w)[kRows * HD + r]);
        float a = 0.f, l = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w) {
            const float mw = warp_state(w)[kRows * HD + r], f = mw == -INFINITY ? 0.f : fast_exp2(mw - m);
            const float lw = warp_state(w)[kRows * HD + kRows + r];
            // A warp without keys for the row has sums of 0; a NaN must stay one (its maximum may be -inf).
            a += mw == -INFINITY ? warp_state(w)[r * HD + d] : warp_state(w)[r * HD + d] * f;
            l += mw == -INFINITY ? lw : lw * f;
        }
        if (splits == 1) {
            finish(r, d, a, l);
        } else {
            parts_out[r * (HD + 2) + d] = a;
            if (d == 0) {
                parts_out[r * (HD + 2) + HD] = m;
                parts_out[r * (HD + 2) + HD + 1] = l;
            }
        }
    }
    if (splits == 1) {
        if (p.out_packed) asm volatile("fence.proxy.async.global;" ::: "memory");  // read by TMA next
        return;
    }
    __threadfence();
    __syncthreads();
    __shared__ uint32_t ticket;
    if (threadIdx.x == 0) ticket = atomicAdd(p.counters + unit, 1u);
    __syncthreads();
    if (ticket != splits - 1) return;
    __threadfence();
    // The splits' maxima and denominators first, all at once, in the warps' stages.
    static_assert(2 * kMaxSplits * kRows * sizeof(float) <= kRowsSmem<HD, NT>, "room for them");
    const float *parts_in = p.partials + (size_t(unit) * p.n_splits + s_first) * kRows * (HD + 2);
    float *maxima = reinterpret_cast<float *>(smem), *sums = maxima + kMaxSplits * kRows;
    for (uint32_t i = threadIdx.x; i < splits * rows; i += kThreads) {
        const float2 ml = __ldcg(reinterpret_cast<const float2 *>(parts_in + (size_t(i / rows) * kRows + i % rows) * (HD + 2) + HD));
        maxima[i] = ml.x;
        sums[i] = ml.y;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < rows * HD; i += kThreads) {
        const uint32_t r = i / HD, d = i % HD;
        float m = -INFINITY;
        for (uint32_t sp = 0; sp < splits; ++sp) m = fmaxf(m, maxima[sp * rows + r]);
        float a = 0.f, l = 0.f;
#pragma unroll 16  // independent loads
        for (uint32_t sp = 0; sp < splits; ++sp) {
            const float ms = maxima[sp * rows + r], f = ms == -INFINITY ? 1.f : fast_exp2(ms - m);
            a += __ldcg(parts_in + (size_t(sp) * kRows + r) * (HD + 2) + d) * f;
            l += sums[sp * rows + r] * f;
        }
        finish(r, d, a, l);
    }
    if (p.out_packed) asm volatile("fence.proxy.async.global;" ::: "memory");
    if (threadIdx.x == 0) p.counters[unit] = 0u;
}

// What a call's shape comes to: tiles of rows, units of work without the key split, and the split.
struct Plan {
    bool prompt;
    uint32_t tile_rows, row_tiles, split_tokens, n_splits;
    uint64_t units;
    size_t bytes;
};
// Scratch: a counter for each unit, then the splits' sums. As many counters for every shape, so that the sums
// of one call never lie where the next one, of another shape, has its counters. More units than that
// fill the SMs several times over and are not split.
constexpr uint32_t kCounters = 2048;
constexpr size_t kPartialsAt = kCounters * sizeof(uint32_t);
// More than kFewRows (query, head) rows per kv head go to the kernel for prompts.
constexpr uint32_t kFewRows = 16;
constexpr uint32_t kMaxUnits = 0x7fffffffu;  // a grid's, and a unit's rows
Plan make_plan(uint32_t n, uint32_t n_rows, uint32_t n_q, uint32_t group, uint32_t n_kv, uint32_t hd, uint32_t max_ctx, uint32_t split_tokens, int sms) {
    Plan p{};
    const uint64_t rows = uint64_t(std::min(n_q, n_rows)) * group;  // no entry has more queries than there are
    p.prompt = rows > kFewRows;
    p.tile_rows = p.prompt ? kKv4PromptRows : rows <= 4 ? 4 : 8;
    const uint64_t per_entry = (rows + p.tile_rows - 1) / p.tile_rows * n_kv;
    if (rows > kMaxUnits || per_entry > kMaxUnits || n * per_entry > kMaxUnits) {
        p.units = ~uint64_t(0);  // refused
        return p;
    }
    p.row_tiles = ceil_div(rows, p.tile_rows);
    p.units = n * per_entry;
    // Splits in steps of a chunk for each warp, or of prompts' tiles.
    const uint64_t unit = p.prompt ? kKv4PromptKeys : kWarps * kChunk, ctx = std::max(max_ctx, 1u);
    uint64_t want;
    if (p.prompt) {
        want = std::min<uint64_t>(16, (uint64_t(sms) + p.units - 1) / p.units);
    } else {
        // As many CTAs as the SMs hold, in splits of 256 keys or more; three times as many where
        // that leaves 2048 keys to a split, so that the last ones to run are short. Measured: 1 x 4001 keys x 3 kv
        // heads 12.0 us in splits of 128, 9.4 in 256; 16 x 5 queries x 2000 35 us in 128, 20 in 512 and
        // 1024; 64 x 32768 x 3 141 us in 4 splits, 122 in 10, 129 in 16; 64 x 4096 x 32 151 us in one, 183 in two.
        const uint64_t slots = uint64_t(sms) * (hd == 64 ? (p.tile_rows == 4 ? kCtasPerSm<64, 1> : kCtasPerSm<64, 2>) : kCtasPerSm<128, 1>);
        want = std::min<uint64_t>((slots + p.units - 1) / p.units, (ctx + unit - 1) / unit);
        want = std::max<uint64_t>(want, std::min<uint64_t>((slots * 3 + p.units - 1) / p.units, ctx / 2048));
    }
    want = std::min<uint64_t>(std::max<uint64_t>(want, 1), std::min<uint64_t>(kMaxSplits, (ctx + unit - 1) / unit));
    uint64_t per = split_tokens ? std::max<uint64_t>(split_tokens, (ctx + kMaxSplits - 1) / kMaxSplits) : (ctx + want - 1) / want;
    if (p.units > kCounters) per = ctx;
    p.split_tokens = uint32_t(std::min<uint64_t>((per + unit - 1) / unit * unit, 0xffffff80u));
    p.n_splits = ceil_div(ctx, p.split_tokens);
    p.bytes = p.n_splits > 1 ? kPartialsAt + size_t(p.units) * p.n_splits * p.tile_rows * (hd + 2) * sizeof(float) : 0;
    return p;
}

}  // namespace
}  // namespace opure

using namespace opure;

extern "C" size_t opure_kv4_attention_scratch_bytes(uint32_t n, uint32_t n_rows, uint32_t n_q, uint32_t n_heads, uint32_t n_kv,
                                                    uint32_t hd, uint32_t max_ctx, uint32_t split_tokens) {
    if (!n || !n_rows || !n_q || !n_heads || !kv4_shape(n_kv, hd, 64) || n_heads % n_kv) return 0;
    int dev = 0, sms = 148;
    if (cudaGetDevice(&dev) == cudaSuccess) cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const Plan p = make_plan(n, n_rows, n_q, n_heads / n_kv, n_kv, hd, max_ctx, split_tokens, sms);
    return p.units > kMaxUnits ? 0 : std::max<size_t>(16, p.bytes);
}

extern "C" opure_status opure_kv4_attention(opure_ctx *ctx, const opure_kv4_attn_args *a) {
    opure_status s = enter(ctx);
    if (s) return s;
    if (!a || type_bytes(a->type) == 0) return OPURE_ERR_INVALID_ARG;
    if ((s = kv4_check(a->kv))) return s;
    const uint32_t hd = a->kv.head_dim;
    const uint64_t cols = uint64_t(a->n_heads) * hd;
    if (!a->n_heads || a->n_heads % a->kv.n_kv || a->q_stride < cols || a->out_stride < cols) return OPURE_ERR_INVALID_ARG;
    if (a->n == 0 || a->n_q == 0 || a->n_rows == 0) return OPURE_OK;
    if (!a->q || !a->out || !a->seq || !a->seq_len || !a->scratch || !type_aligned(a->q, a->type) || !type_aligned(a->out, a->type))
        return OPURE_ERR_INVALID_ARG;
    if (!a->q_begin && uint64_t(a->n) * a->n_q != a->n_rows) return OPURE_ERR_INVALID_ARG;
    if (cols > 0x7fffffffu || a->n_rows > 0x7fffffffu || a->max_ctx > 0x7fffffffu) return OPURE_ERR_UNSUPPORTED;
    const Plan pl = make_plan(a->n, a->n_rows, a->n_q, a->n_heads / a->kv.n_kv, a->kv.n_kv, hd, a->max_ctx, a->split_tokens, ctx->sm_count);
    if (pl.units > kMaxUnits) return OPURE_ERR_UNSUPPORTED;
    if (a->scratch_bytes < pl.bytes || reinterpret_cast<uintptr_t>(a->scratch) % 16) return OPURE_ERR_INVALID_ARG;
    Kv4AttnParams p{};
    p.q = a->q;
    p.out = a->out;
    p.q_stride = a->q_stride;
    p.out_stride = a->out_stride;
    p.seq = a->seq;
    p.seq_len = a->seq_len;
    p.q_begin = a->q_begin;
    p.n = a->n;
    p.n_rows = a->n_rows;
    p.n_q = a->n_q;
    p.n_heads = a->n_heads;
    p.group = a->n_heads / a->kv.n_kv;
    p.row_tiles = pl.row_tiles;
    p.factor = a->scale * 1.4426950408889634f * (a->kv.k_scale == 0.f ? 1.f : a->kv.k_scale);
    p.v_scale = a->kv.v_scale == 0.f ? 1.f : a->kv.v_scale;
    p.split_tokens = pl.split_tokens;
    p.n_splits = pl.n_splits;
    p.counters = static_cast<uint32_t *>(a->scratch);
    p.partials = reinterpret_cast<float *>(static_cast<char *>(a->scratch) + kPartialsAt);
    p.kv = a->kv;
    p.st = ctx->status;
    p.out_packed = reinterpret_cast<__half *>(a->out_packed);
    p.pk_npad = (a->n_rows + 15) & ~15u;
    if (pl.prompt) return kv4_prompt_launch(ctx, p, a->type, uint32_t(pl.units));
    return with_type(a->type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto k, uint32_t smem) -> opure_status {
            OPURE_CUDA_TRY(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
            return launch(ctx, k, dim3(uint32_t(pl.units), pl.n_splits), dim3(kThreads), smem, true, p);
        };
        if (hd == 64) return pl.tile_rows == 4 ? go(rows_kernel<T, 64, 1>, kRowsSmem<64, 1>) : go(rows_kernel<T, 64, 2>, kRowsSmem<64, 2>);
        return pl.tile_rows == 4 ? go(rows_kernel<T, 128, 1>, kRowsSmem<128, 1>) : go(rows_kernel<T, 128, 2>, kRowsSmem<128, 2>);
    });
}
