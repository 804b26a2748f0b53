// score.cu -- log probabilities of given tokens, their ranks, entropies and the most likely tokens
// of rows of logits, in one pass (opure_token_scores).
//
// A thread keeps a reference m, z = sum exp(x - m) and e = sum exp(x - m) (x - m) over its logits x;
// m is the largest logit of the CTA's first loads, raised (and the sums rescaled) when a larger one
// comes. The row's log-sum-exp is then m + log z, its entropy log z - e / z, with m the row's largest:
// with any other reference the two terms of the entropy would cancel.
//
// The most likely tokens: a thread notes in which pieces of the row it saw a logit that reaches a bound,
// a value that `top` logits of the first piece reach (the top-th largest of 32 lanes' maxima, as many of each
// warp). When the row is through, the top-th largest of the threads' maxima over all of it is a bound that
// little more than `top` logits reach. Another warp reads the pieces that the threads above it have noted once
// more (from L2), 32 logits of one thread at a time, collects those that reach the bound as keys (orderable
// value, ~index), and puts them in order by counting, for each, the larger ones.
//
// CTAs go from row to row with three kinds of warps: four that work on values, one that copies the coming
// pieces into a ring of stages, and one that finishes a row (joins its sums, finds its best tokens, writes the
// results) while the others are at the next. Nothing in a piece but a row's first waits for another of the
// four. A row with more keys than the buffer takes (equal values at the bound, large ones all in one thread's
// words) is gone over once more for its keys alone. Where there are few rows each is shared out over a
// cluster of up to 8 CTAs, whose parts meet in distributed shared memory.
// Bound by memory while there are many rows: 4096 rows of 49152 fp32 logits take 139-144 us without best
// tokens and 165-170 us with 5 (5.6 and 4.8 TB/s of 6.5 measured), 203 us with 20. With the finishing done by
// the four warps themselves it was 215 us with 5. In fp16 they take 158 us (2.5 TB/s), and 4096 rows of 4096
// logits 54 us (fp32 59): the finishing of a row, some 9,000 clocks whatever its length, bounds these. A single
// row, a cluster of 8, is latency: 5.5 us, 13.6 us with 20 best tokens (11.1 us when four warps finished it;
// kept, since one way serves all sizes).
#include <algorithm>

#include "attn_core.cuh"
#include "kv4.cuh"
#include "tcgen05.cuh"

namespace opure {
namespace {

constexpr uint32_t kThreads = 128, kWarps = kThreads / 32;
constexpr uint32_t kCtasPerSm = 3;
constexpr uint32_t kMaxCluster = 8;
constexpr uint32_t kBuffer = 512;   // keys
constexpr uint32_t kItems = 512;    // pieces of threads that are read again
constexpr uint32_t kOnce = 32;      // so many of them at once
constexpr uint32_t kValues = 32;    // of a thread in a piece
template <typename T>
constexpr uint32_t kWords = kValues * sizeof(T) / 16;  // 16-byte words of them
template <typename T>
constexpr uint32_t kPiece = kThreads * kWords<T>;      // words of a piece
template <typename T>
constexpr uint32_t kStages = sizeof(T) == 4 ? 3 : 6;   // 48 KB a CTA
constexpr uint32_t kMaxStages = 6;
constexpr uint32_t kSort = 96;      // up to this many keys are put in order as they are
constexpr float kLowest = -3.4028234663852886e38f;  // of fp32: a row may hold nothing larger
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -200.f;                       // exp of it is 0, and 0 times it stays 0 (unlike -inf)

struct ScoreParams {
    const void *logits;
    uint32_t vocab, rows, cluster;
    size_t stride;
    const int32_t *tokens;
    float *logprob;
    int32_t *rank;
    float *entropy, *lse;
    uint32_t top;
    int32_t *top_tokens;
    float *top_logprobs;
    DeviceStatus *st;
};

__device__ __forceinline__ float exp_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * kLog2e));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ uint32_t order_bits(float v) {  // larger for larger values, 0 and -0 the same; NaN below all
    const uint32_t b = __float_as_uint(v + 0.f);
    return v != v ? 0u : b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_value(uint32_t b) { return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b); }

// Sums over part of a row: m, z, e as above.
struct Sums {
    float m, z, e;
    __device__ __forceinline__ void rescale(float to) {  // to >= m
        const float d = m == to ? 0.f : fmaxf(m - to, kFar), f = exp_fast(d);
        e = f * fmaf(z, d, e);
        z *= f;
        m = to;
    }
    __device__ __forceinline__ void join(Sums o) {
        const float big = fmaxf(m, o.m);
        rescale(big);
        o.rescale(big);
        z += o.z;
        e += o.e;
    }
};

using Key = unsigned long long;

// A barrier of the threads that work on values.
__device__ __forceinline__ void sync_values() { asm volatile("barrier.cta.sync 1, %0;" ::"n"(kThreads) : "memory"); }
// What a row's finishing needs of the threads that worked on it.
struct Handed {
    float most[kThreads];        // each one's largest value
    uint32_t noted[kThreads];    // bit i: pieces i, i + 32, .. have one that reaches the first piece's bound
    float m[kWarps], z[kWarps], e[kWarps];
    uint32_t ahead[kWarps];
};
struct RowShared {
    __align__(16) Key buffer[2][kBuffer];        // what lies behind them may be read by sort_keys
    Key best[kMaxCluster][OPURE_SCORE_MAX_TOP];  // each CTA's best in order, 0 for none (the first CTA's copy is used)
    uint32_t items[kItems];
    __align__(16) uint4 again[kOnce * 32 / 4];   // a thread's words of so many pieces
    __align__(16) uint32_t most[64];
    Handed handed[2];
    __align__(16) uint32_t reach[2][32];         // the largest lanes' maxima, as many of each warp, as order bits
    float cm[kMaxCluster], cz[kMaxCluster], ce[kMaxCluster];
    uint32_t cahead[kMaxCluster];
    uint64_t full[kMaxStages], empty[kMaxStages], given[2], taken[2];
};

__device__ __forceinline__ void arrive(uint64_t *bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// The largest value that `top` threads' values (order bits) are known to reach, 0 for none, and the
// largest of all. All threads that work on values; one barrier. A call may use the same `reach` as an
// earlier one if there was another barrier between them.
struct Reach {
    uint32_t bound, highest;
};
static_assert(OPURE_SCORE_MAX_TOP <= 32, "as many maxima are compared");
__device__ __forceinline__ Reach reach_of(uint32_t *reach, uint32_t o, uint32_t top) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    // Of each warp one more than its share of `top`, for a bound with fewer values above it.
    const uint32_t each = min(top / kWarps + 1, 32 / kWarps);
    uint32_t own = 0;
    for (uint32_t k = 0; k < each; ++k) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, o);
        if (lane == k) own = m;
        if (o == m) o = 0;  // equal ones in other lanes go too: the bound is no higher for it
    }
    if (lane < 32 / kWarps) reach[warp * (32 / kWarps) + lane] = own;
    sync_values();
    const uint32_t mine = reach[lane];
    uint32_t as_large = 0;
#pragma unroll
    for (uint32_t j = 0; j < 32; j += 4) {
        const uint4 y = *reinterpret_cast<const uint4 *>(&reach[j]);
        as_large += (y.x >= mine) + (y.y >= mine) + (y.z >= mine) + (y.w >= mine);
    }
    return Reach{__reduce_max_sync(0xffffffffu, as_large >= top ? mine : 0u), __reduce_max_sync(0xffffffffu, mine)};
}

// A value (order bits) that `top` of the warp's 4 x 32 values reach, the top-th largest of the two largest
// of each lane; 0 for none.
__device__ __noinline__ uint32_t nth_of(RowShared &sm, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t top) {
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t x = max(max(a, b), max(c, d)), y = max(max(min(a, b), min(c, d)), min(max(a, b), max(c, d)));
    sm.most[lane] = x;
    sm.most[32 + lane] = y;
    __syncwarp();
    uint32_t nx = 0, ny = 0;
#pragma unroll 4
    for (uint32_t k = 0; k < 64; k += 4) {
        const uint4 o = *reinterpret_cast<const uint4 *>(&sm.most[k]);
        nx += (o.x >= x) + (o.y >= x) + (o.z >= x) + (o.w >= x);
        ny += (o.x >= y) + (o.y >= y) + (o.z >= y) + (o.w >= y);
    }
    __syncwarp();
    return __reduce_max_sync(0xffffffffu, nx >= top ? x : ny >= top ? y : 0u);
}

// The `top` largest of n different keys of a buffer, in order (0 for none), to the other one; returns how many.
// One warp. A lane counts the larger keys for each of its own, after those below a value that `top` of them
// reach have dropped out.
__device__ __noinline__ uint32_t sort_keys(RowShared &sm, Key *src, uint32_t n, Key *dst, uint32_t top) {
    const uint32_t lane = threadIdx.x & 31u;
    __syncwarp();
    if (n > kSort) {
        uint32_t o[4] = {};
#pragma unroll
        for (uint32_t b = 0; b < kBuffer / 32; ++b)
            if (b * 32 + lane < n) o[b % 4] = max(o[b % 4], uint32_t(src[b * 32 + lane] >> 32));
        const uint32_t bound = nth_of(sm, o[0], o[1], o[2], o[3], top);
        uint32_t kept = 0;
        for (uint32_t i0 = 0; i0 < n; i0 += 32) {
            const Key key = i0 + lane < n ? src[i0 + lane] : 0ull;
            const bool keep = uint32_t(key >> 32) >= bound && key != 0;
            const uint32_t who = __ballot_sync(0xffffffffu, keep);
            if (keep) src[kept + __popc(who & ((1u << lane) - 1u))] = key;  // at or before where it was
            kept += __popc(who);
            __syncwarp();
        }
        n = kept;
    }
    if (lane < top) dst[lane] = 0ull;
    __syncwarp();
    const uint32_t from = smem_addr(src);
    for (uint32_t i = lane; i < n; i += 32) {
        const Key key = src[i];
        uint32_t place = 0;
        for (uint32_t j = 0; j < n; j += 8) {
            Key k[8];
#pragma unroll
            for (uint32_t q = 0; q < 8; q += 2)  // up to 7 keys past the end are read, and left out
                asm volatile("ld.shared.v2.u64 {%0, %1}, [%2];" : "=l"(k[q]), "=l"(k[q + 1]) : "r"(from + (j + q) * 8));
#pragma unroll
            for (uint32_t q = 0; q < 8; ++q) place += k[q] > key && j + q < n;
        }
        if (place < top) dst[place] = key;
    }
    __syncwarp();
    return min(n, top);
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads + 64, kCtasPerSm) score_kernel(ScoreParams p) {
    constexpr uint32_t kVec = 16 / sizeof(T), W = kWords<T>, P = kPiece<T>, S = kStages<T>;
    extern __shared__ __align__(128) uint4 stages[];  // [S][P]
    __shared__ RowShared sm;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    if (threadIdx.x < S) {
        mbar_init(&sm.full[threadIdx.x], 1);
        mbar_init(&sm.empty[threadIdx.x], kWarps);
    }
    if (threadIdx.x < 2) {
        mbar_init(&sm.given[threadIdx.x], kWarps);
        mbar_init(&sm.taken[threadIdx.x], 1);
    }
    __syncthreads();
    grid_dependency_wait();
    grid_dependents_launch();
    const uint32_t cr = p.cluster > 1 ? tc::cluster_rank() : 0u;
    if (p.cluster > 1) tc::cluster_arrive();  // met again before anything goes to another CTA

    // A row: values before its first aligned 16-byte word, words (this CTA's share of them), values after.
    struct Row {
        const T *x;
        uint32_t n_head, words, n_tail, begin, end;
    };
    auto row_at = [&](uint32_t row) {
        Row r;
        r.x = static_cast<const T *>(p.logits) + size_t(row) * p.stride;
        const uint32_t mis = uint32_t(reinterpret_cast<uintptr_t>(r.x) % 16 / sizeof(T));
        r.n_head = min(mis ? kVec - mis : 0u, p.vocab);
        r.words = (p.vocab - r.n_head) / kVec;
        r.n_tail = p.vocab - r.n_head - r.words * kVec;
        const uint32_t share = (r.words + p.cluster - 1) / p.cluster;
        r.begin = min(cr * share, r.words);
        r.end = min(r.begin + share, r.words);
        return r;
    };
    const uint32_t step = gridDim.x / p.cluster, row0 = blockIdx.x / p.cluster;

    if (warp == kWarps) {
        uint32_t it = 0;
        bool ok = true;
        if (lane == 0) {
            for (uint32_t row = row0; row < p.rows && ok; row += step) {
                const Row r = row_at(row);
                const uint4 *body = reinterpret_cast<const uint4 *>(r.x + r.n_head);
                for (uint32_t w = r.begin; w < r.end && ok; w += P, ++it) {
                    const uint32_t s = it % S, bytes = min(P, r.end - w) * 16;
                    if (it >= S && !mbar_wait(&sm.empty[s], (it / S - 1) & 1u)) {
                        report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 98, blockIdx.x);
                        ok = false;
                        break;
                    }
                    mbar_expect_tx(&sm.full[s], bytes);
                    bulk_load(stages + s * P, body + w, bytes, &sm.full[s]);
                }
            }
            // No copy may still be landing when the CTA exits.
            for (uint32_t s = 0; s < S && s < it; ++s) (void)mbar_wait(&sm.full[s], ((it - 1 - s) / S) & 1u);
        }
        __syncwarp();
        if (p.cluster > 1) {
            tc::cluster_wait();
            tc::cluster_sync();
        }
        return;
    }

    auto token_at = [&](uint32_t row) { return p.tokens && row < p.rows ? p.tokens[row] : -1; };
    auto value_of = [&](uint32_t row, int32_t token) {
        return token >= 0 && uint32_t(token) < p.vocab ? to_f32(static_cast<const T *>(p.logits)[size_t(row) * p.stride + token]) : 0.f;
    };
    auto key_of = [](float v, uint32_t i) { return static_cast<Key>(order_bits(v)) << 32 | (0xffffffffu - i); };
    auto unpack = [](const uint4 &raw, float *v) {
        if constexpr (sizeof(T) == 4) {
            v[0] = __uint_as_float(raw.x); v[1] = __uint_as_float(raw.y);
            v[2] = __uint_as_float(raw.z); v[3] = __uint_as_float(raw.w);
        } else {
            const T *h = reinterpret_cast<const T *>(&raw);
#pragma unroll
            for (uint32_t j = 0; j < kVec; ++j) v[j] = to_f32(h[j]);
        }
    };
    // (Of the references, a warp's largest; as order bits, for one instruction.)
    auto warp_join = [](Sums &a) {
        a.rescale(order_value(__reduce_max_sync(0xffffffffu, order_bits(a.m))));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            a.z += __shfl_xor_sync(0xffffffffu, a.z, o);
            a.e += __shfl_xor_sync(0xffffffffu, a.e, o);
        }
    };
    // The value outside whole words that is a lane's.
    auto is_edge = [&](const Row &r) { return cr == 0 && lane < r.n_head + r.n_tail; };
    auto edge_index = [&](const Row &r) { return lane < r.n_head ? lane : r.n_head + r.words * kVec + (lane - r.n_head); };

    if (warp == kWarps + 1) {
        uint32_t turn = 0;
        bool ok = true;
        for (uint32_t row = row0; row < p.rows; row += step, ++turn) {
            const Row r = row_at(row);
            const uint4 *body = reinterpret_cast<const uint4 *>(r.x + r.n_head);
            const int32_t token = token_at(row);
            const float xt = value_of(row, token);
            const bool given = token >= 0 && uint32_t(token) < p.vocab;
            const bool edge = is_edge(r);
            const uint32_t edge_i = edge_index(r);
            const float edge_v = TOP && edge ? to_f32(r.x[edge_i]) : -INFINITY;
            if (ok && !mbar_wait(&sm.given[turn & 1u], turn / 2 & 1u)) {
                if (lane == 0) report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 107, blockIdx.x);
                ok = false;
            }
            const Handed &h = sm.handed[turn & 1u];
            Sums t{lane < kWarps ? h.m[lane] : kLowest, lane < kWarps ? h.z[lane] : 0.f, lane < kWarps ? h.e[lane] : 0.f};
            warp_join(t);
            uint32_t ahead = __reduce_add_sync(0xffffffffu, lane < kWarps ? h.ahead[lane] : 0u);
            uint32_t most[4], noted[4];
            if constexpr (TOP) {
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    most[i] = order_bits(h.most[i * 32 + lane]);
                    noted[i] = h.noted[i * 32 + lane];
                }
            }
            __syncwarp();
            if (lane == 0) arrive(&sm.taken[turn & 1u]);
            if constexpr (TOP) {
                // A thread without values has no say: where only its -inf is reached there is no bound.
                uint32_t bound = nth_of(sm, most[0], most[1], most[2], most[3], p.top);
                if (bound <= order_bits(-INFINITY)) bound = 1;
                // Pieces to read again: as many as each lane's four threads noted.
                const uint32_t pieces = (r.end - r.begin + P - 1) / P;
                uint32_t own = 0;
#pragma unroll
                for (uint32_t i = 0; i < 4; ++i) {
                    if (most[i] < bound) noted[i] = 0;
                    if (pieces <= 32) own += __popc(noted[i]);
                    else
                        for (uint32_t bits = noted[i]; bits; bits &= bits - 1) own += (pieces + 32 - __ffs(bits)) / 32;
                }
                uint32_t upto = own;
#pragma unroll
                for (int d = 1; d < 32; d *= 2) {
                    const uint32_t v = __shfl_up_sync(0xffffffffu, upto, d);
                    if (lane >= uint32_t(d)) upto += v;
                }
                const uint32_t n_items = __shfl_sync(0xffffffffu, upto, 31);
                uint32_t count = 0, buf = 0;
                auto collect = [&](Key key, bool want) {
                    const uint32_t who = __ballot_sync(0xffffffffu, want);
                    if (want) sm.buffer[buf][count + __popc(who & ((1u << lane) - 1u))] = key;
                    count += __popc(who);
                };
                bool lost = n_items > kItems;
                if (!lost) {
                    uint32_t at = upto - own;
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i)
                        for (uint32_t bits = noted[i]; bits; bits &= bits - 1)
                            for (uint32_t q = __ffs(bits) - 1; q < pieces; q += 32) sm.items[at++] = q * P + i * 32 + lane;
                    __syncwarp();
                    // A 16-byte word of an item is a lane's to copy, then one of its 32 values to look at. (Loops
                    // as they stand: what runs once a row and is unrolled waits for its instructions instead.)
#pragma unroll 1
                    for (uint32_t k0 = 0; k0 < n_items && !lost; k0 += kOnce) {
                        const uint32_t here = min(kOnce, n_items - k0);
#pragma unroll 1
                        for (uint32_t k = lane; k < here * W; k += 32) {
                            const uint32_t w = r.begin + sm.items[k0 + k / W] + k % W * kThreads;
                            if (w < r.end) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_addr(&sm.again[k])), "l"(body + w) : "memory");
                        }
                        asm volatile("cp.async.wait_all;" ::: "memory");
                        __syncwarp();
#pragma unroll 1
                        for (uint32_t k0v = 0; k0v < here && !lost; k0v += 4) {
                            float v[4];
                            uint32_t w[4];
#pragma unroll
                            for (uint32_t k = 0; k < 4; ++k) {
                                w[k] = k0v + k < here ? r.begin + sm.items[k0 + k0v + k] + lane / kVec * kThreads : r.end;
                                v[k] = to_f32(reinterpret_cast<const T *>(&sm.again[(k0v + k) * W])[lane]);
                            }
                            if (count > kBuffer - 160) lost = true;  // 32 of these for the values outside whole words
                            else
#pragma unroll
                                for (uint32_t k = 0; k < 4; ++k)
                                    collect(key_of(v[k], r.n_head + w[k] * kVec + lane % kVec), w[k] < r.end && order_bits(v[k]) >= bound);
                        }
                        __syncwarp();
                    }
                    if (!lost) collect(key_of(edge_v, edge_i), edge && order_bits(edge_v) >= bound);
                }
                if (lost) {
                    // Once more for the keys: every value, against the best so far.
                    Key least = 1ull << 32;  // a key below it is not wanted (NaN's are)
                    count = 0;
                    __syncwarp();
                    auto offer = [&](float v, uint32_t i, bool is) {
                        if (count > kBuffer - 32) {
                            count = sort_keys(sm, sm.buffer[buf], count, sm.buffer[buf ^ 1u], p.top);
                            buf ^= 1u;
                            if (count == p.top) least = sm.buffer[buf][p.top - 1] + 1;
                        }
                        const Key key = key_of(v, i);
                        collect(key, is && key >= least);
                    };
                    offer(edge_v, edge_i, edge);
                    constexpr uint32_t kWide = 4;
#pragma unroll 1
                    for (uint32_t w0 = r.begin + lane; w0 - lane < r.end; w0 += 32 * kWide) {
                        uint4 raw[kWide];
#pragma unroll
                        for (uint32_t k = 0; k < kWide; ++k) raw[k] = w0 + 32 * k < r.end ? body[w0 + 32 * k] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                        for (uint32_t k = 0; k < kWide; ++k) {
                            float v[kVec];
                            unpack(raw[k], v);
                            bool any = false;
#pragma unroll
                            for (uint32_t j = 0; j < kVec; ++j) any = any || order_bits(v[j]) >= uint32_t(least >> 32);
                            if (!__any_sync(0xffffffffu, any && w0 + 32 * k < r.end)) continue;
#pragma unroll
                            for (uint32_t j = 0; j < kVec; ++j) offer(v[j], r.n_head + (w0 + 32 * k) * kVec + j, w0 + 32 * k < r.end);
                        }
                    }
                }
                sort_keys(sm, sm.buffer[buf], count, sm.best[cr], p.top);
            }
            if (p.cluster > 1) {
                tc::cluster_wait();  // the first CTA runs by now
                // Every CTA sends its part to the first one.
                auto send = [&](const void *ptr, uint32_t v) {
                    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tc::map_rank(smem_addr(ptr), 0)), "r"(v) : "memory");
                };
                if (lane == 0) {
                    send(&sm.cm[cr], __float_as_uint(t.m));
                    send(&sm.cz[cr], __float_as_uint(t.z));
                    send(&sm.ce[cr], __float_as_uint(t.e));
                    send(&sm.cahead[cr], ahead);
                }
                if (TOP && cr != 0)
                    for (uint32_t k = lane; k < 2 * p.top; k += 32) {
                        const uint32_t *word = reinterpret_cast<const uint32_t *>(sm.best[cr]) + k;
                        send(word, *word);
                    }
                tc::cluster_sync();
                if (cr != 0) return;  // one row per cluster
                t = Sums{sm.cm[0], sm.cz[0], sm.ce[0]};
                ahead = sm.cahead[0];
                for (uint32_t c = 1; c < p.cluster; ++c) {
                    t.join(Sums{sm.cm[c], sm.cz[c], sm.ce[c]});
                    ahead += sm.cahead[c];
                }
                if (TOP) {
                    uint32_t count = 0;
                    for (uint32_t c = 0; c < p.cluster; ++c) {
                        const Key key = lane < p.top ? sm.best[c][lane] : 0ull;
                        const uint32_t who = __ballot_sync(0xffffffffu, key != 0);
                        if (key) sm.buffer[0][count + __popc(who & ((1u << lane) - 1u))] = key;
                        count += __popc(who);
                    }
                    sort_keys(sm, sm.buffer[0], count, sm.best[0], p.top);
                }
            }
            const float lz = logf(t.z);
            const bool none = t.z == 0.f;  // a row of -inf alone
            auto log_prob = [&](float v) { return none ? NAN : (v - t.m) - lz; };
            if (lane == 0) {
                if (p.lse) p.lse[row] = none ? -INFINITY : t.m + lz;
                if (p.entropy) p.entropy[row] = none ? NAN : lz - t.e / t.z;
                if (p.tokens) {
                    if (token >= 0 && !given) report(p.st, OPURE_ERR_DEVICE_BOUNDS, 97, uint32_t(token));
                    if (p.logprob) p.logprob[row] = given ? log_prob(xt) : token < 0 ? 0.f : NAN;
                    if (p.rank) p.rank[row] = given ? int32_t(ahead) : 0;
                }
            }
            if (TOP && lane < p.top) {
                const Key key = sm.best[0][lane];
                const size_t at = size_t(row) * p.top + lane;
                p.top_tokens[at] = key ? int32_t(0xffffffffu - uint32_t(key)) : -1;
                p.top_logprobs[at] = key ? log_prob(order_value(uint32_t(key >> 32))) : -INFINITY;
            }
            __syncwarp();
        }
        return;
    }

    int32_t token = token_at(row0);
    float xt = value_of(row0, token);
    uint32_t it = 0, turn = 0, reached = 0;  // reached: rows with a first piece, which alone meet at a barrier
    bool ok = true;
    for (uint32_t row = row0; row < p.rows; row += step, ++turn) {
        const Row r = row_at(row);
        const int32_t next_token = token_at(row + step);
        const bool given = token >= 0 && uint32_t(token) < p.vocab;
        // The smallest value that counts as ahead of xt: itself before the token, the next above it after.
        const float above = xt != xt ? xt : order_value(order_bits(xt) + 1u);
        const uint32_t token_word = given && uint32_t(token) >= r.n_head ? (uint32_t(token) - r.n_head) / kVec : ~0u;
        Sums s{kLowest, 0.f, 0.f};
        float2 z2 = make_float2(0.f, 0.f), e2 = z2;  // s.z and s.e in two parts
        uint32_t ahead = 0;
        auto add2 = [&](float2 v, bool far) {
            float2 d = __fadd2_rn(v, make_float2(-s.m, -s.m));
            if (far) d = make_float2(max_nan(d.x, kFar), max_nan(d.y, kFar));
            const float2 y = __fmul2_rn(d, make_float2(kLog2e, kLog2e));
            const float2 f = make_float2(fast_exp2(y.x), fast_exp2(y.y));
            z2 = __fadd2_rn(z2, f);
            e2 = __ffma2_rn(f, d, e2);
        };
        auto raise = [&](float v) {  // v: the largest of the values to come
            if (v > s.m) {
                s.z = z2.x + z2.y;
                s.e = e2.x + e2.y;
                s.rescale(v);
                z2 = make_float2(s.z, 0.f);
                e2 = make_float2(s.e, 0.f);
            }
        };
        // The values outside whole words: the first warp has one in each lane.
        const bool edge = warp == 0 && is_edge(r);
        const uint32_t edge_i = edge_index(r);
        const float edge_v = edge ? to_f32(r.x[edge_i]) : -INFINITY;
        float floor = -INFINITY, most = -INFINITY;  // bound of the first piece; largest of this thread's values
        uint32_t noted = 0;
        for (uint32_t piece = r.begin; piece < r.end; piece += P, ++it) {
            const uint32_t st = it % S;
            if (ok && !mbar_wait(&sm.full[st], it / S & 1u)) {
                if (lane == 0) report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 99, blockIdx.x);
                ok = false;
            }
            const uint4 *words = stages + st * P + threadIdx.x;
            float v[kValues];
#pragma unroll
            for (uint32_t b = 0; b < W; ++b) unpack(words[b * kThreads], v + b * kVec);
            const uint32_t left = r.end - piece;
            uint32_t n_values = kValues;
            if (left < P) {  // past the end: values that add nothing
                n_values = left > threadIdx.x ? min(W, (left - threadIdx.x + kThreads - 1) / kThreads) * kVec : 0u;
#pragma unroll
                for (uint32_t j = 0; j < kValues; ++j) v[j] = j < n_values ? v[j] : -INFINITY;
            }
            float high = v[0];
#pragma unroll
            for (uint32_t j = 1; j + 1 < kValues; j += 2) high = max3(high, v[j], v[j + 1]);
            high = fmaxf(high, v[kValues - 1]);
            if (piece == r.begin) {
                const Reach reach = reach_of(sm.reach[reached++ & 1u], order_bits(high), p.top);
                s.m = fmaxf(kLowest, order_value(reach.highest));
                // A thread without values has no say: where only its -inf is reached there is no bound.
                if (TOP && reach.bound > order_bits(-INFINITY)) floor = order_value(reach.bound);
            }
            if (TOP && high >= floor && n_values != 0) {
                noted |= 1u << ((piece - r.begin) / P & 31u);
                most = fmaxf(most, high);
            }
            __syncwarp();
            if (lane == 0) arrive(&sm.empty[st]);
            raise(high);
            const float2 z0 = z2, e0 = e2;
#pragma unroll
            for (uint32_t j = 0; j < kValues; j += 2) add2(make_float2(v[j], v[j + 1]), false);
            const float sum = e2.x + e2.y;
            if (sum != sum) {  // a -inf was among them (or a NaN): again, with a product of 0
                z2 = z0;
                e2 = e0;
#pragma unroll
                for (uint32_t j = 0; j < kValues; j += 2) add2(make_float2(v[j], v[j + 1]), true);
            }
            if (given && high >= xt) {
#pragma unroll
                for (uint32_t b = 0; b < W; ++b) {
                    const uint32_t w = piece + b * kThreads + threadIdx.x, i0 = r.n_head + w * kVec;
                    if (w >= r.end) continue;
                    if (w != token_word) {
                        const float from = i0 < uint32_t(token) ? xt : above;
#pragma unroll
                        for (uint32_t j = 0; j < kVec; ++j) ahead += v[b * kVec + j] >= from;
                    } else {
#pragma unroll
                        for (uint32_t j = 0; j < kVec; ++j)
                            ahead += v[b * kVec + j] >= (i0 + j < uint32_t(token) ? xt : above) && i0 + j != uint32_t(token);
                    }
                }
            }
        }
        const float next_xt = value_of(row + step, next_token);
        if (edge) {
            raise(edge_v);
            add2(make_float2(edge_v, -INFINITY), true);
            if (given) ahead += edge_v >= (edge_i < uint32_t(token) ? xt : above) && edge_i != uint32_t(token);
        }
        s.z = z2.x + z2.y;
        s.e = e2.x + e2.y;
        warp_join(s);
        ahead = __reduce_add_sync(0xffffffffu, ahead);
        // To the finishing warp.
        if (turn >= 2 && ok && !mbar_wait(&sm.taken[turn & 1u], (turn / 2 - 1) & 1u)) {
            if (lane == 0) report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 107, blockIdx.x);
            ok = false;
        }
        Handed &h = sm.handed[turn & 1u];
        if (TOP) {
            h.most[threadIdx.x] = most;
            h.noted[threadIdx.x] = noted;
        }
        if (lane == 0) {
            h.m[warp] = s.m;
            h.z[warp] = s.z;
            h.e[warp] = s.e;
            h.ahead[warp] = ahead;
        }
        __syncwarp();
        if (lane == 0) arrive(&sm.given[turn & 1u]);
        token = next_token;
        xt = next_xt;
    }
    if (p.cluster > 1) {
        tc::cluster_wait();
        tc::cluster_sync();
    }
}

}  // namespace
}  // namespace opure

using namespace opure;

extern "C" opure_status opure_token_scores(opure_ctx *ctx, const opure_score_args *a) {
    opure_status s = enter(ctx);
    if (s) return s;
    if (!a || type_bytes(a->type) == 0 || a->vocab == 0 || a->stride < a->vocab || a->top > OPURE_SCORE_MAX_TOP || a->top > a->vocab ||
        (a->top && (!a->top_tokens || !a->top_logprobs)))
        return OPURE_ERR_INVALID_ARG;
    if (a->rows == 0) return OPURE_OK;
    if (!a->logits || !type_aligned(a->logits, a->type)) return OPURE_ERR_INVALID_ARG;
    if (a->vocab > 0x7fffffffu || a->rows > 0x7fffffffu / kMaxCluster) return OPURE_ERR_UNSUPPORTED;
    // A cluster per row while there is room for its CTAs, and each part has half a piece.
    uint32_t cluster = 1;
    const uint32_t piece = kThreads * kValues, slots = uint32_t(ctx->sm_count) * kCtasPerSm;
    while (cluster < kMaxCluster && uint64_t(a->rows) * cluster * 2 <= slots && a->vocab / (cluster * 2) >= piece / 2) cluster *= 2;
    ScoreParams p{a->logits, a->vocab, a->rows, cluster, a->stride, a->tokens, a->logprob, a->rank, a->entropy, a->lse,
                  a->top, a->top_tokens, a->top_logprobs, ctx->status};
    return with_type(a->type, [&](auto t) -> opure_status {
        using T = decltype(t);
        cudaLaunchConfig_t cfg = {};
        const auto kernel = a->top ? score_kernel<T, true> : score_kernel<T, false>;
        constexpr uint32_t kSmem = kStages<T> * kPiece<T> * 16;
        OPURE_CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSmem)));
        cfg.gridDim = dim3(cluster > 1 ? a->rows * cluster : std::min(a->rows, slots));
        cfg.blockDim = dim3(kThreads + 64);
        cfg.dynamicSmemBytes = kSmem;
        cfg.stream = ctx->stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = cluster;
        attr[1].val.clusterDim.y = 1;
        attr[1].val.clusterDim.z = 1;
        cfg.attrs = ctx->pdl ? attr : attr + 1;
        cfg.numAttrs = ctx->pdl ? 2 : 1;
        OPURE_CUDA_TRY(cudaLaunchKernelEx(&cfg, kernel, p));
        return OPURE_OK;
    });
}
