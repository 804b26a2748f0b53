// score.cu -- log probabilities of given tokens, their ranks, entropies and the most likely tokens
// of rows of logits, in one pass (opure_token_scores).
//
// A thread keeps a reference m, z = sum exp(x - m) and e = sum exp(x - m) (x - m) over its logits x;
// m is the largest logit of the CTA's first loads, raised (and the sums rescaled) when a larger one
// comes. The row's log-sum-exp is then m + log z, its entropy log z - e / z, with m the row's largest:
// with any other reference the two terms of the entropy would cancel.
//
// The most likely tokens: logits that reach a bound go to a buffer in shared memory as keys (orderable
// value, ~index). The bound is a value that `top` logits of a row's first piece reach (the top-th largest of
// 32 lanes' maxima, as many of each warp), then the top-th best key of that piece. Keys are put in order by
// counting, for each, the larger ones.
//
// CTAs go from row to row while a warp of theirs copies the coming pieces into a ring of stages, so
// that what a row needs after its last piece (joining the sums, ordering the keys) costs no memory time;
// nothing in a piece but a row's first waits for other warps. A row with more keys than the buffer takes
// (equal values at the bound, rising ones) is gone over once more for its keys alone, a few values a
// thread at a time. Where there are few rows each is shared out over a cluster of up to 8 CTAs, whose
// parts meet in distributed shared memory.
#include <algorithm>

#include "attn_core.cuh"
#include "kv4.cuh"
#include "tcgen05.cuh"

namespace opure {
namespace {

constexpr uint32_t kThreads = 128, kWarps = kThreads / 32;
constexpr uint32_t kCtasPerSm = 3;
constexpr uint32_t kMaxCluster = 8;
constexpr uint32_t kBuffer = 512;   // keys; more than a step of one key a thread and the best so far
constexpr uint32_t kValues = 32;    // of a thread in a piece
template <typename T>
constexpr uint32_t kWords = kValues * sizeof(T) / 16;  // 16-byte words of them
template <typename T>
constexpr uint32_t kPiece = kThreads * kWords<T>;      // words of a piece
template <typename T>
constexpr uint32_t kStages = sizeof(T) == 4 ? 3 : 6;   // 48 KB a CTA
constexpr uint32_t kMaxStages = 6;
constexpr uint32_t kSort = 128;     // up to this many keys are put in order as they are
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

// Barriers of the threads that work on values (all but the copying warp's).
__device__ __forceinline__ void sync_values() { asm volatile("barrier.cta.sync 1, %0;" ::"n"(kThreads) : "memory"); }
__device__ __forceinline__ bool sync_values_or(bool v) {
    uint32_t r;
    asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, %2, p;\n selp.u32 %0, 1, 0, q;\n}"
                 : "=r"(r)
                 : "r"(uint32_t(v)), "n"(kThreads)
                 : "memory");
    return r != 0;
}

struct RowShared {
    __align__(16) Key buffer[2][kBuffer];  // what lies behind them may be read by sort_keys
    Key best[kMaxCluster][OPURE_SCORE_MAX_TOP];  // each CTA's best in order, 0 for none (the first CTA's copy is used)
    uint32_t count[2], valid[2];                 // of each buffer: keys asked for, and up to where they were all stored
    float m[kWarps], z[kWarps], e[kWarps];
    uint32_t ahead[kWarps];
    __align__(16) uint32_t reach[32];            // the largest lanes' maxima, as many of each warp, as order bits
    float cm[kMaxCluster], cz[kMaxCluster], ce[kMaxCluster];
    uint32_t cahead[kMaxCluster];
    uint64_t full[kMaxStages], empty[kMaxStages];
};

// The largest value that `top` threads' values (order bits) are known to reach, 0 for none, and the
// largest of all. All threads that work on values; one barrier.
struct Reach {
    uint32_t bound, highest;
};
static_assert(OPURE_SCORE_MAX_TOP <= 32, "as many maxima are compared");
__device__ __forceinline__ Reach reach_of(RowShared &sm, uint32_t o, uint32_t top) {
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    // Of each warp one more than its share of `top`, for a bound with fewer values above it.
    const uint32_t each = min(top / kWarps + 1, 32 / kWarps);
    uint32_t own = 0;
    for (uint32_t k = 0; k < each; ++k) {
        const uint32_t m = __reduce_max_sync(0xffffffffu, o);
        if (lane == k) own = m;
        if (o == m) o = 0;  // equal ones in other lanes go too: the bound is no higher for it
    }
    if (lane < 32 / kWarps) sm.reach[warp * (32 / kWarps) + lane] = own;
    sync_values();
    const uint32_t mine = sm.reach[lane];
    uint32_t as_large = 0;
#pragma unroll
    for (uint32_t j = 0; j < 32; j += 4) {
        const uint4 y = *reinterpret_cast<const uint4 *>(&sm.reach[j]);
        as_large += (y.x >= mine) + (y.y >= mine) + (y.z >= mine) + (y.w >= mine);
    }
    return Reach{__reduce_max_sync(0xffffffffu, as_large >= top ? mine : 0u), __reduce_max_sync(0xffffffffu, mine)};
}

// The `top` largest of n different keys, in order (0 for none), to dst; both in shared memory, src 16-byte
// aligned. All threads that work on values; no barrier. A thread counts the larger keys for each.
__device__ __forceinline__ void sort_keys(const Key *src, uint32_t n, Key *dst, uint32_t top) {
    if (threadIdx.x < top && threadIdx.x >= n) dst[threadIdx.x] = 0ull;
    const uint32_t from = smem_addr(src);
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
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
}

// Moves the `top` best keys of buffer `at`, in order, to the other one; returns the bound that a later
// key has to reach. All threads that work on values.
__device__ __noinline__ Key cut(RowShared &sm, uint32_t at, uint32_t top, Key least) {
    sync_values();
    uint32_t n = min(min(sm.count[at], sm.valid[at]), kBuffer);
    Key *src = sm.buffer[at];
    if (n > kSort) {
        // Keys below a value that `top` of them reach drop out first.
        uint32_t mine = 0;
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) mine = max(mine, uint32_t(src[i] >> 32));
        const uint32_t bound = reach_of(sm, mine, top).bound;
        if (threadIdx.x == 0) sm.count[at] = 0;
        Key own[(kBuffer + kThreads - 1) / kThreads];
#pragma unroll
        for (uint32_t b = 0; b < (kBuffer + kThreads - 1) / kThreads; ++b) {
            const uint32_t i = threadIdx.x + b * kThreads;
            own[b] = i < n ? src[i] : 0ull;
        }
        sync_values();
#pragma unroll
        for (uint32_t b = 0; b < (kBuffer + kThreads - 1) / kThreads; ++b)
            if (own[b] && uint32_t(own[b] >> 32) >= bound) src[atomicAdd(&sm.count[at], 1u)] = own[b];
        sync_values();
        n = sm.count[at];
    }
    Key *dst = sm.buffer[at ^ 1u];
    sort_keys(src, n, dst, top);
    if (threadIdx.x == 0) {
        sm.count[at ^ 1u] = min(n, top);
        sm.valid[at ^ 1u] = kBuffer;
    }
    sync_values();
    return n >= top ? dst[top - 1] + 1 : least;  // keys to come go behind the first min(n, top)
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads + 32, kCtasPerSm) score_kernel(ScoreParams p) {
    constexpr uint32_t kVec = 16 / sizeof(T), W = kWords<T>, P = kPiece<T>, S = kStages<T>;
    extern __shared__ __align__(128) uint4 stages[];  // [S][P]
    __shared__ RowShared sm;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    if (threadIdx.x < S) {
        mbar_init(&sm.full[threadIdx.x], 1);
        mbar_init(&sm.empty[threadIdx.x], kWarps);
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
    auto given_value = [&](uint32_t row, int32_t token) {
        return token >= 0 && uint32_t(token) < p.vocab ? to_f32(static_cast<const T *>(p.logits)[size_t(row) * p.stride + token]) : 0.f;
    };
    int32_t token = token_at(row0);
    float xt = given_value(row0, token);
    uint32_t it = 0;
    bool ok = true;
    for (uint32_t row = row0; row < p.rows; row += step) {
        const Row r = row_at(row);
        const int32_t next_token = token_at(row + step);
        const bool given = token >= 0 && uint32_t(token) < p.vocab;
        // The smallest value that counts as ahead of xt: itself before the token, the next above it after.
        const float above = xt != xt ? xt : order_value(order_bits(xt) + 1u);
        const uint32_t token_word = given && uint32_t(token) >= r.n_head ? (uint32_t(token) - r.n_head) / kVec : ~0u;
        uint32_t buf = 0;  // the buffer that keys go to
        if (threadIdx.x == 0) {
            sm.count[0] = 0;
            sm.valid[0] = kBuffer;
        }
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
        Key least = 1ull << 32;   // a key below it is not wanted (NaN's are)
        float floor = -INFINITY;  // nor a value below this
        auto key_of = [](float v, uint32_t i) { return static_cast<Key>(order_bits(v)) << 32 | (0xffffffffu - i); };
        auto cut_now = [&]() {
            least = cut(sm, buf, p.top, least);
            buf ^= 1u;
            floor = least >> 32 > 1 ? order_value(uint32_t(least >> 32)) : -INFINITY;
        };
        // `n` keys of this lane go to the buffer (all lanes call it): where to, or ~0 without room.
        auto room = [&](uint32_t n) -> uint32_t {
            uint32_t upto = n;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const uint32_t t = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= uint32_t(o)) upto += t;
            }
            const uint32_t all = __shfl_sync(0xffffffffu, upto, 31);
            uint32_t base = 0;
            if (lane == 0) base = atomicAdd(&sm.count[buf], all);
            base = __shfl_sync(0xffffffffu, base, 0);
            if (base + all > kBuffer) {
                if (lane == 0) atomicMin(&sm.valid[buf], base);
                return ~0u;
            }
            return base + upto - n;
        };
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

        // The values outside whole words: the first warp of the first CTA has one in each lane.
        const bool edge = cr == 0 && warp == 0 && lane < r.n_head + r.n_tail;
        const uint32_t edge_i = lane < r.n_head ? lane : r.n_head + r.words * kVec + (lane - r.n_head);
        const float edge_v = edge ? to_f32(r.x[edge_i]) : -INFINITY;
        auto offer_edge = [&]() -> bool {
            const bool want = edge && edge_v >= floor && key_of(edge_v, edge_i) >= least;
            const uint32_t at = room(want);
            if (want && at != ~0u) sm.buffer[buf][at] = key_of(edge_v, edge_i);
            return at != ~0u;
        };

        bool lost = false;  // keys of this warp found no room
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
                const Reach reach = reach_of(sm, order_bits(high), p.top);
                s.m = fmaxf(kLowest, order_value(reach.highest));
                // A thread without values has no say: where only its -inf is reached there is no bound.
                if (TOP && reach.bound > order_bits(-INFINITY)) {
                    least = static_cast<Key>(reach.bound) << 32;
                    floor = order_value(reach.bound);
                }
            }
            if (TOP && !lost && __any_sync(0xffffffffu, high >= floor)) {
                uint32_t want = 0;
#pragma unroll
                for (uint32_t j = 0; j < kValues; ++j) want |= uint32_t(v[j] >= floor) << j;
                want &= n_values < 32 ? (1u << n_values) - 1u : ~0u;
                uint32_t at = room(__popc(want));
                lost = at == ~0u;
                if (!lost)
                    for (; want; want &= want - 1) {
                        const uint32_t j = __ffs(want) - 1, w = j / kVec * kThreads;
                        sm.buffer[buf][at++] =
                            key_of(to_f32(reinterpret_cast<const T *>(words + w)[j % kVec]), r.n_head + (piece + w + threadIdx.x) * kVec + j % kVec);
                    }
            }
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(&sm.empty[st])) : "memory");
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
            if (TOP && piece == r.begin) {
                if (cr == 0 && warp == 0 && !lost) lost = !offer_edge();
                if (left > P && !sync_values_or(lost)) cut_now();
            }
        }
        const float next_xt = given_value(row + step, next_token);
        if (edge) {
            raise(edge_v);
            add2(make_float2(edge_v, -INFINITY), true);
            if (given) ahead += edge_v >= (edge_i < uint32_t(token) ? xt : above) && edge_i != uint32_t(token);
        }
        if (TOP && sync_values_or(lost || r.begin == r.end)) {
            // Once more for the keys: a word a thread at a time, value by value where one is wanted.
            if (threadIdx.x == 0) {
                sm.count[buf] = 0;
                sm.valid[buf] = kBuffer;
            }
            least = 1ull << 32;
            floor = -INFINITY;
            sync_values();
            const uint4 *body = reinterpret_cast<const uint4 *>(r.x + r.n_head);
#pragma unroll 1
            for (uint32_t w0 = r.begin; w0 < r.end; w0 += kThreads) {
                const uint32_t w = w0 + threadIdx.x;
                const T *x = reinterpret_cast<const T *>(body + w);
                bool any = false;
                for (uint32_t j = 0; j < kVec && w < r.end; ++j) any = any || key_of(to_f32(x[j]), r.n_head + w * kVec + j) >= least;
                if (!sync_values_or(any)) continue;
#pragma unroll 1
                for (uint32_t j = 0; j < kVec; ++j) {
                    const Key key = w < r.end ? key_of(to_f32(x[j]), r.n_head + w * kVec + j) : 0ull;
                    const bool want = key >= least;
                    const uint32_t at = room(want);
                    if (want && at != ~0u) sm.buffer[buf][at] = key;
                    sync_values();
                    if (sync_values_or(sm.count[buf] > kBuffer - kThreads)) cut_now();
                }
                cut_now();
            }
            if (cr == 0 && warp == 0) (void)offer_edge();
        }
        s.z = z2.x + z2.y;
        s.e = e2.x + e2.y;

        // Warp, CTA, cluster. (Of the references, a warp's largest; as order bits, for one instruction.)
        auto warp_join = [](Sums &a) {
            a.rescale(order_value(__reduce_max_sync(0xffffffffu, order_bits(a.m))));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                a.z += __shfl_xor_sync(0xffffffffu, a.z, o);
                a.e += __shfl_xor_sync(0xffffffffu, a.e, o);
            }
        };
        warp_join(s);
        ahead = __reduce_add_sync(0xffffffffu, ahead);
        if (lane == 0) {
            sm.m[warp] = s.m;
            sm.z[warp] = s.z;
            sm.e[warp] = s.e;
            sm.ahead[warp] = ahead;
        }
        if (TOP) {
            cut_now();
            if (threadIdx.x < p.top) sm.best[cr][threadIdx.x] = sm.buffer[buf][threadIdx.x];
        } else {
            sync_values();
        }
        if (warp == 0) {
            Sums t{lane < kWarps ? sm.m[lane] : kLowest, lane < kWarps ? sm.z[lane] : 0.f, lane < kWarps ? sm.e[lane] : 0.f};
            warp_join(t);
            const uint32_t n = __reduce_add_sync(0xffffffffu, lane < kWarps ? sm.ahead[lane] : 0u);
            if (lane == 0) {
                sm.cm[cr] = t.m;
                sm.cz[cr] = t.z;
                sm.ce[cr] = t.e;
                sm.cahead[cr] = n;
            }
        }
        if (p.cluster > 1) {
            sync_values();
            tc::cluster_wait();  // the first CTA runs by now
            // Every CTA sends its part to the first one.
            auto send = [&](const void *ptr, uint32_t v) {
                asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(tc::map_rank(smem_addr(ptr), 0)), "r"(v) : "memory");
            };
            if (cr != 0) {
                if (threadIdx.x == 0) {
                    send(&sm.cm[cr], __float_as_uint(sm.cm[cr]));
                    send(&sm.cz[cr], __float_as_uint(sm.cz[cr]));
                    send(&sm.ce[cr], __float_as_uint(sm.ce[cr]));
                    send(&sm.cahead[cr], sm.cahead[cr]);
                }
                if (TOP && threadIdx.x < 2 * p.top) {
                    const uint32_t *word = reinterpret_cast<const uint32_t *>(sm.best[cr]) + threadIdx.x;
                    send(word, *word);
                }
            }
            tc::cluster_sync();
            if (cr != 0) return;  // one row per cluster
        }
        const Key *best = sm.best[0];
        if (TOP && p.cluster > 1) {
            // Each key's place is the sum of its places in the CTAs' lists, which are in order.
            for (uint32_t k = threadIdx.x; k < p.cluster * OPURE_SCORE_MAX_TOP; k += kThreads) {
                const uint32_t own = k % OPURE_SCORE_MAX_TOP, list = k / OPURE_SCORE_MAX_TOP;
                const Key key = own < p.top ? sm.best[list][own] : 0ull;
                if (!key) continue;
                uint32_t place = 0;
#pragma unroll
                for (uint32_t c = 0; c < kMaxCluster; ++c) {
                    if (c >= p.cluster) continue;
                    uint32_t larger = 0;
#pragma unroll
                    for (uint32_t half = OPURE_SCORE_MAX_TOP / 2; half > 0; half /= 2)
                        if (larger + half <= p.top && sm.best[c][larger + half - 1] > key) larger += half;
                    if (larger < p.top && sm.best[c][larger] > key) ++larger;
                    place += larger;
                }
                if (place < p.top) sm.buffer[1][place] = key;
            }
            uint32_t n_keys = 0;  // fewer than top: none behind them
            for (uint32_t c = 0; c < p.cluster; ++c) n_keys += __popc(__ballot_sync(0xffffffffu, lane < p.top && sm.best[c][lane] != 0));
            if (threadIdx.x >= n_keys && threadIdx.x < p.top) sm.buffer[1][threadIdx.x] = 0ull;
            sync_values();
            best = sm.buffer[1];
        }
        if (warp == 0) {
            __syncwarp();
            Sums t{sm.cm[0], sm.cz[0], sm.ce[0]};
            uint32_t n = sm.cahead[0];
            for (uint32_t c = 1; c < p.cluster; ++c) {
                t.join(Sums{sm.cm[c], sm.cz[c], sm.ce[c]});
                n += sm.cahead[c];
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
                    if (p.rank) p.rank[row] = given ? int32_t(n) : 0;
                }
            }
            if (TOP && lane < p.top) {
                const Key key = best[lane];
                const size_t at = size_t(row) * p.top + lane;
                p.top_tokens[at] = key ? int32_t(0xffffffffu - uint32_t(key)) : -1;
                p.top_logprobs[at] = key ? log_prob(order_value(uint32_t(key >> 32))) : -INFINITY;
            }
        }
        sync_values();  // the next row writes what this one's results were read from
        token = next_token;
        xt = next_xt;
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
        cfg.blockDim = dim3(kThreads + 32);
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
