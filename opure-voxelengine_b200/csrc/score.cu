// score.cu -- log probabilities of given tokens, their ranks, entropies and the most likely tokens
// of rows of logits, in one pass (opure_token_scores).
//
// A thread keeps a reference m, z = sum exp(x - m) and e = sum exp(x - m) (x - m) over its logits x;
// m is raised, and the sums rescaled, only when a logit passes it by 5. The row's log-sum-exp is then
// m + log z, its entropy log z - e / z. A warp keeps its best 32 tokens as keys (orderable value,
// ~index), one per lane, largest first; a logit is looked at again only when it reaches a bound that
// at least `top` tokens of the row are known to reach: each of the W warps publishes a value that
// ceil(top / W) of its logits reach (from the lanes' maxima of its first loads, then from its list), and
// the smallest of these is the bound.
//
// Rows are shared out over a CTA, or over a cluster of up to 8 where there are few of them; the
// parts meet in shared memory (distributed over the cluster).
#include <algorithm>

#include "kv4.cuh"
#include "tcgen05.cuh"

namespace opure {
namespace {

constexpr uint32_t kThreads = 512, kWarps = kThreads / 32;
constexpr uint32_t kMaxCluster = 8;
constexpr float kRaise = 5.f;
constexpr float kLowest = -3.4028234663852886e38f;  // of fp32: a row may hold nothing larger
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kFar = -200.f;                       // exp of it is 0, and 0 times it stays 0 (unlike -inf)

struct ScoreParams {
    const void *logits;
    uint32_t vocab, cluster;
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

struct RowShared {
    float m[kWarps], z[kWarps], e[kWarps];
    uint32_t ahead[kWarps];
    uint32_t bound[kWarps];                                   // order bits of each warp's ceil(top / W)-th best
    unsigned long long keys[kWarps][OPURE_SCORE_MAX_TOP];      // each warp's best
    unsigned long long best[kMaxCluster][OPURE_SCORE_MAX_TOP];  // each CTA's best (rank 0's copy is used)
    float cm[kMaxCluster], cz[kMaxCluster], ce[kMaxCluster];
    uint32_t cahead[kMaxCluster];
};

// A warp's list of best keys, lane i the i-th; a new key goes in where it belongs.
__device__ __forceinline__ void insert(unsigned long long &mine, unsigned long long key, uint32_t lane) {
    const uint32_t before = __popc(__ballot_sync(0xffffffffu, mine > key));
    const unsigned long long up = __shfl_up_sync(0xffffffffu, mine, 1);
    if (lane == before) mine = key;
    if (lane > before) mine = up;
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kThreads, 2) score_kernel(ScoreParams p) {
    constexpr uint32_t kVec = 16 / sizeof(T), kBatch = 4;  // values of a load, loads in flight
    __shared__ RowShared sm;
    grid_dependency_wait();
    grid_dependents_launch();
    const uint32_t cr = p.cluster > 1 ? tc::cluster_rank() : 0u;
    const uint32_t row = blockIdx.x / p.cluster, warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const T *x = static_cast<const T *>(p.logits) + size_t(row) * p.stride;
    if (TOP && threadIdx.x < kWarps) sm.bound[threadIdx.x] = 0u;
    const int32_t token = p.tokens ? p.tokens[row] : -1;
    const bool given = token >= 0 && uint32_t(token) < p.vocab;
    const float xt = given ? to_f32(x[token]) : 0.f;
    // The smallest value that counts as ahead of xt: itself before the token, the next above it after.
    const float above = xt != xt ? xt : order_value(order_bits(xt) + 1u);
    const uint32_t published = (p.top + kWarps - 1) / kWarps;  // the place that each warp publishes
    if (p.cluster > 1) tc::cluster_arrive();  // met again before anything goes to another CTA
    if (TOP) __syncthreads();

    Sums s{kLowest, 0.f, 0.f};
    float2 z2 = make_float2(0.f, 0.f), e2 = z2;  // s.z and s.e in two parts
    uint32_t ahead = 0;
    unsigned long long mine = 0ull;

    // One value of each lane (all lanes call it): sums, rank, best list.
    auto offer = [&](float v, uint32_t i, bool valid) {
        uint32_t cand = __ballot_sync(0xffffffffu, valid && v == v);
        while (cand) {
            const uint32_t src = __ffs(cand) - 1;
            cand &= cand - 1;
            const float cv = __shfl_sync(0xffffffffu, v, src);
            const uint32_t ci = __shfl_sync(0xffffffffu, i, src);
            const unsigned long long key = static_cast<unsigned long long>(order_bits(cv)) << 32 | (0xffffffffu - ci);
            if (key > __shfl_sync(0xffffffffu, mine, p.top - 1)) insert(mine, key, lane);
        }
    };
    auto add2 = [&](float2 v) {
        float2 d = __fadd2_rn(v, make_float2(-s.m, -s.m));
        d.x = max_nan(d.x, kFar);
        d.y = max_nan(d.y, kFar);
        const float2 f = make_float2(exp_fast(d.x), exp_fast(d.y));
        z2 = __fadd2_rn(z2, f);
        e2 = __ffma2_rn(f, d, e2);
    };
    auto raise = [&](float v) {  // v: the largest of the values to come
        if (v > s.m + kRaise) {
            s.z = z2.x + z2.y;
            s.e = e2.x + e2.y;
            s.rescale(v);
            z2 = make_float2(s.z, 0.f);
            e2 = make_float2(s.e, 0.f);
        }
    };

    auto unpack = [](const uint4 &raw, float (&v)[kVec]) {
        if constexpr (sizeof(T) == 4) {
            v[0] = __uint_as_float(raw.x); v[1] = __uint_as_float(raw.y);
            v[2] = __uint_as_float(raw.z); v[3] = __uint_as_float(raw.w);
        } else {
            const T *h = reinterpret_cast<const T *>(&raw);
#pragma unroll
            for (uint32_t j = 0; j < kVec; ++j) v[j] = to_f32(h[j]);
        }
    };
    // Head and tail values outside whole aligned 16-byte words, then this CTA's share of the words.
    const uint32_t mis = uint32_t(reinterpret_cast<uintptr_t>(x) % 16 / sizeof(T));
    const uint32_t n_head = min(mis ? kVec - mis : 0u, p.vocab), words = (p.vocab - n_head) / kVec, n_tail = p.vocab - n_head - words * kVec;
    if (cr == 0 && warp == 0) {
        const bool valid = lane < n_head + n_tail;
        const uint32_t i = lane < n_head ? lane : n_head + words * kVec + (lane - n_head);
        const float v = valid ? to_f32(x[i]) : 0.f;
        if (valid) {
            raise(v);
            add2(make_float2(v, -INFINITY));
            if (given) ahead += v >= (i < uint32_t(token) ? xt : above) && i != uint32_t(token);
        }
        if (TOP) offer(v, i, valid);
    }
    const uint4 *body = reinterpret_cast<const uint4 *>(x + n_head);
    const uint32_t share = (words + p.cluster - 1) / p.cluster, w_begin = min(cr * share, words), w_end = min(w_begin + share, words);
    const uint32_t token_word = given && uint32_t(token) >= n_head ? (uint32_t(token) - n_head) / kVec : given ? 0u : words;
    const uint32_t rounds = (w_end - w_begin + kThreads * kBatch - 1) / (kThreads * kBatch);
    for (uint32_t round = 0; round < rounds; ++round) {
        const uint32_t w0 = w_begin + round * kThreads * kBatch + threadIdx.x;
        uint4 raw[kBatch];
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
            const uint32_t w = w0 + b * kThreads;
            raw[b] = w < w_end ? ldg_stream(body + w) : make_uint4(0, 0, 0, 0);
        }
        float high[kBatch];  // the largest value of each load; -inf where there is none
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
            float v[kVec];
            unpack(raw[b], v);
            high[b] = v[0];
#pragma unroll
            for (uint32_t j = 1; j < kVec; ++j) high[b] = fmaxf(high[b], v[j]);
            if (w0 + b * kThreads >= w_end) high[b] = -INFINITY;
        }
        uint32_t least = 0;
        if (TOP) {
            if (round == 0) {
                // Values that `published` (1 or 2) lanes reach.
                uint32_t o = order_bits(fmaxf(fmaxf(high[0], high[1]), fmaxf(high[2], high[3])));
                uint32_t reach = __reduce_max_sync(0xffffffffu, o);
                if (published > 1) {
                    if (lane == uint32_t(__ffs(__ballot_sync(0xffffffffu, o == reach))) - 1) o = 0;
                    reach = __reduce_max_sync(0xffffffffu, o);
                }
                // A lane without values has no say: its -inf is no token.
                if (lane == 0) sm.bound[warp] = reach > order_bits(-INFINITY) ? reach : 0u;
                __syncthreads();
            }
            const uint32_t bound = __reduce_min_sync(0xffffffffu, lane < kWarps ? *const_cast<volatile uint32_t *>(&sm.bound[lane]) : ~0u);
            least = max(bound, uint32_t(__shfl_sync(0xffffffffu, mine, p.top - 1) >> 32));
        }
#pragma unroll
        for (uint32_t b = 0; b < kBatch; ++b) {
            const uint32_t w = w0 + b * kThreads, i0 = n_head + w * kVec;
            const bool valid = w < w_end;
            float v[kVec];
            unpack(raw[b], v);
            if (valid) {
                raise(high[b]);
#pragma unroll
                for (uint32_t j = 0; j < kVec; j += 2) add2(make_float2(v[j], v[j + 1]));
                if (given) {
                    if (w != token_word) {
                        const float from = i0 < uint32_t(token) ? xt : above;
#pragma unroll
                        for (uint32_t j = 0; j < kVec; ++j) ahead += v[j] >= from;
                    } else {
#pragma unroll
                        for (uint32_t j = 0; j < kVec; ++j) ahead += v[j] >= (i0 + j < uint32_t(token) ? xt : above) && i0 + j != uint32_t(token);
                    }
                }
            }
            if (TOP && __any_sync(0xffffffffu, valid && order_bits(high[b]) >= least)) {
#pragma unroll
                for (uint32_t j = 0; j < kVec; ++j) offer(v[j], i0 + j, valid && order_bits(v[j]) >= least);
                const uint32_t reach = uint32_t(__shfl_sync(0xffffffffu, mine, published - 1) >> 32);
                if (lane == 0 && reach > sm.bound[warp]) *const_cast<volatile uint32_t *>(&sm.bound[warp]) = reach;
                least = max(least, uint32_t(__shfl_sync(0xffffffffu, mine, p.top - 1) >> 32));
            }
        }
    }
    s.z = z2.x + z2.y;
    s.e = e2.x + e2.y;

    // Warp, CTA, cluster.
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s.join(Sums{__shfl_xor_sync(0xffffffffu, s.m, o), __shfl_xor_sync(0xffffffffu, s.z, o), __shfl_xor_sync(0xffffffffu, s.e, o)});
    }
    ahead = __reduce_add_sync(0xffffffffu, ahead);
    if (lane == 0) {
        sm.m[warp] = s.m;
        sm.z[warp] = s.z;
        sm.e[warp] = s.e;
        sm.ahead[warp] = ahead;
    }
    if (TOP && lane < p.top) sm.keys[warp][lane] = mine;
    __syncthreads();
    if (TOP) {
        // Each key's place among all warps' keys; keys differ, but for 0, which stands for none.
        for (uint32_t t = threadIdx.x; t < kWarps * p.top; t += kThreads) {
            const unsigned long long key = sm.keys[t / p.top][t % p.top];
            uint32_t place = 0;
            for (uint32_t w = 0; w < kWarps; ++w)
                for (uint32_t q = 0; q < p.top; ++q) {
                    const unsigned long long other = sm.keys[w][q];
                    place += other > key || (other == key && w * p.top + q < t);
                }
            if (place < p.top) sm.best[cr][place] = key;
        }
    }
    if (warp == 0) {
        Sums t{lane < kWarps ? sm.m[lane] : kLowest, lane < kWarps ? sm.z[lane] : 0.f, lane < kWarps ? sm.e[lane] : 0.f};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
            t.join(Sums{__shfl_xor_sync(0xffffffffu, t.m, o), __shfl_xor_sync(0xffffffffu, t.z, o), __shfl_xor_sync(0xffffffffu, t.e, o)});
        const uint32_t n = __reduce_add_sync(0xffffffffu, lane < kWarps ? sm.ahead[lane] : 0u);
        if (lane == 0) {
            sm.cm[cr] = t.m;
            sm.cz[cr] = t.z;
            sm.ce[cr] = t.e;
            sm.cahead[cr] = n;
        }
    }
    __syncthreads();
    if (p.cluster > 1) {
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
        if (cr != 0) return;
    }
    Sums t{sm.cm[0], sm.cz[0], sm.ce[0]};
    uint32_t n = sm.cahead[0];
    for (uint32_t r = 1; r < p.cluster; ++r) {
        t.join(Sums{sm.cm[r], sm.cz[r], sm.ce[r]});
        n += sm.cahead[r];
    }
    const float lz = logf(t.z);
    const bool none = t.z == 0.f;  // a row of -inf alone
    auto log_prob = [&](float v) { return none ? NAN : (v - t.m) - lz; };
    if (threadIdx.x == 0) {
        if (p.lse) p.lse[row] = none ? -INFINITY : t.m + lz;
        if (p.entropy) p.entropy[row] = none ? NAN : lz - t.e / t.z;
        if (p.tokens) {
            if (token >= 0 && !given) report(p.st, OPURE_ERR_DEVICE_BOUNDS, 97, uint32_t(token));
            if (p.logprob) p.logprob[row] = given ? log_prob(xt) : token < 0 ? 0.f : NAN;
            if (p.rank) p.rank[row] = given ? int32_t(n) : 0;
        }
    }
    if (TOP) {
        const uint32_t total = p.cluster * p.top;
        for (uint32_t k = threadIdx.x; k < total; k += kThreads) {
            const unsigned long long key = sm.best[k / p.top][k % p.top];
            uint32_t place = 0;
            for (uint32_t r = 0; r < p.cluster; ++r)
                for (uint32_t q = 0; q < p.top; ++q) {
                    const unsigned long long other = sm.best[r][q];
                    place += other > key || (other == key && r * p.top + q < k);
                }
            if (place < p.top) {
                const size_t at = size_t(row) * p.top + place;
                p.top_tokens[at] = key ? int32_t(0xffffffffu - uint32_t(key)) : -1;
                p.top_logprobs[at] = key ? log_prob(order_value(uint32_t(key >> 32))) : -INFINITY;
            }
        }
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
    // A cluster per row while two CTAs per SM are not all taken, and each part has a batch of loads.
    uint32_t cluster = 1;
    const uint32_t batch = kThreads * 4 * (16 / type_bytes(a->type));
    while (cluster < kMaxCluster && uint64_t(a->rows) * cluster * 2 <= uint64_t(ctx->sm_count) * 2 && a->vocab / (cluster * 2) >= batch / 4)
        cluster *= 2;
    ScoreParams p{a->logits, a->vocab, cluster, a->stride, a->tokens, a->logprob, a->rank, a->entropy, a->lse,
                  a->top, a->top_tokens, a->top_logprobs, ctx->status};
    return with_type(a->type, [&](auto t) -> opure_status {
        using T = decltype(t);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(a->rows * cluster);
        cfg.blockDim = dim3(kThreads);
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
        OPURE_CUDA_TRY(cudaLaunchKernelEx(&cfg, a->top ? score_kernel<T, true> : score_kernel<T, false>, p));
        return OPURE_OK;
    });
}
