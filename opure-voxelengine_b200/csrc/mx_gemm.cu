// mx_gemm.cu -- the product of microscaled (MX) matrices: y[i][r] = sum_k x[i][k] w[r][k], with
// the linear layer's epilogues (store, residual add, SwiGLU with an MX result).
//
// With block b's scales sx and sw and its codes' values cx and cw,
//   y[i][r] = sum_b sx[i][b] sw[r][b] (sum_{k in b} cx[i][k] cw[r][k]),
// which is what tcgen05.mma kind::mxf8f6f4 computes 32 columns at a time, with fp32 sums: the
// tokens are its M side (128 TMEM lanes), weight rows its N side. 4-bit codes cross HBM and L2
// packed; TMA spreads them into the byte-wide slots that this kind reads.
//
// mx_gemm_kernel  one CTA per (128 tokens, 128 weight rows, K split). Warps 0 and 3 stream 128
//     columns a stage (codes by tiled TMA, scale tiles by bulk copies) into a ring of
//     shared-memory stages; warp 1 copies the scale tiles to TMEM and issues the MMAs. A K
//     split is a thread-block cluster whose CTAs share the epilogue: each sends its sums to the
//     CTAs that finish them (counted by the receiver's mbarrier), which add the splits in rank
//     order, so that results do not depend on timing. Few tokens' sums go from registers
//     (st.async); many are laid out in shared memory and go as one bulk copy per receiver, which
//     is several times as fast per byte but needs a cluster barrier before a CTA may leave
//     (8 splits of 64 tokens: 9.3 us against 11.2; of 3 tokens: 6.9 against 6.1). In SwiGLU a
//     tile is 64 gate rows and the 64 up rows that go with them.
// All waits are bounded (1 s); a timeout is reported in the ctx status word.
//
// Bound by latency: the first data is there 1,500 clocks after the launch, a stage takes 140 ns with
// 4 tokens and 250 ns with 64 (the tensor cores work on 128 token rows, 262 clocks, whatever their
// number), the epilogue 1,300 clocks. Measured: 64 x 6144 x 2048 to fp32 7.4 us, 37 x 1003 x 1100
// with 4-bit tokens to bf16 5.3 us, SwiGLU of 64 x 16384 x 2048 8.5 us.
#include <algorithm>
#include <type_traits>

#include "mx_gemm.cuh"

namespace opure {
namespace {

constexpr uint32_t kM = 128;       // tokens per tile = TMEM lanes
constexpr uint32_t kN = 128;       // weight rows per tile
constexpr uint32_t kK = 128;       // columns per stage: one 128-byte swizzled row of byte slots
constexpr uint32_t kThreads = 256;
constexpr uint32_t kMaxStages = 10;
constexpr uint32_t kMaxSplits = 8;  // portable cluster size
constexpr uint32_t kDirect = 16;    // tokens whose sums go straight from registers
constexpr uint32_t kPrefetch = 8;   // stages of weights that are asked for ahead
constexpr uint32_t kBBytes = kN * kK;
constexpr uint32_t kScaleBytes = 2048;  // per stage: x tile, w (or gate) tile, up tile; keeps 1 KB alignment
constexpr uint32_t kScaleCols = 12;     // TMEM columns of a stage's scales
constexpr uint32_t kTmemCols = 256;
constexpr size_t kHalfSmem = 112 * 1024;  // dynamic shared memory of two CTAs on an SM
constexpr uint32_t kUnit = 512;           // partial sums of 4 tokens x 32 columns, bytes
static_assert(kN + kMaxStages * kScaleCols <= kTmemCols, "TMEM columns");

struct GemmParams {
    const uint8_t *ws, *us, *xs;  // scale tiles: weights (or gate rows), up rows, tokens
    uint32_t n, rows, kblocks, splits, stages;
    uint32_t a_rows;              // token rows that a stage holds: multiple of 8, at most 128
    uint32_t half;                // SwiGLU: first up row = result columns
    uint32_t sums_offset;         // of the received sums from the ring's start
    bool apart;                   // they are past the ring
    bool vec;                     // rows of y and residual allow accesses of 4 values
    uint32_t x_format;
    void *y;
    size_t y_stride;
    const void *residual;
    uint8_t *out, *outs;          // SwiGLU
    DeviceStatus *st;
};

// T: the type of y, or for SwiGLU uint8_t (E4M3) or uint32_t (E2M1).
template <int EPI, typename T>
__global__ void __launch_bounds__(kThreads, 2)
    mx_gemm_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap, GemmParams p) {
    constexpr bool kSwiglu = EPI == OPURE_EPI_SWIGLU;
    constexpr uint32_t kTileRows = kSwiglu ? kN / 2 : kN;  // result columns per tile
    constexpr uint32_t kChunks = kTileRows / 32, kSides = kSwiglu ? 2 : 1;
    extern __shared__ uint8_t dsm[];
    __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], done, recv;
    __shared__ uint32_t tmem_base;
    __shared__ uint32_t issued_s[2], consumed_s;
    __shared__ int fail;

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t tile = blockIdx.x / p.splits, split = blockIdx.x % p.splits;
    const uint32_t m0 = blockIdx.y * kM, r0 = tile * kTileRows;
    const uint32_t kb0 = uint32_t(uint64_t(p.kblocks) * split / p.splits);
    const uint32_t nk = uint32_t(uint64_t(p.kblocks) * (split + 1) / p.splits) - kb0;
    const uint32_t a_bytes = p.a_rows * kK, stage_bytes = kBBytes + kScaleBytes + a_bytes;
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(dsm) + 1023) & ~uintptr_t(1023));
    // Stage: [A][B 16 KB][scales 2 KB]. The MMA reads 128 rows of A whatever a_rows is; rows past
    // a_rows are the stage's B and only reach accumulator lanes of tokens that are not there.
    auto a_tile = [&](uint32_t s) { return base + size_t(s) * stage_bytes; };
    auto b_tile = [&](uint32_t s) { return base + size_t(s) * stage_bytes + a_bytes; };
    auto sf_tile = [&](uint32_t s) { return base + size_t(s) * stage_bytes + a_bytes + kBBytes; };
    // Results in units of 4 tokens x 32 columns (and 2 sides in SwiGLU). Unit u is finished by CTA
    // u % splits, as its unit u / splits. Every CTA lays its sums out by receiver (`mine`, in the
    // ring's place) and sends each its part, which arrives in that one's `sums`, one part per split:
    // past the ring where there is room, else after `mine`, and the splits wait for one another
    // before they send. Without splits sums is mine. A token's eight pieces of 16 bytes stand in an
    // order of its own (piece ^ token % 8), so that 32 tokens' stores spread over all banks.
    uint8_t *mine = base, *sums = base + p.sums_offset;
    const uint32_t n = min(p.n - m0, kM), units = (n + 3) / 4 * kChunks;
    const uint32_t own_units = (units + p.splits - 1 - split) / p.splits;
    const uint32_t part_bytes = (units + p.splits - 1) / p.splits * kSides * kUnit;  // room per split

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < p.stages; ++s) {
            mbar_init(&full[s], 2);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&done, 1);
        mbar_init(&recv, 1);
        if (p.splits > 1) mbar_expect_tx(&recv, own_units * p.splits * kSides * kUnit);
        fail = 0;
        issued_s[0] = issued_s[1] = consumed_s = 0;
        tc::prefetch_map(&wmap);
        tc::prefetch_map(&xmap);
    }
    if (warp == 2) tc::alloc(&tmem_base, kTmemCols);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = tmem_base;
    // The weights may be asked for before the kernel that this one waits for has ended.
    if (warp == 0) {
        const bool one = tc::elect();
        for (uint32_t i = 0; i < min(nk, kPrefetch); ++i) {
            tc::prefetch_2d(one, &wmap, (kb0 + i) * kK, r0);
            if (kSwiglu) tc::prefetch_2d(one, &wmap, (kb0 + i) * kK, p.half + r0);
        }
    }
    if (p.splits > 1 && p.apart) tc::cluster_arrive();  // this CTA can receive
    grid_dependency_wait();
    grid_dependents_launch();

    if (warp == 0 || warp == 3) {
        // Warp 0 loads the weights, warp 3 the tokens.
        const bool one = tc::elect();
        uint32_t s = 0, phase = 1, i = 0;
        for (; i < nk; ++i) {
            if (i >= p.stages && !mbar_wait(&empty[s], phase)) {
                if (one) report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 80, blockIdx.x);
                fail = 1;
                break;
            }
            const uint32_t kb = kb0 + i;
            if (warp == 0) {
                // A spreading copy counts the bytes that it reads, not the slots that it fills.
                tc::expect_tx(one, &full[s], kBBytes / 2 + kMxTileBytes * (kSwiglu ? 2 : 1));
                tc::load_2d(one, b_tile(s), &wmap, kb * kK, r0, &full[s]);
                if (kSwiglu) tc::load_2d(one, b_tile(s) + kBBytes / 2, &wmap, kb * kK, p.half + r0, &full[s]);
                const size_t tile = (size_t(r0 / 128) * p.kblocks + kb) * kMxTileBytes;
                tc::bulk(one, sf_tile(s) + 512, p.ws + tile, kMxTileBytes, &full[s]);
                if (kSwiglu) tc::bulk(one, sf_tile(s) + 1024, p.us + tile, kMxTileBytes, &full[s]);
            } else {
                tc::expect_tx(one, &full[s], a_bytes * p.x_format / 8 + kMxTileBytes);
                tc::load_2d(one, a_tile(s), &xmap, kb * kK, m0, &full[s]);
                tc::bulk(one, sf_tile(s), p.xs + (size_t(m0 / 128) * p.kblocks + kb) * kMxTileBytes, kMxTileBytes, &full[s]);
            }
            if (++s == p.stages) {
                s = 0;
                phase ^= 1;
            }
        }
        if (one) issued_s[warp / 3] = i;
    } else if (warp == 1) {
        const bool one = tc::elect();
        const uint32_t idesc =
            tc::idesc_mx(p.x_format == OPURE_MX_FP8 ? tc::kE4M3 : tc::kE2M1, tc::kE2M1, kM, kSwiglu ? kN / 2 : kN);
        // In SwiGLU a tile's 64 rows are the first or the second half of their scale tile.
        const uint32_t shift = kSwiglu ? r0 / 32 % 4 : 0, tbase = __shfl_sync(0xffffffffu, tmem, 0);
        uint32_t s = 0, phase = 0, i = 0;
        for (; i < nk; ++i) {
            if (!mbar_wait(&full[s], phase)) {
                if (one) report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 81, blockIdx.x);
                fail = 1;
                break;
            }
            tc::fence_after();
            // Each stage has TMEM columns of its own for its scales, so a copy never meets an
            // MMA that still reads them: the stage was freed by that MMA's commit.
            const uint32_t sf = tbase + kN + s * kScaleCols;
            const uint64_t ds = tc::desc_scales(smem_addr(sf_tile(s)));
            const uint64_t da = tc::desc_sw128(smem_addr(a_tile(s))), db = tc::desc_sw128(smem_addr(b_tile(s)));
            tc::copy_scales(one, sf, ds);
            tc::copy_scales(one, sf + 4, ds + (512 >> 4));
            if (kSwiglu) tc::copy_scales(one, sf + 8, ds + (1024 >> 4));
#pragma unroll
            for (uint32_t k = 0; k < kK / 32; ++k) {
                const uint32_t id = idesc | tc::idesc_block(k), acc = (i | k) != 0;
                tc::mma_mxf8f6f4(one, tbase, da + 2 * k, db + 2 * k, id, sf, sf + 4 + shift, acc);
                if (kSwiglu)
                    tc::mma_mxf8f6f4(one, tbase + kN / 2, da + 2 * k, db + 2 * k + (kBBytes / 2 >> 4), id, sf, sf + 8 + shift, acc);
            }
            tc::commit(one, &empty[s]);
            if (i + 1 == nk) tc::commit(one, &done);
            if (++s == p.stages) {
                s = 0;
                phase ^= 1;
            }
        }
        consumed_s = i;
    }
    if (!mbar_wait(&done, 0)) {
        report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 82, blockIdx.x);
        fail = 1;
    }
    tc::fence_after();
    __syncthreads();
    const bool failed = fail;
    if (failed && threadIdx.x == 0)  // leave no copy in flight into this CTA's shared memory
        for (uint32_t i = consumed_s; i < max(issued_s[0], issued_s[1]); ++i) mbar_wait(&full[i % p.stages], (i / p.stages) & 1u);

    // Accumulators -> `mine`, or to the receivers. Warps w and w + 4 share TMEM lanes 32 (w % 4) ..
    // (tokens); each takes half of the columns.
    const bool direct = p.splits > 1 && n <= kDirect;
    if (p.splits > 1 && !p.apart) tc::cluster_arrive();
    if (direct) tc::cluster_wait();
    const uint32_t quarter = warp & 3u, part = warp >> 2, token = quarter * 32 + lane;
    if (!failed && quarter * 32 < n) {
#pragma unroll
        for (uint32_t c = 0; c < 2; ++c) {
            uint32_t r[32];
            tc::ld32(tmem + ((quarter * 32) << 16) + part * (kN / 2) + c * 32, r);
            tc::wait_ld();
            if (token < (n + 3) / 4 * 4) {
                const uint32_t u = token / 4 * kChunks + (kSwiglu ? c : part * 2 + c), to = u % p.splits;
                const uint32_t at = (u / p.splits * kSides + (kSwiglu ? part : 0)) * kUnit + token % 4 * 128;
                if (direct) {
                    const uint32_t dst = tc::map_rank(smem_addr(sums + split * part_bytes + at), to), bar = tc::map_rank(smem_addr(&recv), to);
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j)
                        tc::st_async_f4(dst + ((j ^ (lane & 7u)) << 4), r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3], bar);
                } else {
                    uint8_t *dst = mine + to * part_bytes + at;
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j)
                        *reinterpret_cast<uint4 *>(dst + ((j ^ (lane & 7u)) << 4)) =
                            make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
                }
            }
        }
    }
    bool got = !failed;
    if (!direct) {
        tc::fence_async_shared();
        __syncthreads();
    }
    if (p.splits > 1) {
        if (!direct) {
            tc::cluster_wait();
            if (!failed && threadIdx.x < p.splits) {
                const uint32_t to = threadIdx.x, bytes = (units + p.splits - 1 - to) / p.splits * kSides * kUnit;
                if (bytes)
                    tc::bulk_send(tc::map_rank(smem_addr(sums + split * part_bytes), to), mine + to * part_bytes, bytes,
                                  tc::map_rank(smem_addr(&recv), to));
            }
        }
        got = mbar_wait(&recv, 0);
        if (!got && threadIdx.x == 0) report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 83, blockIdx.x);
        got = __all_sync(0xffffffffu, got);
        if (!direct) tc::cluster_arrive();  // has all that was sent to it
    }

    // Epilogue: a warp takes a unit, a lane 4 columns of a token.
    for (uint32_t l = warp; got && l < own_units; l += kThreads / 32) {
        const uint32_t u = l * p.splits + split, token0 = u / kChunks * 4, col0 = r0 + u % kChunks * 32;
        if constexpr (!kSwiglu) {
            if (!p.vec) {
                // Unaligned rows: a lane one column of each token, so that neighbouring lanes touch
                // neighbouring values.
                const uint32_t col = col0 + lane;
                const size_t at = (m0 + token0) * p.y_stride + col;
                const uint32_t tokens = col < p.rows ? columns_left(n, token0) : 0;
                float res[4] = {};
                if constexpr (EPI == OPURE_EPI_ADD)
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k)
                        if (k < tokens) res[k] = to_f32(static_cast<const T *>(p.residual)[at + k * p.y_stride]);
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) {
                    const uint8_t *src = sums + l * kUnit + k * 128 + (((lane >> 2) ^ ((token0 + k) & 7u)) << 4) + (lane & 3u) * 4;
                    float v = 0.f;
                    for (uint32_t q = 0; q < p.splits; ++q) v += *reinterpret_cast<const float *>(src + q * part_bytes);
                    if (k < tokens) static_cast<T *>(p.y)[at + k * p.y_stride] = from_f32<T>(v + res[k]);
                }
                continue;
            }
        }
        const uint32_t i = m0 + token0 + lane / 8, col = col0 + lane % 8 * 4;
        const uint32_t piece = lane / 8 * 128 + ((lane ^ (token0 + lane / 8)) & 7u) * 16;
        float v[kSides][4] = {};
#pragma unroll
        for (uint32_t q = 0; q < kMaxSplits; ++q) {
            if (q >= p.splits) break;
#pragma unroll
            for (uint32_t s = 0; s < kSides; ++s) {
                const float4 f = lds_f4(reinterpret_cast<const float *>(sums + q * part_bytes + (l * kSides + s) * kUnit + piece));
                v[s][0] += f.x; v[s][1] += f.y; v[s][2] += f.z; v[s][3] += f.w;
            }
        }
        if constexpr (kSwiglu) {
            constexpr uint32_t kF = sizeof(T) == 1 ? OPURE_MX_FP8 : OPURE_MX_FP4;
#pragma unroll
            for (uint32_t j = 0; j < 4; j += 2) swiglu2(v[0][j], v[0][j + 1], v[1][j], v[1][j + 1]);
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j)
                if (col + j >= p.half) v[0][j] = 0.f;  // gate rows past the half are up rows
            store_block<kF>(v[0], p.out + i * mx_row_bytes(kF, p.half) + size_t(col0) * kF / 8,
                            p.outs + mx_scale_offset(p.half, i, col0 / 32), i < p.n && col0 < mx_kp(p.half));
        } else if (i < p.n) {
            const size_t at = i * p.y_stride + col;
            store_quad<EPI>(v[0], static_cast<T *>(p.y) + at, static_cast<const T *>(p.residual) + at, columns_left(p.rows, col));
        }
    }
    tc::fence_before();
    __syncthreads();
    if (warp == 2) tc::dealloc(tmem, kTmemCols);
    // A CTA leaves when what it sent by bulk copies has arrived (or its receiver gave up). Registers
    // need no such wait, unless this CTA gave up: then the others may still send to it.
    if (p.splits > 1 && !direct) tc::cluster_wait();
    if (direct && !__syncthreads_and(got)) tc::cluster_sync();
}

// Scale tiles of the two halves of a matrix, each as a matrix of its own, one after the other:
// what SwiGLU on the tensor cores needs when the second half does not start on a tile. One thread per (row, 128
// columns).
__global__ void __launch_bounds__(256) mx_split_scales_kernel(const uint8_t *src, uint8_t *dst, uint32_t half, uint32_t kblocks) {
    grid_dependency_wait();
    grid_dependents_launch();
    const uint64_t t = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x;
    const uint32_t kb = uint32_t(t / (2 * half)), r = uint32_t(t - uint64_t(kb) * (2 * half));
    if (kb >= kblocks) return;
    const uint32_t cols = kblocks * 128;
    if (r >= half) dst += size_t((half + 127) / 128) * kblocks * kMxTileBytes;
    *reinterpret_cast<uint32_t *>(dst + mx_scale_offset(cols, r >= half ? r - half : r, kb * 4)) =
        *reinterpret_cast<const uint32_t *>(src + mx_scale_offset(cols, r, kb * 4));
}

// ---- host -------------------------------------------------------------------------------
// K splits, at most one CTA per SM, by the least estimated time (returned, in ns). Measured on one
// B200: a stage takes 270 ns (SwiGLU, with twice the MMAs, 400), with two CTAs on an SM 670 for
// both; launch, first loads and a plain epilogue 6 us, SwiGLU's 9; joining splits 1 us and, as all
// SMs exchange more sums, up to 8 us more for 128 tokens on every SM.
uint64_t choose_splits(GemmParams &p, uint64_t tiles, bool swiglu, uint32_t sms) {
    const uint64_t waves = (tiles + 2 * sms - 1) / (2 * sms), n = std::min(p.n, kM);
    const uint64_t stage = tiles > sms ? (swiglu ? 1000 : 670) : swiglu ? 400 : 270;
    uint64_t best = ~uint64_t(0);
    for (uint32_t s = 1; s == 1 || (s <= std::min(kMaxSplits, p.kblocks) && s * tiles <= sms); ++s) {
        const uint64_t ctas = s * tiles, join = s > 1 ? 1000 + n * ctas * ctas * 8000 / (uint64_t(kM) * sms * sms) : 0;
        const uint64_t ns = 4000 + waves * (ceil_div(p.kblocks, s) * stage + (swiglu ? 5000 : 2000) + join);
        if (ns < best) {
            best = ns;
            p.splits = s;
        }
    }
    return best;
}

template <int EPI, typename T>
opure_status launch_gemm(opure_ctx *ctx, const CUtensorMap &wm, const CUtensorMap &xm, const GemmParams &p, uint32_t tiles,
                         size_t smem) {
    auto *kernel = mx_gemm_kernel<EPI, T>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e != cudaSuccess) return cuda_status(e);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(tiles * p.splits, (p.n + kM - 1) / kM);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = p.splits;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = ctx->pdl ? 2 : 1;
    e = cudaLaunchKernelEx(&cfg, kernel, wm, xm, p);
    return e == cudaSuccess ? OPURE_OK : cuda_status(e);
}

}  // namespace
}  // namespace opure

using namespace opure;

extern "C" {

opure_status opure_mx_gemm(opure_ctx *ctx, const opure_mx_gemm_args *a) {
    opure_status s = enter(ctx);
    if (s) return s;
    if (!a || !mx_valid(a->w) || !mx_valid(a->x) || a->w.cols != a->x.cols) return OPURE_ERR_INVALID_ARG;
    if (a->w.format != OPURE_MX_FP4) return OPURE_ERR_UNSUPPORTED;
    const bool swiglu = a->epilogue == OPURE_EPI_SWIGLU;
    if (swiglu) {
        if (a->w.rows % 2 || !mx_valid(a->out) || a->out.rows != a->x.rows || a->out.cols != a->w.rows / 2)
            return OPURE_ERR_INVALID_ARG;
    } else if (a->epilogue == OPURE_EPI_STORE || a->epilogue == OPURE_EPI_ADD) {
        if (!type_aligned(a->y, a->y_type) || a->y_stride < a->w.rows) return OPURE_ERR_INVALID_ARG;
        if (a->epilogue == OPURE_EPI_ADD && !type_aligned(a->residual, a->y_type)) return OPURE_ERR_INVALID_ARG;
    } else {
        return a->epilogue == OPURE_EPI_ARGMAX ? OPURE_ERR_UNSUPPORTED : OPURE_ERR_INVALID_ARG;
    }
    if (a->x.rows == 0 || a->w.rows == 0) return OPURE_OK;
    if (!swiglu && (!a->y || (a->epilogue == OPURE_EPI_ADD && !a->residual))) return OPURE_ERR_INVALID_ARG;

    GemmParams p{};
    p.n = a->x.rows;
    p.rows = a->w.rows;
    p.half = a->w.rows / 2;
    p.kblocks = mx_kp(a->w.cols) / kK;
    p.x_format = a->x.format;
    p.ws = a->w.scales;
    p.xs = a->x.scales;
    p.y = a->y;
    p.y_stride = a->y_stride;
    p.residual = a->residual;
    p.out = a->out.codes;
    p.outs = a->out.scales;
    p.st = ctx->status;
    // Grid dimensions and TMA's 32-bit signed coordinates.
    if (p.n > 65535u * kM || p.rows > (1u << 30) || a->w.cols > (1u << 30)) return OPURE_ERR_UNSUPPORTED;
    if (mx_gemv_suits(a)) return mx_gemv(ctx, a);
    const uint32_t tiles = swiglu ? mx_kp(p.half) / (kN / 2) : ceil_div(p.rows, kN);
    const uint32_t mtiles = ceil_div(p.n, kM);
    const uint64_t here_ns = choose_splits(p, uint64_t(tiles) * mtiles, swiglu, uint32_t(ctx->sm_count));
    p.a_rows = std::min(kM, (p.n + 7) & ~7u);
    const uint32_t stage_bytes = kBBytes + kScaleBytes + p.a_rows * kK;
    // Before the ring 1 KB to align it, after it the rest of the last stage's 128 rows of A and, where
    // that leaves the ring 4 stages or all that it needs, the received sums; else these and the sums
    // to send take the ring's place.
    const uint32_t chunks = swiglu ? kN / 64 : kN / 32, units = ceil_div(std::min(p.n, kM), 4) * chunks;
    const size_t sums = size_t(ceil_div(units, p.splits)) * p.splits * (swiglu ? 2 : 1) * kUnit;
    // Two CTAs per SM (TMEM's 512 columns allow it and, above 75 KB each, no third), so that the
    // next kernel's CTAs set up while this one's work: a chain of 8-token 8192 -> 2048 products
    // took 5.8 us a call with half of the shared memory each, 9.7 us with all of it. Only the sums
    // of more than 100 tokens with splits need more than half.
    auto stages_in = [&](size_t bytes) {
        return std::min<uint32_t>({kMaxStages, uint32_t((bytes - 1024) / stage_bytes), ceil_div(p.kblocks, p.splits)});
    };
    p.stages = stages_in(kHalfSmem);
    p.apart = p.splits > 1 && sums < kHalfSmem / 2 && stages_in(kHalfSmem - sums) >= std::min(4u, p.stages);
    if (p.apart) p.stages = stages_in(kHalfSmem - sums);
    const size_t ring = size_t(p.stages) * stage_bytes;
    p.sums_offset = p.splits == 1 ? 0 : uint32_t(p.apart ? std::max(ring, sums) : sums);
    const size_t smem = std::max<size_t>({1024 + ring, 1024 + p.sums_offset + sums, 80 * 1024});
    p.vec = rows_aligned16(a->y, a->y_type, a->y_stride) && rows_aligned16(a->residual, a->y_type, a->y_stride);
    if (swiglu) {
        const size_t side = opure_mx_scale_bytes(p.half, a->w.cols);
        if (p.half % 128) {
            if (2 * side > kScratchBytes) return OPURE_ERR_UNSUPPORTED;
            uint8_t *split = static_cast<uint8_t *>(ctx->ws);
            s = launch(ctx, mx_split_scales_kernel, dim3(ceil_div(uint64_t(p.rows) * p.kblocks, 256)), dim3(256), 0, true, p.ws, split,
                       p.half, p.kblocks);
            if (s) return s;
            p.ws = split;
        }
        p.us = p.ws + side;
    }
    if (mx_gemm_pair_ns(ctx, a) < here_ns) return mx_gemm_pair(ctx, a, p.ws);
    CUtensorMap wm, xm;
    if (!make_slot_map(&wm, a->w, swiglu ? kN / 2 : kN) || !make_slot_map(&xm, a->x, p.a_rows)) return OPURE_ERR_UNSUPPORTED;
    if (swiglu)
        return a->out.format == OPURE_MX_FP4 ? launch_gemm<OPURE_EPI_SWIGLU, uint32_t>(ctx, wm, xm, p, tiles, smem)
                                             : launch_gemm<OPURE_EPI_SWIGLU, uint8_t>(ctx, wm, xm, p, tiles, smem);
    return with_type(a->y_type, [&](auto t) {
        using T = decltype(t);
        return a->epilogue == OPURE_EPI_ADD ? launch_gemm<OPURE_EPI_ADD, T>(ctx, wm, xm, p, tiles, smem)
                                            : launch_gemm<OPURE_EPI_STORE, T>(ctx, wm, xm, p, tiles, smem);
    });
}

}  // extern "C"
