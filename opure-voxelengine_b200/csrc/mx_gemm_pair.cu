// mx_gemm_pair.cu -- the product of microscaled matrices for many tokens: persistent pairs of
// SMs (cta_group::2), each working through tiles of 256 tokens x 256 weight rows.
//
// Bound by the tensor cores. With 8-bit tokens the weights' 4-bit codes are spread into byte
// slots by TMA (kind::mxf8f6f4, 128 columns a stage); with 4-bit tokens both sides stay packed
// (kind::mxf4, twice the rate, 256 columns a stage). In a pair each CTA holds 128 rows of either
// operand, so that an SM's shared memory feeds 256 x 256 results from 32 KB a stage: a single
// CTA's 128 x 256 tile would need 48 KB, and both its reads and TMA's writes would pass what
// shared memory delivers.
//
//   warp 0   loads: codes, scale tiles; every load of either CTA completes on the even CTA's
//            barrier
//   warp 1   (even CTA) copies scale tiles to TMEM and issues the MMAs
//   warps 4-11  results: two accumulators alternate, so that a tile's results leave while the
//            next is computed. TMEM's 512 columns hold two of 256 and 128 of scales by letting
//            the two overlap by 128 columns, which are read first; then the next tile may begin.
//
// Results go through shared memory, a slab of 32 tokens x 128 bytes at a time, which TMA stores, or,
// where y's alignment forbids that, a warp row by row. The residual comes into the slab by the same
// ways, the first two slabs of a tile while its products still run. In SwiGLU the
// even CTA holds gate rows and the odd CTA the up rows that go with them; a thread owns a token's
// 32 columns, which is a block of the MX result.
//
// Measured back to back, where the power limit lowers the clock: 4096 x 16384 x 2048 with 8-bit tokens
// and SwiGLU 118 us (102 to 107 us on another B200), 2.3 PFLOP/s; 8192 x 16384 x 2048 with 4-bit
// tokens to fp16 141 us, 3.9 PFLOP/s. Of a tile's clocks with 8-bit tokens the tensor cores need 8,192;
// 2,300 go where the next tile waits for the shared columns.
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>
#include <type_traits>

#include "mx_gemm.cuh"

namespace opure {
namespace {

constexpr uint32_t kTile = 256;    // tokens and weight rows per tile
constexpr uint32_t kHalf = 128;    // of each, per CTA
constexpr uint32_t kThreads = 384;
constexpr uint32_t kEpiWarp = 4, kEpiWarps = 8;
constexpr uint32_t kOperand = kHalf * 128;  // bytes of a CTA's part of one operand of a stage
constexpr uint32_t kSlab = 4096;            // 32 rows of 128 bytes
constexpr uint32_t kTmemCols = 512, kAcc1 = 128, kScaleCol = 384;  // accumulator 0 starts at column 0

template <uint32_t XF, int EPI>
struct Shape {
    // Slabs per warp (two where residuals are fetched ahead), and the stages that leaves room for.
    static constexpr uint32_t kSlabs = EPI == OPURE_EPI_ADD ? 2 : 1, kStages = EPI == OPURE_EPI_ADD ? 4 : 5;
    static constexpr uint32_t kBlocks = XF == OPURE_MX_FP8 ? 1 : 2;  // scale tiles (128 columns) per stage
    static constexpr uint32_t kScaleBytes = kBlocks * 3 * kMxTileBytes;
    static constexpr uint32_t kStageBytes = 2 * kOperand + kScaleBytes;
    static constexpr uint32_t kScaleCols = kBlocks * 12;
    // Each stage has TMEM columns of its own for its scales, so a copy never meets an MMA that
    // still reads them: that MMA's commit freed the stage.
    static_assert(kStages * kScaleCols <= kTmemCols - kScaleCol, "TMEM columns");
    // Bytes that arrive per CTA and stage; a copy that spreads codes counts what it reads.
    static constexpr uint32_t kTx = kOperand + (XF == OPURE_MX_FP8 ? kOperand / 2 : kOperand) + kScaleBytes;
    static constexpr size_t kSmem = 1024 + size_t(kStages) * kStageBytes + kEpiWarps * kSlabs * kSlab;
    static_assert(kSmem <= 226 * 1024, "shared memory");
};

struct PairParams {
    uint32_t n, rows, half, kblocks, mtiles, ntiles;
    void *y;
    size_t y_stride;
    const void *residual;
    uint8_t *out, *outs;
    bool tma;        // rows of y and residual are whole, aligned 16-byte pieces
    uint32_t grain;  // without tma: bytes that a lane moves at once, 8, 4 or (0) a value
    DeviceStatus *st;
};

// 32 values of a thread -> 32 codes in global memory (dst 16-byte aligned); returns the scale byte.
template <uint32_t FMT>
__device__ __forceinline__ uint32_t quantize_block(float (&v)[32], uint8_t *dst, bool in) {
    float m = max_abs3(v[0], v[1], 0.f);
#pragma unroll
    for (int j = 2; j < 32; j += 2) m = max_abs3(m, v[j], v[j + 1]);
    const uint32_t byte = mx_scale_byte<FMT>(__float_as_uint(m) & 0x7fffffffu);
    const float inv = mx_inverse(byte);
    const uint32_t keep = byte == 255u ? 0u : ~0u;
#pragma unroll
    for (int j = 0; j < 32; ++j) v[j] *= inv;
    constexpr int kWords = FMT == OPURE_MX_FP4 ? 4 : 8;
    uint32_t c[kWords];
#pragma unroll
    for (int j = 0; j < kWords; ++j) {
        if constexpr (FMT == OPURE_MX_FP4) {
            float f[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) f[q] = v[8 * j + q];
            c[j] = mx_pack_fp4(f) & keep;
        } else {
            c[j] = mx_pack_fp8(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]) & keep;
        }
    }
    if (in)
#pragma unroll
        for (int j = 0; j < kWords; j += 4) reinterpret_cast<uint4 *>(dst)[j / 4] = make_uint4(c[j], c[j + 1], c[j + 2], c[j + 3]);
    return byte;
}

// The results' warps stop together when one of their lanes gives up.
__device__ __forceinline__ bool warp_wait(uint64_t *bar, uint32_t phase) {
    return __all_sync(0xffffffffu, mbar_wait(bar, phase));
}

template <uint32_t XF, int EPI, typename T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    mx_gemm_pair_kernel(const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap,
                        const __grid_constant__ CUtensorMap wsmap, const __grid_constant__ CUtensorMap xsmap,
                        const __grid_constant__ CUtensorMap ymap, const __grid_constant__ CUtensorMap rmap, PairParams p) {
    using S = Shape<XF, EPI>;
    constexpr uint32_t kStages = S::kStages;
    constexpr bool kSwiglu = EPI == OPURE_EPI_SWIGLU;
    constexpr uint32_t kResult = kSwiglu ? kHalf : kTile;  // result columns per tile
    extern __shared__ uint8_t dsm[];
    __shared__ __align__(8) uint64_t full[kStages], empty[kStages], acc_full[2], drained, fetched[kEpiWarps][2];
    __shared__ uint32_t tmem_base;
    __shared__ volatile int fail;

    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    const uint32_t rank = tc::cluster_rank();
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(dsm) + 1023) & ~uintptr_t(1023));
    auto a_tile = [&](uint32_t s) { return base + s * 2 * kOperand; };
    auto b_tile = [&](uint32_t s) { return base + s * 2 * kOperand + kOperand; };
    uint8_t *slabs = base + kStages * 2 * kOperand;
    auto sf_tile = [&](uint32_t s) { return slabs + kEpiWarps * S::kSlabs * kSlab + s * S::kScaleBytes; };

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < kStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        mbar_init(&acc_full[0], 1);
        mbar_init(&acc_full[1], 1);
        mbar_init(&drained, 2 * kEpiWarps);
        for (uint32_t w = 0; w < kEpiWarps; ++w) {
            mbar_init(&fetched[w][0], 1);
            mbar_init(&fetched[w][1], 1);
        }
        fail = 0;
        tc::prefetch_map(&wmap);
        tc::prefetch_map(&xmap);
        tc::prefetch_map(&wsmap);
        tc::prefetch_map(&xsmap);
    }
    if (warp == 2) tc::alloc_pair(&tmem_base, kTmemCols);
    tc::fence_before();
    tc::cluster_sync();
    tc::fence_after();
    const uint32_t tmem = tmem_base;
    grid_dependency_wait();
    grid_dependents_launch();

    const uint32_t tiles = p.mtiles * p.ntiles, pairs = gridDim.x / 2, first = blockIdx.x / 2;
    const uint32_t stages = (p.kblocks + S::kBlocks - 1) / S::kBlocks;  // per tile
    uint32_t issued = 0;

    if (warp == 0) {
        const bool one = tc::elect();
        const uint32_t full0 = tc::map_rank(smem_addr(&full[0]), 0);
        uint32_t s = 0, phase = 1;  // the first round finds every stage free
        bool ok = true;
        for (uint32_t t = first; ok && t < tiles; t += pairs) {
            const uint32_t m0 = t % p.mtiles * kTile + rank * kHalf, r0 = t / p.mtiles * kResult;
            // This CTA's half of the weight rows, and the scale tiles of both halves.
            const uint32_t w_row = kSwiglu ? (rank ? p.half + r0 : r0) : r0 + rank * kHalf;
            for (uint32_t i = 0; i < stages; ++i, ++issued) {
                if (issued >= kStages && !mbar_wait(&empty[s], phase)) {
                    if (one) report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 84, blockIdx.x);
                    fail = 1;
                    ok = false;
                    break;
                }
                const uint32_t bar = full0 + s * 8, kb = i * S::kBlocks;
                tc::expect_tx(one && rank == 0, &full[s], 2 * S::kTx);
                tc::load_2d_pair(one, a_tile(s), &xmap, i * 128, m0, bar);
                tc::load_2d_pair(one, b_tile(s), &wmap, i * 128, w_row, bar);
                tc::load_4d_pair(one, sf_tile(s), &xsmap, 0, kb, m0 / 128, 0, bar);
                tc::load_4d_pair(one, sf_tile(s) + S::kBlocks * kMxTileBytes, &wsmap, 0, kb, r0 / 128, 0, bar);
                if (++s == kStages) {
                    s = 0;
                    phase ^= 1;
                }
            }
        }
    } else if (warp == 1 && rank == 0) {
        constexpr uint32_t idesc = XF == OPURE_MX_FP8 ? tc::idesc_mx(tc::kE4M3, tc::kE2M1, kTile, kTile)
                                                      : tc::idesc_mx(tc::kPackedE2M1, tc::kPackedE2M1, kTile, kTile);
        const bool one = tc::elect();
        const uint32_t tbase = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t da0 = tc::desc_sw128(smem_addr(a_tile(0))), ds0 = tc::desc_scales(smem_addr(sf_tile(0)));
        uint32_t s = 0, phase = 0, lt = 0;
        bool ok = true;
        for (uint32_t t = first; ok && t < tiles; t += pairs, ++lt) {
            const uint32_t acc = tbase + (lt & 1u) * kAcc1;
            // The tile before last has left this accumulator, and the last one the columns
            // that the two share.
            if (lt && !mbar_wait(&drained, (lt - 1) & 1u)) {
                if (one) report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 85, blockIdx.x);
                fail = 1;
                break;
            }
            for (uint32_t i = 0; i < stages; ++i) {
                if (!mbar_wait(&full[s], phase)) {
                    if (one) report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 86, blockIdx.x);
                    fail = 1;
                    ok = false;
                    break;
                }
                tc::fence_after();
                const uint32_t sfa = tbase + kScaleCol + s * S::kScaleCols, sfb = sfa + S::kBlocks * 4;
                const uint64_t da = da0 + s * (2 * kOperand >> 4), db = da + (kOperand >> 4);
                const uint64_t ds = ds0 + s * (S::kScaleBytes >> 4);
                constexpr uint32_t kTile16 = kMxTileBytes >> 4;
                uint64_t *const release = &empty[s];
                if (++s == kStages) {
                    s = 0;
                    phase ^= 1;
                }
#pragma unroll
                for (uint32_t b = 0; b < S::kBlocks; ++b) {
                    tc::copy_scales_pair(one, sfa + b * 4, ds + b * kTile16);
                    tc::copy_scales_pair(one, sfb + b * 8, ds + (S::kBlocks + b) * kTile16);
                    tc::copy_scales_pair(one, sfb + b * 8 + 4, ds + (2 * S::kBlocks + b) * kTile16);
                }
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) {
                    const uint32_t more = (i | k) != 0;
                    if constexpr (XF == OPURE_MX_FP8)
                        tc::mma_mxf8f6f4_pair(one, acc, da + 2 * k, db + 2 * k, idesc | tc::idesc_block(k), sfa, sfb, more);
                    else
                        tc::mma_mxf4_pair(one && i * 2 + k / 2 < p.kblocks, acc, da + 2 * k, db + 2 * k,
                                          idesc | tc::idesc_block(k % 2 * 2), sfa + k / 2 * 4, sfb + k / 2 * 8, more);
                }
                tc::commit_pair(one, release);
                if (i + 1 == stages) tc::commit_pair(one, &acc_full[lt & 1u]);
            }
        }
    } else if (warp >= kEpiWarp) {
        const uint32_t quarter = warp & 3u, part = (warp - kEpiWarp) >> 2;  // TMEM lanes, 64 columns of either half
        const uint32_t drain_bar = tc::map_rank(smem_addr(&drained), 0);
        uint8_t *slab0 = slabs + (warp - kEpiWarp) * S::kSlabs * kSlab;
        uint32_t fetch_phase[2] = {0, 0};
        uint32_t lt = 0;
        for (uint32_t t = first; t < tiles; t += pairs, ++lt) {
            const uint32_t b = lt & 1u;
            const uint32_t row0 = t % p.mtiles * kTile + rank * kHalf + quarter * 32, row = row0 + lane;
            const uint32_t r0 = t / p.mtiles * kResult;
            const uint32_t acc = tmem + b * kAcc1 + ((quarter * 32) << 16);
            const uint32_t shared_side = b ? 0 : kHalf, other_side = kHalf - shared_side, c0 = part * 64;
            // Without SwiGLU: this warp's 128 columns in steps of a slab, the shared ones first.
            constexpr uint32_t kCols = kSwiglu ? 64 : 128 / sizeof(T), kSteps = 128 / kCols;
            auto step_col = [&](uint32_t step) {
                return (step < kSteps / 2 ? shared_side : other_side) + c0 + step % (kSteps / 2) * kCols;
            };
            auto slab_of = [&](uint32_t step) { return slab0 + step % S::kSlabs * kSlab; };
            auto inside = [&](uint32_t step) { return row0 < p.n && r0 + step_col(step) < p.rows; };
            // Without TMA: slab rows to and from memory, `grain` bytes a lane, so that one or two rows
            // go at a time. move(slab place, row's place in memory, whole grain, values of it inside).
            auto by_rows = [&](auto grain, uint32_t col, uint8_t *slab, auto move) {
                constexpr uint32_t G = decltype(grain)::value, kLanes = 128 / G, kValues = G / sizeof(T);
                const uint32_t l = lane % kLanes, at = l * G, rows = min(p.n - row0, 32u);
                const uint32_t left = columns_left(p.rows, col + l * kValues);
                size_t place = size_t(row0 + lane / kLanes) * p.y_stride + col + l * kValues;
#pragma unroll 8
                for (uint32_t r = lane / kLanes; r < rows; r += 32 / kLanes, place += 32 / kLanes * p.y_stride)
                    move(slab + r * 128 + (((at >> 4) ^ (r & 7u)) << 4) + (at & 15u), place, left >= kValues, left);
            };
            auto with_grain = [&](auto f) {
                if (p.grain == 8)
                    f(std::integral_constant<uint32_t, 8>(), true);
                else
                    f(std::integral_constant<uint32_t, 4>(), p.grain == 4);
            };
            auto fetch = [&](uint32_t step) {
                if constexpr (EPI == OPURE_EPI_ADD) {
                    if (!inside(step)) return;
                    const uint32_t col = r0 + step_col(step);
                    uint8_t *slab = slab_of(step);
                    __syncwarp();
                    if (p.tma) {
                        if (lane == 0) tc::store_wait_read();  // what was in the slab has left
                        uint64_t *bar = &fetched[warp - kEpiWarp][step % 2];
                        tc::expect_tx(lane == 0, bar, kSlab);
                        tc::load_2d(lane == 0, slab, &rmap, col, row0, bar);
                    } else {
                        with_grain([&](auto grain, bool whole) {
                            constexpr uint32_t G = decltype(grain)::value;
                            by_rows(grain, col, slab, [&](uint8_t *dst, size_t place, bool all, uint32_t left) {
                                const T *src = static_cast<const T *>(p.residual) + place;
                                if (whole && all)
                                    tc::copy_async<G>(dst, src);
                                else
#pragma unroll
                                    for (uint32_t k = 0; k < G / sizeof(T); ++k)
                                        if (k < left) reinterpret_cast<T *>(dst)[k] = src[k];
                            });
                        });
                    }
                }
            };
            if constexpr (!kSwiglu) {
                fetch(0);
                fetch(1);
            }
            if (!warp_wait(&acc_full[b], (lt >> 1) & 1u)) {
                if (lane == 0 && !fail) report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 87, blockIdx.x);
                fail = 1;
                break;
            }
            tc::fence_after();
            // Accumulator 0 shares its last 128 columns, accumulator 1 its first 128. Each warp has
            // 64 of them and 64 others; it reads the shared ones first and lets the next tile begin.
            auto release = [&] {
                tc::fence_before();
                __syncwarp();
                if (lane == 0) tc::arrive_cluster(drain_bar);
            };
            if constexpr (kSwiglu) {
                // Blocks 2 part and 2 part + 1 of the tile's four: gate columns 32 j, up 128 + 32 j.
                constexpr uint32_t kF = sizeof(T) == 1 ? OPURE_MX_FP8 : OPURE_MX_FP4;
                uint32_t pre[2][32], cur[32];
                tc::ld32(acc + shared_side + c0, pre[0]);
                tc::ld32(acc + shared_side + c0 + 32, pre[1]);
                tc::wait_ld();
                release();
                tc::ld32(acc + other_side + c0, cur);
                tc::wait_ld();
                uint32_t bytes = 0;
#pragma unroll
                for (uint32_t j = 0; j < 2; ++j) {
                    if (j) {
                        tc::ld32(acc + other_side + c0 + 32, cur);
                        tc::wait_ld();
                    }
                    const uint32_t col = r0 + c0 + 32 * j;
                    float v[32];
                    if (b) {
#pragma unroll
                        for (int q = 0; q < 32; ++q) v[q] = __uint_as_float(pre[j][q]);
#pragma unroll
                        for (int q = 0; q < 32; q += 2) swiglu2(v[q], v[q + 1], __uint_as_float(cur[q]), __uint_as_float(cur[q + 1]));
                    } else {
#pragma unroll
                        for (int q = 0; q < 32; ++q) v[q] = __uint_as_float(cur[q]);
#pragma unroll
                        for (int q = 0; q < 32; q += 2) swiglu2(v[q], v[q + 1], __uint_as_float(pre[j][q]), __uint_as_float(pre[j][q + 1]));
                    }
                    if (col + 32 > p.half) {
#pragma unroll
                        for (int q = 0; q < 32; ++q)
                            if (col + q >= p.half) v[q] = 0.f;  // gate rows past the half are up rows
                    }
                    const bool in = row < p.n && col < mx_kp(p.half);
                    bytes |= quantize_block<kF>(v, p.out + row * mx_row_bytes(kF, p.half) + size_t(col) * kF / 8, in) << (8 * j);
                }
                if (row < p.n && r0 + c0 < mx_kp(p.half))
                    *reinterpret_cast<uint16_t *>(p.outs + mx_scale_offset(p.half, row, (r0 + c0) / 32)) = uint16_t(bytes);
            } else {
#pragma unroll 1
                for (uint32_t h = 0; h < 2; ++h) {
                    uint32_t v[2][32];
                    const uint32_t c = (h ? other_side : shared_side) + c0;
                    tc::ld32(acc + c, v[0]);
                    tc::ld32(acc + c + 32, v[1]);
                    tc::wait_ld();
                    if (h == 0) release();
#pragma unroll
                    for (uint32_t q = 0; q < kSteps / 2; ++q) {
                        const uint32_t step = h * (kSteps / 2) + q, col = r0 + step_col(step);
                        uint8_t *slab = slab_of(step);
                        if (inside(step)) {
                            if constexpr (EPI == OPURE_EPI_ADD) {
                                if (p.tma) {
                                    if (!mbar_wait(&fetched[warp - kEpiWarp][step % 2], fetch_phase[step % 2]))
                                        report(p.st, OPURE_ERR_DEVICE_TIMEOUT, 88, blockIdx.x);
                                    fetch_phase[step % 2] ^= 1;
                                } else {
                                    tc::copy_async_wait();
                                }
                            } else if (p.tma && lane == 0) {
                                tc::store_wait_read();
                            }
                            __syncwarp();
#pragma unroll
                            for (uint32_t e = 0; e < 8; ++e) {  // 16 bytes each
                                uint4 *at = reinterpret_cast<uint4 *>(slab + lane * 128 + ((e ^ (lane & 7u)) << 4));
                                uint4 u = {};
                                if constexpr (EPI == OPURE_EPI_ADD) u = *at;
                                T *h8 = reinterpret_cast<T *>(&u);
#pragma unroll
                                for (uint32_t k = 0; k < 16 / sizeof(T); ++k) {
                                    const uint32_t i = q * kCols + e * (16 / sizeof(T)) + k;
                                    float f = __uint_as_float(v[i / 32][i % 32]);
                                    if constexpr (EPI == OPURE_EPI_ADD) f += to_f32(h8[k]);
                                    h8[k] = from_f32<T>(f);
                                }
                                *at = u;
                            }
                            if (p.tma) {
                                tc::fence_async_shared();
                                __syncwarp();
                                if (lane == 0) tc::store_2d(&ymap, col, row0, slab);
                            } else {
                                __syncwarp();
                                with_grain([&](auto grain, bool whole) {
                                    using Word = std::conditional_t<decltype(grain)::value == 8, uint2, uint32_t>;
                                    by_rows(grain, col, slab, [&](uint8_t *src, size_t place, bool all, uint32_t left) {
                                        const Word w = *reinterpret_cast<const Word *>(src);
                                        T *dst = static_cast<T *>(p.y) + place;
                                        if (whole && all)
                                            *reinterpret_cast<Word *>(dst) = w;
                                        else
#pragma unroll
                                            for (uint32_t k = 0; k < sizeof(Word) / sizeof(T); ++k)
                                                if (k < left) dst[k] = reinterpret_cast<const T *>(&w)[k];
                                    });
                                });
                                __syncwarp();
                            }
                        }
                        if (step + 2 < kSteps) fetch(step + 2);
                    }
                }
            }
        }
        if (!kSwiglu && p.tma && lane == 0) tc::store_wait();
        __syncwarp();
    }
    tc::fence_before();
    __syncthreads();
    // After a failure: leave no copy in flight into the pair's shared memory.
    if (fail && threadIdx.x == 0 && rank == 0)
        for (uint32_t i = issued > kStages ? issued - kStages : 0; i < issued; ++i) mbar_wait(&full[i % kStages], (i / kStages) & 1u);
    tc::cluster_sync();
    if (warp == 2) tc::dealloc_pair(tmem, kTmemCols);
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
    static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
    });
    return fn;
}

template <uint32_t XF, int EPI, typename T>
opure_status launch_pair(opure_ctx *ctx, const CUtensorMap (&m)[6], const PairParams &p) {
    auto *kernel = mx_gemm_pair_kernel<XF, EPI, T>;
    const cudaError_t e =
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(Shape<XF, EPI>::kSmem));
    if (e != cudaSuccess) return cuda_status(e);
    const uint32_t pairs = std::min(uint32_t(ctx->sm_count) / 2, p.mtiles * p.ntiles);
    return launch(ctx, kernel, dim3(2 * pairs), dim3(kThreads), Shape<XF, EPI>::kSmem, true, m[0], m[1], m[2], m[3], m[4], m[5], p);
}

}  // namespace

bool make_map(CUtensorMap *m, CUtensorMapDataType type, uint32_t rank, const void *p, const uint64_t *dims, const uint64_t *strides,
              const uint32_t *box, CUtensorMapSwizzle swizzle) {
    auto fn = encode_fn();
    if (!fn) return false;
    const cuuint32_t es[4] = {1, 1, 1, 1};
    static_assert(sizeof(cuuint64_t) == sizeof(uint64_t) && sizeof(cuuint32_t) == sizeof(uint32_t), "map dimensions");
    return fn(m, type, rank, const_cast<void *>(p), reinterpret_cast<const cuuint64_t *>(dims),
              reinterpret_cast<const cuuint64_t *>(strides), box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

uint64_t mx_gemm_pair_ns(const opure_ctx *ctx, const opure_mx_gemm_args *a) {
    const uint64_t ntiles = a->epilogue == OPURE_EPI_SWIGLU ? mx_kp(a->w.rows / 2) / kHalf : (uint64_t(a->w.rows) + kTile - 1) / kTile;
    const uint64_t tiles = (uint64_t(a->x.rows) + kTile - 1) / kTile * ntiles, pairs = uint64_t(ctx->sm_count) / 2;
    const uint64_t stages = ceil_div(mx_kp(a->w.cols), a->x.format == OPURE_MX_FP8 ? 128 : 256);
    return a->x.rows <= kHalf ? ~uint64_t(0) : 4300 + (tiles + pairs - 1) / pairs * (stages * 360 + 1000);
}

opure_status mx_gemm_pair(opure_ctx *ctx, const opure_mx_gemm_args *a, const uint8_t *w_scales) {
    const bool swiglu = a->epilogue == OPURE_EPI_SWIGLU, fp8 = a->x.format == OPURE_MX_FP8;
    PairParams p{};
    p.n = a->x.rows;
    p.rows = a->w.rows;
    p.half = a->w.rows / 2;
    p.kblocks = mx_kp(a->w.cols) / 128;
    p.mtiles = (p.n + kTile - 1) / kTile;
    p.ntiles = swiglu ? mx_kp(p.half) / kHalf : (p.rows + kTile - 1) / kTile;
    p.y = a->y;
    p.y_stride = a->y_stride;
    p.residual = a->residual;
    p.out = a->out.codes;
    p.outs = a->out.scales;
    p.st = ctx->status;
    // Maps: w, x, their scale tiles, y, residual.
    CUtensorMap m[6] = {};
    auto codes = [&](CUtensorMap *t, const opure_mx_matrix &q) {
        if (fp8) return make_slot_map(t, q, kHalf);
        const size_t bytes = mx_row_bytes(q.format, q.cols);
        return make_map(t, CU_TENSOR_MAP_DATA_TYPE_UINT8, q.codes, bytes, q.rows, bytes, 128, kHalf, CU_TENSOR_MAP_SWIZZLE_128B);
    };
    // Scale tiles as [sides][rows of tiles][tiles][128 words]: boxes of a stage's tiles of one row
    // of tiles (x), of two neighbouring ones (w), or of one in either half of w (SwiGLU).
    const uint32_t blocks = fp8 ? 1 : 2;
    auto scales = [&](CUtensorMap *t, const uint8_t *s, uint32_t rows, uint32_t sides, uint32_t box_rows) {
        const uint64_t row = uint64_t(p.kblocks) * kMxTileBytes, tile_rows = (uint64_t(rows) + 127) / 128;
        const uint64_t dims[4] = {128, p.kblocks, tile_rows, sides}, strides[3] = {kMxTileBytes, row, row * tile_rows};
        const uint32_t box[4] = {128, blocks, box_rows, sides};
        return make_map(t, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, s, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
    };
    if (!codes(&m[0], a->w) || !codes(&m[1], a->x) || !scales(&m[2], w_scales, swiglu ? p.half : p.rows, swiglu ? 2 : 1, swiglu ? 1 : 2) ||
        !scales(&m[3], a->x.scales, p.n, 1, 1))
        return OPURE_ERR_UNSUPPORTED;
    m[4] = m[5] = m[3];
    if (!swiglu) {
        const bool add = a->epilogue == OPURE_EPI_ADD;
        const uint32_t size = type_bytes(a->y_type);
        const CUtensorMapDataType type = a->y_type == OPURE_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                         : a->y_type == OPURE_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                  : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
        auto rows = [&](CUtensorMap *t, const void *ptr) {
            // A store that ends inside 16 bytes wrote all of them: rows have to be whole pieces.
            return rows_aligned16(ptr, a->y_type, a->y_stride) && size_t(p.rows) * size % 16 == 0 &&
                   make_map(t, type, ptr, p.rows, p.n, a->y_stride * size, 128 / size, 32, CU_TENSOR_MAP_SWIZZLE_128B);
        };
        p.tma = rows(&m[4], a->y) && (!add || rows(&m[5], a->residual));
        for (uint32_t grain : {8u, 4u})
            if (!p.grain && (a->y_stride * size | reinterpret_cast<uintptr_t>(a->y) | (add ? reinterpret_cast<uintptr_t>(a->residual) : 0)) % grain == 0)
                p.grain = grain;
    }
    auto go = [&](auto t, auto epi) {
        using T = decltype(t);
        constexpr int kEpi = decltype(epi)::value;
        return fp8 ? launch_pair<OPURE_MX_FP8, kEpi, T>(ctx, m, p) : launch_pair<OPURE_MX_FP4, kEpi, T>(ctx, m, p);
    };
    if (swiglu) {
        const std::integral_constant<int, OPURE_EPI_SWIGLU> epi;
        return a->out.format == OPURE_MX_FP4 ? go(uint32_t(), epi) : go(uint8_t(), epi);
    }
    return with_type(a->y_type, [&](auto t) {
        return a->epilogue == OPURE_EPI_ADD ? go(t, std::integral_constant<int, OPURE_EPI_ADD>())
                                            : go(t, std::integral_constant<int, OPURE_EPI_STORE>());
    });
}

}  // namespace opure
