// Float32 products on the tensor cores whose results go through an operator of their own before they are stored, or are
// not stored at all: the kernel, its operand planes, and the plain store.
//
// A value is a pair of float16 terms under an exact power of two (half_split.cuh): hi = half(v s), lo = half((v s - hi) 2^11), s bringing
// the largest magnitude of its line to [2^14, 2^15).  Three MMAs of kind::f16 per 16 values of k: lo.hi and hi.lo into an accumulator of
// cross products (weight 2^-11), hi.hi into the leading one.  Here a pair holds what it can of every value - to 2^-23 of itself down to 2^-27 of
// its line's largest, below that to 2^-50 of the largest - and nothing is listed apart, so that a line's bits depend on that line
// alone: |error| <= 2^-21 sum |a||b| (2^-23 of each value, 2^-22 the lo.lo left out) + 2^-48 max|a| max|b| k, and the additions'.  Scales take
// any exponent.
//
// The tensor core truncates at every addition, always towards zero, which shows in sums of one sign as a bias: the leading
// accumulator is drained into registers every 128 values of k (8 additions) and summed there with rounding.  The drain has the
// next stage's cross products to hide behind, and every 256 values 8192 x 2048 x 11008 takes as long; with 1024 it was 2.5e-6 off (2-norm against
// 64 bits).

// Planes are row-major [rows][ld] float16, ld a multiple of eight.  An operand's rows may be its outer index (K-major) or its k
// (MN-major): the same planes of d serve d . w^T and x^T . d, and the weights [k][n] are never transposed.  MN-major stages hold 64
// columns of 64 values of k in 8 KB, the next 64 columns behind them.
//
// Structure as gemm_half.cu: pairs of CTAs (cta_group::2) with tiles of 256 x 256, or single CTAs with 128 x 128 and two sets of
// accumulators; TMA warp, issuing warp, sixteen epilogue warps; a lane has a row and its registers a quarter of the tile's columns.  What
// an epilogue does has the next tile's first 256 values of k to hide behind, some 8000 clocks.  All waits are bounded.
#pragma once

#include "common.cuh"
#include "tc_ptx.cuh"
#include "tmap.cuh"

#include <cuda_fp16.h>

#include <algorithm>

namespace ct {
namespace fused {

using namespace ptx;

constexpr float kLoScale = 2048.0f, kLoInv = 1.0f / 2048.0f;

// From the largest finite magnitude of a line: the factor that brings it to [2^14, 2^15), and its inverse; both normal numbers.
__host__ __device__ __forceinline__ int line_exponent(uint32_t max_bits) {
    const int e = (int)(max_bits >> 23) - 127;
    return e < -100 ? -100 : e; // a line of zeros: its factor widens no other line's range
}
#ifdef __CUDACC__
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ float line_scale(uint32_t max_bits) { return pow2(14 - line_exponent(max_bits)); }
__device__ __forceinline__ float line_inverse(uint32_t max_bits) { return pow2(line_exponent(max_bits) - 14); }
__device__ __forceinline__ uint32_t finite_bits(float v) {
    const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
    return u < 0x7f800000u ? u : 0u;
}
// Scaled values to their terms; an infinity or NaN is hi's alone.
__device__ __forceinline__ void split2(float a, float b, __half2 &hi, __half2 &lo) {
    hi = __floats2half2_rn(a, b);
    const float da = __fmul_rn(__fsub_rn(a, __low2float(hi)), kLoScale), db = __fmul_rn(__fsub_rn(b, __high2float(hi)), kLoScale);
    lo = __floats2half2_rn(fabsf(a) < INFINITY ? da : 0.0f, fabsf(b) < INFINITY ? db : 0.0f);
}
// The weight of an accumulated value: the product of two inverse scales, kept finite (2^127) so that a sum of zero stays zero; NaN stays.
__device__ __forceinline__ float weight(float row, float col) {
    float w;
    asm("min.NaN.f32 %0, %1, 0f7F000000;" : "=f"(w) : "f"(__fmul_rn(row, col)));
    return w;
}
#endif

// Sizes that tile coordinates of 32 bits hold, two matrices side by side and what is rounded up included.
constexpr int64_t kMostSize = 1 << 29;

// Planes of a matrix [rows][cols], and where one factor per row or column stands (the caller knows which).
struct Planes {
    __half *hi = nullptr, *lo = nullptr;
    int64_t rows = 0, cols = 0, ld = 0;
};
inline int64_t padded(int64_t cols) { return (cols + 7) / 8 * 8; }

struct Maps {
    CUtensorMap a_hi, a_lo, b_hi, b_lo;
};

struct Product {
    int64_t m, n;     // of the result
    int stages;       // of 64 values of k
    int stages_split; // > 0: k is cut in slices of that many stages, slice z stores its own result
    int tiles_m, tiles_n, group_m, total;
    int chunk_first; // stages until a tile's first drain
    int twin_offset; // twin epilogues: column of the planes of B where the second matrix begins
    const float *row_scale, *col_scale; // null: the columns' are one
    uint32_t *flags;
};

constexpr int kRows     = 128; // accumulator rows of a CTA
constexpr int kEpiWarps = 16;
constexpr int kThreads  = 64 + 32 * kEpiWarps;
constexpr int kTile     = 128 * 128;  // bytes of one plane of one operand in a stage
constexpr int kStage    = 4 * kTile;
constexpr int kStages   = 3;
// Stages per drain of the leading accumulator: two, and four in the first of a tile that has another tile's epilogue to wait for.
constexpr int kChunk = 2, kChunkFirst = 4;
constexpr int kSmem     = kStages * kStage + kEpiWarps * 2048 + 1024;

#ifdef __CUDACC__

// 128-byte swizzle; leading byte offset: the next 64 columns; stride byte offset: the next 8 values of k.
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr) {
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | (uint64_t)(8192 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ uint64_t desc(bool mn, uint32_t addr) { return mn ? desc_mn(addr) : smem_desc_k<128>(addr); }

__device__ __forceinline__ void tile_of(const Product &p, int tile, int &tm, int &tn, int &tz) {
    // groups of row tiles sweep the column tiles, so that CTAs running together share operands in L2
    const int per   = p.tiles_m * p.tiles_n;
    tz              = tile / per;
    const int bid   = tile - tz * per;
    const int g     = bid / (p.group_m * p.tiles_n);
    const int first = g * p.group_m;
    const int gm    = p.tiles_m - first < p.group_m ? p.tiles_m - first : p.group_m;
    const int in    = bid - g * p.group_m * p.tiles_n;
    tm              = first + in % gm;
    tn              = in / gm;
}

// EPI: kTwin - the tile's columns are half of one matrix and half of another, and a thread has the same columns of both;
// Params; store(p, e, acc, row0, lane, col0, z, part, stage): acc holds unscaled sums of row row0 + lane, columns col0 .. (twin: COLS / 2
// columns from col0 of the first matrix, then those of the second), the part-th quarter of the tile's; stage is the warp's 2 KB.
// Tiles is which tiles of which products this CTA has: start, is there one, the next (the i-th).  kTwo: of two products the first (A_MN, B_MN
// false) is K-major and the second MN-major.
struct TilesOfOne {
    static constexpr bool kTwo = false;
    int first, stride;
    __device__ __forceinline__ void start(int &job, int &tile) const { job = 0, tile = first; }
    __device__ __forceinline__ bool has(const Product &p, int, int tile) const { return tile < p.total; }
    __device__ __forceinline__ void next(int, int &, int &tile) const { tile += stride; }
};
// A tile of the product whose tiles take longer to each of the first CTAs; the others begin with `turns` tiles of the other one each, and then all
// share what is left of it, those others first.
struct TilesOfTwo {
    static constexpr bool kTwo = true;
    int block, blocks, longer, long_total, other_total, turns;
    __device__ __forceinline__ void start(int &job, int &tile) const {
        job  = block < long_total ? longer : 1 - longer;
        tile = block < long_total ? block : block - long_total;
    }
    __device__ __forceinline__ bool has(const Product &, int job, int tile) const { return job == longer || tile < other_total; }
    __device__ __forceinline__ void next(int i, int &job, int &tile) const {
        const int spare = blocks - long_total;
        job = 1 - longer;
        if (block < long_total)
            tile = turns * spare + (i - 1) * blocks + block + spare;
        else
            tile = i < turns ? i * spare + block - long_total : turns * spare + (i - turns) * blocks + block - long_total;
    }
};
template <class EPI, int BN, int CG, bool A_MN, bool B_MN, class Tiles>
__device__ __forceinline__ void product_body(
    const Maps &maps0, const Product &p0, const typename EPI::Params &e0, const Maps &maps1, const Product &p1, const typename EPI::Params &e1, const Tiles &tiles) {
    static_assert(BN / CG == 128, "128 columns of B to a CTA");
    static_assert(!Tiles::kTwo || (CG == 1 && !A_MN && !B_MN), "two products");
    constexpr int SETS = 512 / (2 * BN), COLS = BN / 4;
    const int rank = CG == 2 ? (int)cluster_rank() : 0;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bar_full[kStages], bar_empty[kStages];
    __shared__ uint64_t bar_acc_full[2 * SETS], bar_acc_empty[2 * SETS]; // [set * 2 + which]: 0 leading accumulator, 1 cross products
    __shared__ uint64_t bar_done;
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag_s;
    volatile int *abort_flag = &abort_flag_s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0)
        abort_flag_s = *reinterpret_cast<volatile uint32_t *>(p0.flags + FLAG_TIMEOUT) != 0 ? 1 : 0;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(smem_u32(&bar_full[s]), 1);
            mbar_init(smem_u32(&bar_empty[s]), 1);
        }
        for (int b = 0; b < 2 * SETS; ++b) {
            mbar_init(smem_u32(&bar_acc_full[b]), 1);
            mbar_init(smem_u32(&bar_acc_empty[b]), kEpiWarps * CG);
        }
        mbar_init(smem_u32(&bar_done), 1);
        mbar_fence_init();
        prefetch_tensormap(&maps0.a_hi);
        prefetch_tensormap(&maps0.a_lo);
        prefetch_tensormap(&maps0.b_hi);
        prefetch_tensormap(&maps0.b_lo);
    }
    if (warp == 1) {
        if (CG == 2) {
            tmem_alloc_pair(smem_u32(&tmem_base_slot), 512);
            tmem_relinquish_pair();
        } else {
            tmem_alloc(smem_u32(&tmem_base_slot), 512);
            tmem_relinquish();
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (CG == 2)
        cluster_sync(); // the partner's barriers exist before anything is signalled on them
    tc_fence_after_sync();
    const uint32_t tmem_base = tmem_base_slot;
    const bool failed        = abort_flag_s != 0; // an earlier launch failed: no work
    __syncthreads(); // every thread has read abort_flag_s before a role may raise it
    griddep_wait();
    griddep_launch_dependents();
    auto stage_addr = [&](int s) { return smem_base + (uint32_t)s * kStage; };
    auto k_range    = [&](const Product &p, int tz, int &from, int &count) {
        from           = p.stages_split > 0 ? tz * p.stages_split : 0;
        const int left = p.stages > from ? p.stages - from : 0;
        count          = p.stages_split > 0 && left > p.stages_split ? p.stages_split : left;
    };

    if (failed) {
    } else if (warp == 0) {
        // ===== TMA producer: stages numbered across tiles =====
        if (elect_one()) {
            int s = 0, issued = 0;
            uint32_t phase = 1;
            bool ok        = true;
            int job, tile, i = 0;
            for (tiles.start(job, tile); tiles.has(p0, job, tile) && ok; tiles.next(++i, job, tile)) {
                const bool two   = Tiles::kTwo && job == 1, a_mn = A_MN || two, b_mn = B_MN || two;
                const Product &p = two ? p1 : p0;
                const Maps &maps = two ? maps1 : maps0;
                int tm, tn, tz, from, count;
                tile_of(p, tile, tm, tn, tz);
                k_range(p, tz, from, count);
                const int32_t a_row = (tm * CG + rank) * kRows;
                // the two blocks of 64 columns of B; a K-major operand's are one box
                const int32_t b_first  = !EPI::kTwin ? tn * BN + rank * 128 : (CG == 2 ? rank * p.twin_offset + tn * 128 : tn * 64);
                const int32_t b_second = !EPI::kTwin || CG == 2 ? b_first + 64 : p.twin_offset + tn * 64;
                for (int kb = 0; kb < count; ++kb, ++issued) {
                    if (!mbar_wait(smem_u32(&bar_empty[s]), phase, abort_flag)) {
                        ok = false;
                        break;
                    }
                    uint32_t full = smem_u32(&bar_full[s]);
                    if (rank == 0) // both CTAs' bytes are counted on the leader's barrier
                        mbar_expect_tx(full, (uint32_t)(CG * kStage));
                    if (CG == 2)
                        full = leader_addr(full);
                    auto load = [&](uint32_t dst, const CUtensorMap *map, int32_t x, int32_t y) {
                        if (CG == 2)
                            tma_load_2d_pair(dst, map, full, x, y);
                        else
                            tma_load_2d(dst, map, full, x, y);
                    };
                    const uint32_t dst = stage_addr(s);
                    const int32_t k0   = (from + kb) * 64;
                    auto load_a = [&](uint32_t to, const CUtensorMap *map) {
                        if (a_mn) {
                            load(to, map, a_row, k0);
                            load(to + 8192, map, a_row + 64, k0);
                        } else {
                            load(to, map, k0, a_row);
                        }
                    };
                    auto load_b = [&](uint32_t to, const CUtensorMap *map) {
                        if (b_mn) {
                            load(to, map, b_first, k0);
                            load(to + 8192, map, b_second, k0);
                        } else {
                            load(to, map, k0, b_first);
                        }
                    };
                    load_a(dst + kTile, &maps.a_lo);
                    load_b(dst + 2 * kTile, &maps.b_hi);
                    load_a(dst, &maps.a_hi);
                    load_b(dst + 3 * kTile, &maps.b_lo);
                    if (++s == kStages)
                        s = 0, phase ^= 1u;
                }
            }
            if (*abort_flag && rank == 0) {
                // unwind: let the copies still in flight land before the CTA goes away (the leader's barriers
                // count the partner's copies too, and neither CTA leaves before the other)
                for (int k2 = issued - kStages < 0 ? 0 : issued - kStages; k2 < issued; ++k2) {
                    const uint64_t t0 = globaltimer_ns();
                    while (!mbar_try_wait(smem_u32(&bar_full[k2 % kStages]), (uint32_t)(k2 / kStages) & 1u) && globaltimer_ns() - t0 < kWaitBudgetNs) {
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ===== MMA issuer (the leader's, for the pair) =====
        if (elect_one() && rank == 0) {
            constexpr uint32_t kIdesc = make_idesc(0u, kRows * CG, BN);
            int s = 0;
            uint32_t phase = 0, empty_phase = (1u << (2 * SETS)) - 1u; // bit per accumulator: parity to wait for
            bool ok  = true;
            auto mma = [&](uint32_t idesc, uint32_t d, uint64_t da, uint64_t db, uint32_t accumulate) {
                if (CG == 2)
                    mma_f16_pair(d, da, db, idesc, accumulate);
                else
                    mma_f16(d, da, db, idesc, accumulate);
            };
            auto commit = [&](uint32_t bar) {
                if (CG == 2)
                    tc_commit_pair(bar);
                else
                    tc_commit(bar);
            };
            auto wait_empty = [&](int acc) {
                const bool got = mbar_wait<CG == 2 ? kClusterRead : kCta>(smem_u32(&bar_acc_empty[acc]), (empty_phase >> acc) & 1u, abort_flag);
                empty_phase ^= 1u << acc;
                tc_fence_after_sync();
                return got;
            };
            int job, tile, i = 0;
            for (tiles.start(job, tile); tiles.has(p0, job, tile) && ok; tiles.next(++i, job, tile)) {
                const bool two = Tiles::kTwo && job == 1, a_mn = A_MN || two, b_mn = B_MN || two;
                const Product &p     = two ? p1 : p0;
                const uint32_t idesc = kIdesc | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u);
                const int a_step = a_mn ? 128 : 2, b_step = b_mn ? 128 : 2; // descriptor units of 16 bytes per 16 values of k
                int tm, tn, tz, from, count;
                tile_of(p, tile, tm, tn, tz);
                k_range(p, tz, from, count);
                const int set         = SETS == 1 ? 0 : (i & (SETS - 1));
                const uint32_t d_main = tmem_base + (uint32_t)(set * 2 * BN), d_cross = d_main + BN;
                int in_chunk = 0, chunk = p.chunk_first;
                for (int kb = 0; kb < count; ++kb) {
                    if (!mbar_wait(smem_u32(&bar_full[s]), phase, abort_flag)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after_sync();
                    const uint32_t at    = stage_addr(s);
                    const uint64_t a_hi = desc(a_mn, at), a_lo = desc(a_mn, at + kTile);
                    const uint64_t b_hi = desc(b_mn, at + 2 * kTile), b_lo = desc(b_mn, at + 3 * kTile);
                    const bool last = kb + 1 == count;
                    if (kb == 0 && !wait_empty(set * 2 + 1)) {
                        ok = false;
                        break;
                    }
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk) {
                        mma(idesc, d_cross, a_lo + a_step * kk, b_hi + b_step * kk, kb == 0 && kk == 0 ? 0u : 1u);
                        mma(idesc, d_cross, a_hi + a_step * kk, b_lo + b_step * kk, 1u);
                    }
                    if (in_chunk == 0 && !wait_empty(set * 2)) {
                        ok = false;
                        break;
                    }
#pragma unroll
                    for (int kk = 0; kk < 4; ++kk)
                        mma(idesc, d_main, a_hi + a_step * kk, b_hi + b_step * kk, in_chunk == 0 && kk == 0 ? 0u : 1u);
                    commit(smem_u32(&bar_empty[s])); // stage reusable once these MMAs retire
                    if (++s == kStages)
                        s = 0, phase ^= 1u;
                    if (++in_chunk == chunk || last) {
                        commit(smem_u32(&bar_acc_full[set * 2]));
                        in_chunk = 0, chunk = kChunk;
                    }
                    if (last)
                        commit(smem_u32(&bar_acc_full[set * 2 + 1]));
                }
            }
            if (!ok || *abort_flag) {
                // unwind: wait until every MMA issued so far has retired
                commit(smem_u32(&bar_done));
                const uint64_t t0 = globaltimer_ns();
                while (!mbar_try_wait(smem_u32(&bar_done), 0) && globaltimer_ns() - t0 < kWaitBudgetNs) {
                }
            }
        }
    } else {
        // ===== epilogue =====
        const int quarter = warp & 3;       // TMEM lanes this warp may read: 32 * quarter ..
        const int part    = (warp - 2) >> 2; // which quarter of the tile's columns
        uint8_t *stage = smem_raw + (smem_base - smem_u32(smem_raw)) + kStages * kStage + (warp - 2) * 2048;
        uint32_t full_phase = 0;
        int job, tile, i = 0;
        for (tiles.start(job, tile); tiles.has(p0, job, tile); tiles.next(++i, job, tile)) {
            const bool two                 = Tiles::kTwo && job == 1;
            const Product &p               = two ? p1 : p0;
            const typename EPI::Params &e = two ? e1 : e0;
            int tm, tn, tz, from, count;
            tile_of(p, tile, tm, tn, tz);
            k_range(p, tz, from, count);
            const int set    = SETS == 1 ? 0 : (i & (SETS - 1));
            const int chunks = count == 0 ? 0 : count <= p.chunk_first ? 1 : 1 + (count - p.chunk_first + kChunk - 1) / kChunk;
            float acc[COLS];
            const uint32_t lane_base = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(set * 2 * BN);
            auto column = [&](int c) { // of the accumulator, of acc[c]
                return !EPI::kTwin ? part * COLS + c : (c < COLS / 2 ? part * (COLS / 2) + c : BN / 2 + part * (COLS / 2) + c - COLS / 2);
            };
            bool ok    = true;
            auto await = [&](int which) {
                const int a    = set * 2 + which;
                const bool got = mbar_wait(smem_u32(&bar_acc_full[a]), (full_phase >> a) & 1u, abort_flag);
                full_phase ^= 1u << a;
                ok = __all_sync(0xffffffffu, got);
                tc_fence_after_sync();
                return ok;
            };
            auto hand_back = [&](int which) {
                const uint32_t bar = smem_u32(&bar_acc_empty[set * 2 + which]);
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    if (CG == 2)
                        mbar_arrive_peer_read(leader_addr(bar));
                    else
                        mbar_arrive(bar);
                }
            };
            // the leading accumulator of every chunk but the last, then the cross products (the next tile starts with those), then
            // the last chunk
            const int events = count == 0 ? 0 : chunks + 1;
#pragma unroll
            for (int c = 0; c < COLS; ++c)
                acc[c] = 0.0f;
#pragma unroll 1
            for (int ev = 0; ev < events; ++ev) {
                const int which = ev == chunks - 1 ? 1 : 0;
                const float by  = which ? kLoInv : 1.0f;
                if (!await(which))
                    break;
#pragma unroll
                for (int g = 0; g < COLS / 16; ++g) {
                    uint32_t r[16];
                    tmem_ld_32x16(lane_base + (uint32_t)(which * BN + column(g * 16)), r);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        acc[g * 16 + j] = __fmaf_rn(__uint_as_float(r[j]), by, acc[g * 16 + j]);
                }
                hand_back(which);
            }
            if (!ok)
                break;
            const int64_t row0 = (int64_t)(tm * CG + rank) * kRows + quarter * 32;
            const int64_t col0 = EPI::kTwin ? (int64_t)tn * (BN / 2) + part * (COLS / 2) : (int64_t)tn * BN + part * COLS;
            EPI::template store<COLS>(p, e, acc, row0, lane, col0, tz, tn * 4 + part, stage);
        }
    }

    tc_fence_before_sync();
    __syncthreads();
    if (CG == 2)
        cluster_sync(); // neither CTA goes while the other's MMAs, copies or arrivals may still reach it
    if (warp == 1) {
        __syncwarp();
        tc_fence_after_sync();
        if (CG == 2)
            tmem_dealloc_pair(tmem_base, 512);
        else
            tmem_dealloc(tmem_base, 512);
    }
    if (threadIdx.x == 0 && !failed && *abort_flag)
        atomicExch(p0.flags + FLAG_TIMEOUT, 1u + (uint32_t)blockIdx.x);
}
template <class EPI, int BN, int CG, bool A_MN, bool B_MN>
__global__ void __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Product p, const __grid_constant__ typename EPI::Params e) {
    product_body<EPI, BN, CG, A_MN, B_MN>(maps, p, e, maps, p, e, TilesOfOne{(int)blockIdx.x / CG, (int)gridDim.x / CG});
}

// The inverse scales of columns col0 + 4 j .. + 3: one address for the warp.  Arrays of scales reach to the end of the last tile.
__device__ __forceinline__ float4 scales4(const float *scale, int64_t col) {
    return scale ? __ldg(reinterpret_cast<const float4 *>(scale + col)) : make_float4(1.0f, 1.0f, 1.0f, 1.0f);
}

// 32 rows x 16 columns of a warp, lane = row, to row-major memory through the warp's 2 KB: float4 slots XOR-swizzled by row, written
// as runs of 64 bytes per row.  value(j): column j of the lane's row.  dst: row 0, column 0 of the block; `cols` of them exist, from `skip` on.
__device__ __forceinline__ uint32_t stage_slot(int row, int slot) { return (uint32_t)(row * 64 + ((slot ^ (row >> 1 & 3)) << 4)); }
template <bool ADD, typename F>
__device__ __forceinline__ void store_block(
    float *dst, int64_t stride, int rows, int skip, int cols, bool vec, uint8_t *stage, int lane, F &&value) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
        *reinterpret_cast<float4 *>(stage + stage_slot(lane, j)) = make_float4(value(4 * j), value(4 * j + 1), value(4 * j + 2), value(4 * j + 3));
    __syncwarp();
    if (vec && cols == 16 && skip == 0) {
        const int sub = lane & 3, rr = lane >> 2;
        float *to = dst + rr * stride + sub * 4;
#pragma unroll
        for (int it = 0; it < 4; ++it, to += 8 * stride) {
            const int r = it * 8 + rr;
            float4 v    = *reinterpret_cast<const float4 *>(stage + stage_slot(r, sub));
            if (r < rows) {
                if (ADD) {
                    const float4 o = *reinterpret_cast<const float4 *>(to);
                    v = make_float4(__fadd_rn(o.x, v.x), __fadd_rn(o.y, v.y), __fadd_rn(o.z, v.z), __fadd_rn(o.w, v.w));
                }
                *reinterpret_cast<float4 *>(to) = v;
            }
        }
    } else {
        const int c = lane & 15; // a column per lane, two rows at a time
        float *to   = dst + (int64_t)(lane >> 4) * stride + c;
#pragma unroll 4
        for (int r = lane >> 4; r < rows; r += 2, to += 2 * stride) {
            const float v = *reinterpret_cast<const float *>(stage + stage_slot(r, c >> 2) + (c & 3) * 4);
            if (c >= skip && c < cols)
                *to = ADD ? __fadd_rn(*to, v) : v;
        }
    }
    __syncwarp(); // the block is rewritten
}

// The product itself.  Columns from `second` on belong to another matrix (both have n columns, row after row).
struct Store {
    static constexpr bool kTwin = false;
    struct Params {
        float *out, *out2; // out2: columns second .. second + n - 1
        int64_t n, second; // columns of out, and of out2
        int64_t stride;    // values between their rows
        int64_t slice;     // values between the results of two slices
        int add, vec;
    };
    template <int COLS>
    __device__ static __forceinline__ void store(
        const Product &p, const Params &e, float (&acc)[COLS], int64_t row0, int lane, int64_t col0, int z, int, uint8_t *stage) {
        const int64_t left = p.m - row0;
        const int rows     = left < 0 ? 0 : (left < 32 ? (int)left : 32);
        if (rows == 0)
            return;
        // kNoPart: a row of +0.  Other than scales, a row's weight may be infinite: its sums, of terms of both signs, are then NaN.
        float rs = lane < rows ? __fadd_rn(__ldg(p.row_scale + row0 + lane), 0.0f) : 0.0f;
        rs       = fabsf(rs) < INFINITY ? rs : NAN;
#pragma unroll
        for (int g = 0; g < COLS / 16; ++g) {
            const int64_t col = col0 + g * 16;
            if (col >= p.n)
                break;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 c = scales4(p.col_scale, col + 4 * j);
                float *a       = acc + g * 16 + 4 * j;
                a[0] = __fmul_rn(a[0], weight(rs, c.x)), a[1] = __fmul_rn(a[1], weight(rs, c.y));
                a[2] = __fmul_rn(a[2], weight(rs, c.z)), a[3] = __fmul_rn(a[3], weight(rs, c.w));
            }
            auto value = [&](int j) { return acc[g * 16 + j]; };
            // of the first matrix (or the only one), of the second, or of both where the block straddles its beginning
            const bool sec = e.out2 && col >= e.second;
            float *base    = (sec ? e.out2 : e.out) + (int64_t)z * e.slice + row0 * e.stride;
            const int64_t at = sec ? col - e.second : col, many = e.n - at;
            if (many > 0) {
                if (e.add)
                    store_block<true>(base + at, e.stride, rows, 0, many < 16 ? (int)many : 16, e.vec != 0, stage, lane, value);
                else
                    store_block<false>(base + at, e.stride, rows, 0, many < 16 ? (int)many : 16, e.vec != 0, stage, lane, value);
            }
            if (e.out2 && !sec && col + 16 > e.second) {
                const int skip = (int)(e.second - col);
                store_block<false>(e.out2 + (int64_t)z * e.slice + row0 * e.stride - skip, e.stride, rows, skip, e.n < 16 - skip ? (int)e.n + skip : 16,
                                   false, stage, lane, value);
            }
        }
    }
};

inline ct_status operand_map(CUtensorMap *map, const __half *base, const Planes &x, bool mn) {
    const uint64_t dims[2] = {(uint64_t)x.cols, (uint64_t)x.rows}, strides[1] = {(uint64_t)x.ld * 2};
    const uint32_t box[2]  = {64, mn ? 64u : 128u};
    return encode_tiled_map_f16(map, base, 2, dims, strides, box, 128);
}

// The product of prepared planes; a.rows (K-major) or a.cols (MN-major) is m, b's likewise n (twin: of one matrix); k the other index of
// both.  `splits` slices of k.
template <class EPI, int BN, int CG, bool A_MN, bool B_MN>
ct_status prepare(DeviceState *st, const Planes &a, const Planes &b, int splits, Maps &maps, Product &p, const char *name) {
    CT_TRY(operand_map(&maps.a_hi, a.hi, a, A_MN));
    CT_TRY(operand_map(&maps.a_lo, a.lo, a, A_MN));
    CT_TRY(operand_map(&maps.b_hi, b.hi, b, B_MN));
    CT_TRY(operand_map(&maps.b_lo, b.lo, b, B_MN));
    const int64_t k = A_MN ? a.rows : a.cols;
    p.stages        = (int)((k + 63) / 64);
    p.stages_split  = splits > 1 ? (p.stages + splits - 1) / splits : 0;
    constexpr int TN = EPI::kTwin ? BN / 2 : BN;
    p.tiles_m = (int)((p.m + kRows * CG - 1) / (kRows * CG));
    p.tiles_n = (int)((p.n + TN - 1) / TN);
    p.group_m = 16 / CG;
    p.flags   = st->flags_dev;
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n * splits;
    if (tiles > 0x3fffffff)
        return fail(CT_ERR_TOO_LARGE, "%s: too many tiles", name);
    p.total       = (int)tiles;
    p.chunk_first = tiles <= st->sm_count / CG ? kChunk : kChunkFirst;
    return CT_OK;
}
template <typename K> ct_status allow_shared(const DeviceState *st, K kernel, bool (&set_dev)[16]) { // the attribute belongs to a device's context
    if (!set_dev[st->device & 15]) {
        CT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
        set_dev[st->device & 15] = true;
    }
    return CT_OK;
}
template <class EPI, int BN, int CG, bool A_MN, bool B_MN>
ct_status launch(DeviceState *st, const Planes &a, const Planes &b, Product p, const typename EPI::Params &e, int splits, const char *name) {
    Maps maps;
    CT_TRY((prepare<EPI, BN, CG, A_MN, B_MN>(st, a, b, splits, maps, p, name)));
    auto kernel = product_kernel<EPI, BN, CG, A_MN, B_MN>;
    static bool set_dev[16] = {};
    CT_TRY(allow_shared(st, kernel, set_dev));
    const int units = st->sm_count / CG;
    CT_CUDA(launch_dependent_cluster(kernel, CG, dim3((unsigned)(std::min(p.total, units) * CG)), dim3(kThreads), (size_t)kSmem, stream(), maps, p, e));
    CT_LAUNCH_CHECK(name);
    return CT_OK;
}

// Pairs of CTAs with tiles of 256 x 256 (of both matrices, twin), or single ones with 128 x 128: pairs from where those are more than the machine
// has at a time and there are rows for both.  Single and pairs (us, k = 1024; cross entropy): 300 x 4736 (111 single tiles) 40 and 51, 512 x 4096 (128) 39 and 49, 768 x
// 3200 (150) 47 and 49, 512 x 8192 (256) 62 and 60, 1024 x 8192 84 and 81; gated 512 x 2048 (128) 37 and 47, 512 x 4096 58 and 58, 2048 x 5504 158 and 151;
// 128 x 32000, gradient, 215 and 232.
inline bool takes_pairs(const DeviceState *st, int64_t m, int64_t columns) { return m > 128 && (m + 127) / 128 * ((columns + 127) / 128) > st->sm_count; }

#endif // __CUDACC__

// ---- fused_product.cu ----------------------------------------------------------------------------

// Scale arrays hold `scales(n)` values: kernels read them to the end of a tile.
inline int64_t scales(int64_t n) { return (n + 255) / 256 * 256 + 256; }
// Parts of one piece of scratch, each on a 256-byte boundary.
struct Parts {
    size_t bytes = 0;
    size_t take(size_t size) {
        const size_t at = bytes;
        bytes += (size + 255) & ~(size_t)255;
        return at;
    }
    size_t planes(int64_t rows, int64_t ld) { return take((size_t)(rows * ld) * 4); }
};
inline Planes planes_at(const Scratch &s, size_t at, int64_t rows, int64_t cols, int64_t ld) {
    Planes p;
    p.hi = s.as<__half>(at), p.lo = p.hi + rows * ld, p.rows = rows, p.cols = cols, p.ld = ld;
    return p;
}
// Columns from .. from + cols - 1; from is a multiple of eight.
inline Planes columns_of(Planes p, int64_t from, int64_t cols) {
    p.hi += from, p.lo += from, p.cols = cols;
    return p;
}

// The factor of a row that takes no part, whatever it holds: -0.  Under a factor of 0 what is no number stays (0 x NaN is a term of a sum).
constexpr uint32_t kNoPart = 0x80000000u;

// What planes are made of, some matrices in one launch.
struct Split {
    const float *in, *in2; // in2 (may be null): a matrix of the same shape whose columns follow those of in at column padded(cols) of the planes
    int64_t rows, cols;
    bool by_column;        // a scale per column, else per row (over both matrices)
    const float *row_factor; // by_column, may be null: row r is taken times row_factor[r], and as zeros where that is kNoPart
    Planes to;
    float *inverse;        // [rows], or scales(columns of the planes)
    const float *col_factor = nullptr; // else, may be null: column c is taken times col_factor[c] (a multiple of four of them)
};
ct_status split(DeviceState *st, const Split *what, int count);

// out = a . b, [m][n] with rows `stride` apart; k sliced where there are few tiles, with partial sums in scratch of the call.  With out2 the
// columns from `second` on are a matrix of its own (both have `cols` columns).  add: to what out holds.
struct Result {
    float *out, *out2 = nullptr;
    int64_t cols, stride, second = 0;
    bool add = false;
};
// A product to be: a [m][k] and b [n][k] K-major, or both MN-major.
struct Wanted {
    Planes a, b;
    bool mn;
    int64_t m, n;
    const float *row_scale, *col_scale;
    Result to;
};
// One, or a K-major and an MN-major one.
ct_status products(DeviceState *st, const Wanted *what, int count);
// Slices of rows for sums over columns, a row to each of eight warps in turn: as many as six blocks to an SM, of 32 rows at least, and of 2048 at most
// (chains of 256) while a grid has that many.
inline int64_t row_slices(const DeviceState *st, int64_t rows, int64_t strips) {
    const int64_t fill = std::min<int64_t>((rows + 31) / 32, (int64_t)st->sm_count * 6 / strips), least = std::max<int64_t>(1, (rows + 2047) / 2048);
    return std::min<int64_t>(std::max(fill, least), 65535);
}
// out[c] = sum over the rows of row_weight[r] * planes[r][c].
ct_status column_sums(DeviceState *st, const Planes &x, const float *row_weight, float *out);
// first[c] = sum over parts of partial[part][c] for c < n, second[c] of partial[part][n + c] for n + c < width; either may be null.
ct_status join_columns(const double *partial, int64_t parts, int64_t n, int64_t width, float *first, float *second);

// Whether a product of m rows and that many columns (of both matrices) is few_rows': its passes have eight rows, the second of which reads
// the weights from L2 where they fit, while the streamed product has some 15 us of its own: 16 x 1024 x 2000 20 us against 29, x 8000 37
// against 29, x 32000 94 against 48; two matrices 16 x 1024 x 2048 18 against 25, x 4096 32 against 25.
inline bool takes_few_rows(int64_t m, int64_t columns) { return m <= 8 || (m <= 16 && columns < 6144); }
// out[m][n] = x . w + bias for at most kFewRows rows, or gate(x . w + bias) * (x . w_up + b_up) (w_up non-null), float32 on the CUDA cores.
constexpr int64_t kFewRows = 16;
ct_status few_rows(
    DeviceState *st, const float *x, const float *w, const float *bias, const float *w_up, const float *b_up, int64_t m, int64_t k, int64_t n, int gate,
    float *out, float *gate_pre, float *up_pre);

} // namespace fused
} // namespace ct
