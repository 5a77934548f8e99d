// Products of 17 to 128 rows (takes_stream): the weights are streamed through the tensor cores as they lie, float32, and read once for 64 rows.
//
// With so few rows a product is as long as it takes to read the weights, and writing their planes and reading them again is three times that
// (64 x 1024 x 32003: 76 us of pre-pass, 33 of product; here 63 in all).  So four warps fetch the weights, 64 values of k of 128 columns a stage
// (cp.async in the 16-byte pieces that they lie in), and two groups of eight, which take stages in turn, split them under a scale per
// column and stage, and write the planes to shared memory.  The weights' columns are the rows of the accumulator (128 lanes), the rows
// of x its columns (32 or 64; more rows go by 64, a launch each), so that a scale belongs to a lane and a stage: eight warps drain every
// stage and add it up in registers under its scale.  x comes as planes (K-major, a scale per row) by TMA.
// What bounds it: HBM would bring a stage's 32 KB in 1400 clocks, the MMAs take 12 x 54 of them (64 rows); splitting, scaling and draining
// keep the issue slots 62 % busy and a stage takes some 2000.  64 x 1024 x 128000 takes 147 us, 3.6 TB/s.
// A CTA has a range of columns, a multiple of 16, so that all CTAs have as much to read.
//
// Epilogue: the tile's sums go to shared memory as [row of x][column], 16 rows at a time; the draining warps do with them what EPI says.
#pragma once

#include "fastmath.cuh"
#include "fused_product.cuh"

#include <type_traits>

namespace ct {
namespace fused {

// Whether a product of more than 16 rows is streamed, `columns` those of both matrices: a CTA has an even share of them, of at least 16, and tiles of
// 128 are the emptier the fewer there are, while a pre-pass takes as long as there are weights; of more than 64 rows they are read twice.
// Streamed, and by tiles of planes (us; cross entropy over n classes, gated of two matrices of n; the first three lines without flushing L2):
//   17 rows, k = 128: gated x 300 8.7 and 10.2, x 2000 9.1 and 12.0; cross entropy x 1000 12.0 and 12.8; k = 1024: gated x 300 24 and 22, x 1000 25 and
//     25, x 2000 25 and 26; cross entropy x 1000 28 and 25, x 2000 29 and 26, x 4000 29 and 28; k = 4096: x 1000 82 and 67, x 4000 83 and 116
//   64 rows, k = 128: gated x 1000 11.7 and 11.0, x 2000 12.0 and 12.1; k = 1024: x 1000 28 and 26, x 2000 29 and 26, x 4000 29 and 33; k = 4096: x 1000
//     83 and 73, x 2000 83 and 116; cross entropy k = 1024: x 2000 33 and 26, x 4000 33 and 28; k = 4096: x 2000 88 and 73, x 4000 89 and 118
//   64 rows, k = 1024: cross entropy x 8192 41 and 45, x 32000 63 and 129; 128 rows: x 8192 68 and 47, x 16384 72 and 78, x 32000 111 and 130; gated
//     x 8192 68 and 62 (k = 2048 105 and 182), x 16384 115 and 111, x 32000 189 and 199
inline bool takes_stream(int64_t m, int64_t k, int64_t columns) {
    if (m <= 32)
        return k <= 384 || columns >= 2048; // k = 300: gated x 1000 13 and 14, cross entropy x 1000 17 and 15
    if (m <= 64)
        return columns >= (k < 2048 ? 4096 : 3000);
    return m <= 128 && columns >= 16384;
}
constexpr int kStreamSlots   = 2;
// Warps: of a stage fetched by the warps that convert it all did the same at the same time, and a stage of 64 x 1024 x 128000 took 3350 clocks.
constexpr int kStreamDrain = 8, kStreamFetch = 4, kStreamConvert = 8; // kStreamConvert: of a group
constexpr int kStreamThreads = (2 + kStreamDrain + kStreamFetch + 2 * kStreamConvert) * 32; // TMA, MMA
constexpr int kStreamPitch   = 129;
constexpr int kStreamSlot = 2 * kTile;     // the weights' planes
constexpr int kStreamX = 3;                 // stages of x, whose copies take a few of the weights' stages under load
constexpr int kStreamSets = 4;              // pairs of accumulators: a tile's epilogue does not stop the tensor core at once
constexpr int kStreamPass = 16;             // rows of x in an epilogue's pass
template <int NT> constexpr int kStreamXBytes = 2 * NT * 128;
// Weights as they lie: stages of 64 rows of two halves of 64 columns, a half 68 words (up to three from a row's 16-byte boundary).  Rows 2 apart,
// which a warp reads together, lie half of the banks apart.
constexpr int kStreamRaw = 3, kStreamHalf = 68, kStreamRow = 2 * kStreamHalf, kStreamRawBytes = 64 * kStreamRow * 4;
template <int NT> constexpr int kStreamSmem = kStreamSlots * kStreamSlot + kStreamX * kStreamXBytes<NT> + kStreamRaw * kStreamRawBytes + kStreamPass * kStreamPitch * 4 + 1024;

struct Stream {
    const float *w, *w2; // w2: twin epilogues, the second matrix (tiles of 64 columns of both)
    int64_t k, n, ld;    // ld: values between the weights' rows
    int m, per;          // rows of x; columns of a CTA
    int stages;
    int pieces;          // the matrices begin on 16-byte boundaries
    int whole;           // and so do their rows
    const float *row_scale;
    uint32_t *flags;
};
struct StreamMaps {
    CUtensorMap x_hi, x_lo;
};

// Sums are kept 2^14 lower, as those of x itself are: weights of 1e36 then overflow no earlier than the result.
constexpr float kStreamDown = 1.0f / 16384.0f, kStreamUp = 16384.0f;

#ifdef __CUDACC__

// A bounded wait that leaves the issue slots to others: the hardware suspends the thread until the phase completes.
__device__ __forceinline__ bool stream_wait(uint32_t bar, uint32_t parity, volatile int *abort_flag) { return mbar_wait_patient(bar, parity, abort_flag); }

// Where a role stands in a ring of N: the place, and the parity of its phase.
template <int N> struct Ring {
    int at = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next() {
        if (++at == N)
            at = 0, phase ^= 1u;
    }
};

// EPI: kTwin; Params; State (of a draining thread, across the CTA's tiles); tile<Q>(p, e, state, z, c0, cols, t): rows 16 Q .. of x,
// z[(row - 16 Q) * kStreamPitch + c] the sums over 2^14, but for the row's scale, of the tile's columns c0 + c < c0 + cols (twin: the second
// matrix's at 64 + c), t the thread of kStreamDrain * 32; finish(p, e, state, z, t), which all those threads call.
__device__ __forceinline__ void stream_epilogue_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kStreamDrain * 32) : "memory"); }
template <class EPI, int NT>
__global__ void __launch_bounds__(kStreamThreads, 1)
    stream_kernel(const __grid_constant__ StreamMaps maps, const __grid_constant__ Stream p, const __grid_constant__ typename EPI::Params e) {
    constexpr int TILE = EPI::kTwin ? 64 : 128, SLOT = kStreamSlot;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bar_raw[kStreamRaw], bar_raw_empty[kStreamRaw], bar_full[kStreamSlots], bar_empty[kStreamSlots], bar_x[kStreamX],
        bar_x_empty[kStreamX], bar_scale[8], bar_acc_full[kStreamSets], bar_acc_empty[kStreamSets], bar_done;
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag_s;
    __shared__ __align__(2) int8_t exponent_s[8][128]; // of a stage's columns' largest magnitudes; a converting warp is at most six stages ahead of the draining ones
    volatile int *abort_flag = &abort_flag_s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0)
        abort_flag_s = *reinterpret_cast<volatile uint32_t *>(p.flags + FLAG_TIMEOUT) != 0 ? 1 : 0;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem            = smem_raw + (smem_base - smem_u32(smem_raw));
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStreamSlots; ++s) {
            mbar_init(smem_u32(&bar_full[s]), kStreamConvert);
            mbar_init(smem_u32(&bar_empty[s]), 1);
        }
        for (int s = 0; s < kStreamRaw; ++s) {
            mbar_init(smem_u32(&bar_raw[s]), kStreamFetch * 32);
            mbar_init(smem_u32(&bar_raw_empty[s]), kStreamConvert);
        }
        for (int s = 0; s < kStreamX; ++s) {
            mbar_init(smem_u32(&bar_x[s]), 1);
            mbar_init(smem_u32(&bar_x_empty[s]), 1);
        }
        for (int s = 0; s < 8; ++s)
            mbar_init(smem_u32(&bar_scale[s]), kStreamConvert);
        for (int s = 0; s < kStreamSets; ++s) {
            mbar_init(smem_u32(&bar_acc_full[s]), 1);
            mbar_init(smem_u32(&bar_acc_empty[s]), kStreamDrain);
        }
        mbar_init(smem_u32(&bar_done), 1);
        mbar_fence_init();
        prefetch_tensormap(&maps.x_hi);
        prefetch_tensormap(&maps.x_lo);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(&tmem_base_slot), 512);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = tmem_base_slot;
    const bool failed        = abort_flag_s != 0;
    __syncthreads(); // every thread has read abort_flag_s before a role may raise it
    griddep_wait();
    griddep_launch_dependents();
    const int64_t begin = (int64_t)blockIdx.x * p.per, end = min(p.n, begin + p.per);
    const int tiles = (int)((end - begin + TILE - 1) / TILE), total = tiles * p.stages; // stages numbered across tiles

    if (failed) {
    } else if (warp == 0) {
        // ===== x =====
        if (elect_one()) {
            int issued = 0;
            Ring<kStreamX> ring;
            for (int s = 0, kb = 0; s < total; ++s, ring.next()) {
                if (!stream_wait(smem_u32(&bar_x_empty[ring.at]), ring.phase ^ 1u, abort_flag))
                    break;
                const uint32_t full = smem_u32(&bar_x[ring.at]), dst = smem_base + kStreamSlots * SLOT + ring.at * kStreamXBytes<NT>;
                mbar_expect_tx(full, kStreamXBytes<NT>);
                tma_load_2d(dst, &maps.x_hi, full, kb * 64, 0);
                tma_load_2d(dst + NT * 128, &maps.x_lo, full, kb * 64, 0);
                issued = s + 1;
                kb     = kb + 1 == p.stages ? 0 : kb + 1;
            }
            if (*abort_flag) { // unwind: let the copies still in flight land before the CTA goes away
                for (int s = issued - kStreamX < 0 ? 0 : issued - kStreamX; s < issued; ++s) {
                    const uint64_t t0 = globaltimer_ns();
                    while (!mbar_try_wait(smem_u32(&bar_x[s % kStreamX]), (uint32_t)(s / kStreamX) & 1u) && globaltimer_ns() - t0 < kWaitBudgetNs) {
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ===== MMA =====
        if (elect_one()) {
            constexpr uint32_t idesc = make_idesc(0u, 128, NT) | 1u << 15; // the weights are MN-major
            bool ok = true;
            Ring<kStreamSlots> planes;
            Ring<kStreamX> xs;
            Ring<kStreamSets> sets;
            for (int s = 0; s < total && ok; ++s, planes.next(), xs.next(), sets.next()) {
                const int slot = planes.at, set = sets.at, from = xs.at;
                ok = stream_wait(smem_u32(&bar_full[slot]), planes.phase, abort_flag) && stream_wait(smem_u32(&bar_x[from]), xs.phase, abort_flag) &&
                     stream_wait(smem_u32(&bar_acc_empty[set]), sets.phase ^ 1u, abort_flag);
                if (!ok)
                    break;
                tc_fence_after_sync();
                const uint32_t at    = smem_base + slot * SLOT;
                const uint64_t w_hi = desc_mn(at), w_lo = desc_mn(at + kTile);
                const uint32_t x_at = smem_base + kStreamSlots * SLOT + from * kStreamXBytes<NT>;
                const uint64_t x_hi = smem_desc_k<128>(x_at), x_lo = smem_desc_k<128>(x_at + NT * 128);
                const uint32_t d_main = tmem_base + set * 128, d_cross = d_main + 64;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    mma_f16(d_cross, w_lo + 128 * kk, x_hi + 2 * kk, idesc, kk > 0);
                    mma_f16(d_cross, w_hi + 128 * kk, x_lo + 2 * kk, idesc, 1u);
                    mma_f16(d_main, w_hi + 128 * kk, x_hi + 2 * kk, idesc, kk > 0);
                }
                tc_commit(smem_u32(&bar_empty[slot]));
                tc_commit(smem_u32(&bar_x_empty[from]));
                tc_commit(smem_u32(&bar_acc_full[set]));
            }
            if (!ok || *abort_flag) {
                tc_commit(smem_u32(&bar_done));
                const uint64_t t0 = globaltimer_ns();
                while (!mbar_try_wait(smem_u32(&bar_done), 0) && globaltimer_ns() - t0 < kWaitBudgetNs) {
                }
            }
        }
    } else if (warp < 2 + kStreamDrain) {
        // ===== draining =====
        // A thread's row is a column of the tile; it has half of the rows of x.
        constexpr int OWN = NT / 2;
        const int quarter = warp & 3, t = (warp - 2) * 32 + lane, row = quarter * 32 + lane, which = (warp - 2) >> 2;
        float *z = reinterpret_cast<float *>(smem + kStreamSlots * SLOT + kStreamX * kStreamXBytes<NT> + kStreamRaw * kStreamRawBytes);
        typename EPI::State state;
        EPI::init(state);
        bool ok = true;
        Ring<kStreamSets> sets;
        Ring<8> scales;
        for (int tile = 0; tile < tiles; ++tile) { // all warps take all tiles' barriers, also after a failed wait
            float acc[OWN];
#pragma unroll
            for (int j = 0; j < OWN; ++j)
                acc[j] = 0.0f;
#pragma unroll 1
            for (int kb = 0; kb < p.stages; ++kb, sets.next(), scales.next()) {
                const int set = sets.at;
                if (ok)
                    ok = __all_sync(0xffffffffu, stream_wait(smem_u32(&bar_acc_full[set]), sets.phase, abort_flag) &&
                                                     stream_wait(smem_u32(&bar_scale[scales.at]), scales.phase, abort_flag)) != 0;
                if (!ok)
                    continue;
                tc_fence_after_sync();
                const float by = __fmul_rn(pow2(exponent_s[scales.at][row]), kStreamDown * kStreamDown);
                const uint32_t at = tmem_base + ((uint32_t)(quarter * 32) << 16) + set * 128 + which * OWN;
#pragma unroll
                for (int g = 0; g < OWN / 8; ++g) {
                    uint32_t a[8], b[8];
                    tmem_ld_32x8(at + g * 8, a);
                    tmem_ld_32x8(at + 64 + g * 8, b);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 8; j += 2) {
                        const f32x2 m = pack2(__uint_as_float(a[j]), __uint_as_float(a[j + 1])), c = pack2(__uint_as_float(b[j]), __uint_as_float(b[j + 1]));
                        unpack2(fma2(fma2(c, dup2(0x3A000000u), m), pack2(by, by), pack2(acc[g * 8 + j], acc[g * 8 + j + 1])), acc[g * 8 + j], acc[g * 8 + j + 1]); // 2^-11
                    }
                }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(smem_u32(&bar_acc_empty[set]));
            }
            const int64_t c0 = begin + (int64_t)tile * TILE;
            auto pass        = [&](auto Q) {
                stream_epilogue_sync(); // the last sums have been read
                if (which == Q.value * kStreamPass / OWN)
#pragma unroll
                    for (int j = 0; j < kStreamPass; ++j)
                        z[j * kStreamPitch + row] = acc[Q.value * kStreamPass % OWN + j];
                stream_epilogue_sync();
                if (ok)
                    EPI::template tile<Q.value>(p, e, state, z, c0, (int)(end - c0 < TILE ? end - c0 : TILE), t);
            };
            pass(std::integral_constant<int, 0>{});
            pass(std::integral_constant<int, 1>{});
            if constexpr (NT == 64) {
                pass(std::integral_constant<int, 2>{});
                pass(std::integral_constant<int, 3>{});
            }
        }
        EPI::finish(p, e, state, z, t);
    } else if (warp < 2 + kStreamDrain + kStreamFetch) {
        // ===== fetching =====
        // What the matrix lacks is not fetched: columns past the CTA's are not looked at behind the product, values of k past the last are
        // zeroed when they are converted.
        // A thread's rows are four apart, so that all begin as far from a boundary, and its addresses a constant: worked out for every piece
        // (a mask, bounds) they took the four warps 2800 clocks a stage.
        static_assert(kStreamFetch == 4, "rows of a thread");
        const int who = warp - 2 - kStreamDrain, h = lane >> 4, q = 4 * (lane & 15);
        const int r17 = (who * 32 + lane) >> 1, h17 = lane & 1; // the row and half whose seventeenth piece this thread fetches
        const float *matrix = EPI::kTwin && h ? p.w2 : p.w, *matrix17 = EPI::kTwin && h17 ? p.w2 : p.w;
        const int64_t values = (p.k - 1) * p.ld + p.n, step = kStreamFetch * p.ld;
        bool ok = true;
        Ring<kStreamRaw> ring;
        for (int tile = 0; tile < tiles && ok; ++tile) {
            const int64_t col0 = begin + (int64_t)tile * TILE, col = col0 + (EPI::kTwin ? 0 : 64 * h);
            int64_t at         = (((int64_t)who * p.ld + col) & ~(int64_t)3) + q; // the thread's first piece in its matrix
            const int64_t own  = (int64_t)r17 * p.ld + col0 + (EPI::kTwin ? 0 : 64 * h17);
            int64_t at17       = (own & ~(int64_t)3) + 64;
            const bool here = col + q - 3 < end, need17 = !p.whole && (own & 3) != 0;
            for (int kb = 0; kb < p.stages; ++kb, at += 64 * p.ld, at17 += 64 * p.ld, ring.next()) {
                const int slot = ring.at, row = kb * 64 + who;
                ok = stream_wait(smem_u32(&bar_raw_empty[slot]), ring.phase ^ 1u, abort_flag);
                if (!ok)
                    break;
                const uint32_t to = smem_u32(smem) + kStreamSlots * SLOT + kStreamX * kStreamXBytes<NT> + slot * kStreamRawBytes;
                if (p.pieces) {
                    const uint32_t dst = to + (who * kStreamRow + h * kStreamHalf + q) * 4;
                    if (kb * 64 + 64 <= p.k && at + 64 * p.ld + 8 <= values) {
                        const float *src = matrix + at;
                        if (here)
#pragma unroll
                            for (int i = 0; i < 64 / kStreamFetch; ++i, src += step)
                                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + i * kStreamFetch * kStreamRow * 4), "l"(src) : "memory");
                    } else { // the matrix's last rows: pieces may reach past it
                        for (int i = 0; i < 64 / kStreamFetch; ++i) {
                            const int64_t from = at + i * step;
                            const int bytes    = values - from < 4 ? (int)(values - from) * 4 : 16;
                            if (here && row + kStreamFetch * i < p.k && bytes > 0)
                                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + i * kStreamFetch * kStreamRow * 4), "l"(matrix + from),
                                             "r"(bytes)
                                             : "memory");
                        }
                    }
                    if (need17) {
                        const int bytes = values - at17 < 4 ? (int)(values - at17) * 4 : 16;
                        if (kb * 64 + r17 < p.k && bytes > 0)
                            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + (r17 * kStreamRow + h17 * kStreamHalf + 64) * 4),
                                         "l"(matrix17 + at17), "r"(bytes)
                                         : "memory");
                    }
                } else { // value by value
#pragma unroll 4
                    for (int i = 0; i < 256 / kStreamFetch; ++i) {
                        const int r = (i >> 2) * kStreamFetch + who, c = (i & 3) * 32 + lane, half = c >> 6;
                        const int64_t at1 = begin + (int64_t)tile * TILE + (EPI::kTwin ? c & 63 : c);
                        if (kb * 64 + r < p.k && at1 < end)
                            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + (r * kStreamRow + half * kStreamHalf + (c & 63)) * 4),
                                         "l"((EPI::kTwin && half ? p.w2 : p.w) + (int64_t)(kb * 64 + r) * p.ld + at1)
                                         : "memory");
                    }
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&bar_raw[slot])) : "memory");
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory"); // none of this thread's copies is in flight when the CTA goes
    } else {
        // ===== converting =====
        // A warp has 16 columns, a lane two of them and of each eight values of k two at 2 g: with the 128-byte swizzle the four rows that a store
        // touches then lie in different banks, and so do those that it reads.
        const int who = (warp - 2 - kStreamDrain - kStreamFetch) % kStreamConvert, group = (warp - 2 - kStreamDrain - kStreamFetch) / kStreamConvert;
        const int g = lane >> 3, pair = lane & 7, local = who * 16 + pair * 2; // row of the accumulator
        const float *raw = reinterpret_cast<float *>(smem + kStreamSlots * SLOT + kStreamX * kStreamXBytes<NT>) + 2 * g * kStreamRow + (local >> 6) * kStreamHalf + (local & 63);
        const int chunk  = (local & 63) >> 3, ld3 = p.pieces ? (int)(p.ld & 3) : 0;
        int kb = group < p.stages ? group : 0;
        int tile_col = (int)(begin & 3) + (EPI::kTwin ? 0 : local & 64) + (group < p.stages ? 0 : TILE); // of the half that this warp converts, but for multiples of four
        static_assert(kStreamSlots == 2, "a group has a slot of its own");
        Ring<kStreamRaw> ring;
        Ring<8> scales;
        if (group)
            ring.next(), scales.next();
        uint32_t empty_phase = 1u;
        for (int s = group; s < total; s += 2, ring.next(), ring.next(), scales.next(), scales.next(), empty_phase ^= 1u) {
            const int slot = group, from_slot = ring.at;
            if (!__all_sync(0xffffffffu, stream_wait(smem_u32(&bar_raw[from_slot]), ring.phase, abort_flag)))
                break;
            const float *from = raw + from_slot * (kStreamRawBytes / 4);
            float2 x[16];
            if (p.whole) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    x[i] = *reinterpret_cast<const float2 *>(from + ((i >> 1) * 8 + (i & 1)) * kStreamRow);
            } else { // eight rows on, and 64 values of k, a row begins as far from a boundary
                const int even = p.pieces ? (2 * g * ld3 + tile_col) & 3 : 0, odd = p.pieces ? ((2 * g + 1) * ld3 + tile_col) & 3 : 0;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float *at = from + ((i >> 1) * 8 + (i & 1)) * kStreamRow + (i & 1 ? odd : even);
                    x[i]            = make_float2(at[0], at[1]);
                }
            }
            __syncwarp();
            if (lane == 0)
                mbar_arrive(smem_u32(&bar_raw_empty[from_slot]));
            const int left = (int)(p.k - kb * 64 < 64 ? p.k - kb * 64 : 64);
            if (left < 64)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (2 * g + (i >> 1) * 8 + (i & 1) >= left)
                        x[i] = make_float2(0.0f, 0.0f);
            for (kb += 2; kb >= p.stages; kb -= p.stages)
                tile_col += TILE;
            float m0 = 0.0f, m1 = 0.0f; // a NaN is passed over
#pragma unroll
            for (int i = 0; i < 16; ++i)
                m0 = fmaxf(m0, fabsf(x[i].x)), m1 = fmaxf(m1, fabsf(x[i].y));
#pragma unroll
            for (int o = 8; o < 32; o *= 2)
                m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o)), m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
            const bool finite = __all_sync(0xffffffffu, fmaxf(m0, m1) < INFINITY) != 0;
            if (!finite) { // rare: the scales are those of the finite values
                m0 = m1 = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    m0 = fmaxf(m0, __uint_as_float(finite_bits(x[i].x))), m1 = fmaxf(m1, __uint_as_float(finite_bits(x[i].y)));
#pragma unroll
                for (int o = 8; o < 32; o *= 2)
                    m0 = fmaxf(m0, __shfl_xor_sync(0xffffffffu, m0, o)), m1 = fmaxf(m1, __shfl_xor_sync(0xffffffffu, m1, o));
            }
            const float s0 = line_scale(__float_as_uint(m0)), s1 = line_scale(__float_as_uint(m1));
            if (!__all_sync(0xffffffffu, stream_wait(smem_u32(&bar_empty[slot]), empty_phase, abort_flag)))
                break;
            uint8_t *plane = smem + slot * SLOT + (local >> 6) * 8192 + (local & 7) * 2 + 2 * g * 128;
            const f32x2 by = pack2(s0, s1), by_lo = pack2(s0 * kLoScale, s1 * kLoScale);
            uint8_t *to[2] = {plane + ((chunk ^ (2 * g)) << 4), plane + 128 + ((chunk ^ (2 * g + 1)) << 4)};
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                // both columns at once: hi of v s, lo of v s 2^11 - hi 2^11, which is exact
                const f32x2 v = pack2(x[i].x, x[i].y);
                float a, b;
                unpack2(mul2(v, by), a, b);
                __half2 hi = __floats2half2_rn(a, b), lo;
                if (finite) {
                    float c, d;
                    unpack2(fma2(pack2(__low2float(hi), __high2float(hi)), dup2(0xC5000000u), mul2(v, by_lo)), c, d); // - 2048
                    lo = __floats2half2_rn(c, d);
                } else {
                    split2(a, b, hi, lo);
                }
                *reinterpret_cast<__half2 *>(to[i & 1] + (i >> 1) * 1024)         = hi;
                *reinterpret_cast<__half2 *>(to[i & 1] + kTile + (i >> 1) * 1024) = lo;
            }
            if (g == 0)
                *reinterpret_cast<char2 *>(&exponent_s[scales.at][local]) =
                    make_char2((signed char)line_exponent(__float_as_uint(m0)), (signed char)line_exponent(__float_as_uint(m1)));
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // written here, read by the tensor core
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(smem_u32(&bar_scale[scales.at]));
                mbar_arrive(smem_u32(&bar_full[slot]));
            }
        }
    }

    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, 512);
    }
    if (threadIdx.x == 0 && !failed && *abort_flag)
        atomicExch(p.flags + FLAG_TIMEOUT, 1u + (uint32_t)blockIdx.x);
}

inline int stream_grid(const DeviceState *st, int64_t n, int *per) {
    int64_t each = (n + st->sm_count - 1) / st->sm_count;
    each         = (each + 15) / 16 * 16;
    *per         = (int)each;
    return (int)((n + each - 1) / each);
}

template <class EPI, int NT>
ct_status launch_stream_of(DeviceState *st, const Planes &x, Stream p, const typename EPI::Params &e, const char *name) {
    StreamMaps maps;
    const uint64_t dims[2] = {(uint64_t)x.cols, (uint64_t)x.rows}, strides[1] = {(uint64_t)x.ld * 2};
    const uint32_t box[2]  = {64, NT};
    CT_TRY(encode_tiled_map_f16(&maps.x_hi, x.hi, 2, dims, strides, box, 128));
    CT_TRY(encode_tiled_map_f16(&maps.x_lo, x.lo, 2, dims, strides, box, 128));
    p.m      = (int)x.rows;
    p.stages = (int)((p.k + 63) / 64);
    auto whole = [](const void *q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; };
    p.pieces = whole(p.w) && whole(p.w2) ? 1 : 0;
    p.whole  = p.pieces && (p.ld & 3) == 0 ? 1 : 0;
    p.flags  = st->flags_dev;
    const int grid = stream_grid(st, p.n, &p.per);
    auto kernel    = stream_kernel<EPI, NT>;
    static bool attr_set_dev[16] = {};
    if (!attr_set_dev[st->device & 15]) {
        CT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kStreamSmem<NT>));
        attr_set_dev[st->device & 15] = true;
    }
    CT_CUDA(launch_dependent(kernel, dim3((unsigned)grid), dim3(kStreamThreads), (size_t)kStreamSmem<NT>, stream(), maps, p, e));
    CT_LAUNCH_CHECK(name);
    return CT_OK;
}
// Rows of x as planes [m][k], 64 a launch.  rows_from(e, r): the parameters for the rows from r on.
template <class EPI, typename F>
ct_status launch_stream(DeviceState *st, const Planes &x, Stream p, const typename EPI::Params &e, const char *name, F &&rows_from) {
    const float *row_scale = p.row_scale;
    for (int64_t r = 0; r < x.rows; r += 64) {
        Planes part = x;
        part.hi += r * x.ld, part.lo += r * x.ld, part.rows = std::min<int64_t>(64, x.rows - r);
        p.row_scale = row_scale + r;
        const typename EPI::Params f = rows_from(e, r);
        CT_TRY(x.rows <= 32 ? (launch_stream_of<EPI, 32>(st, part, p, f, name)) : (launch_stream_of<EPI, 64>(st, part, p, f, name)));
    }
    return CT_OK;
}

#endif // __CUDACC__

} // namespace fused
} // namespace ct
