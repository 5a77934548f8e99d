// Products of 17 to 128 rows: the weights are streamed through the tensor cores as they lie, float32, and read once.
//
// With so few rows a product is as long as it takes to read the weights, and writing their planes and reading them again is three times that
// (64 x 1024 x 32003: 76 us of pre-pass, 33 of product).  So eight warps load the weights into registers, 64 values of k of 128 columns a stage,
// split them under a scale per column and stage, and write the planes to shared memory.  The weights' columns are the rows of the accumulator
// (128 lanes), the rows of x its columns (32 or 64; more rows go by 64, a launch each), so that a scale belongs to a lane and a stage: four warps drain every stage and add it up
// in registers under its scale.  x comes as planes (K-major, a scale per row) by TMA.
// What bounds it is HBM; per stage the MMAs take 12 x 54 clocks (64 rows) of the 1400 in which its 32 KB arrive.
// A CTA has a range of columns, a multiple of 16, so that all CTAs have as much to read.
//
// Epilogue: the tile's sums go to shared memory as [row of x][column]; the draining warps do with them what EPI says.
#pragma once

#include "fused_product.cuh"

namespace ct {
namespace fused {

constexpr int64_t kStreamRows = 128; // at most, 64 a launch
constexpr int kStreamSlots   = 2;
constexpr int kStreamThreads = 14 * 32; // TMA, MMA, four draining, eight converting warps
constexpr int kStreamPitch   = 129;
template <int NT> constexpr int kStreamSlot = 2 * kTile + 2 * NT * 128; // planes of the weights, then of x
template <int NT> constexpr int kStreamSmem = kStreamSlots * kStreamSlot<NT> + NT * kStreamPitch * 4 + 1024;

struct Stream {
    const float *w, *w2; // w2: twin epilogues, the second matrix (tiles of 64 columns of both)
    int64_t k, n, ld;    // ld: values between the weights' rows
    int m, per;          // rows of x; columns of a CTA
    int stages;
    int pairs;           // two columns of a row are an aligned 8 bytes
    const float *row_scale;
    uint32_t *flags;
};
struct StreamMaps {
    CUtensorMap x_hi, x_lo;
};

// Sums are kept 2^14 lower, as those of x itself are: weights of 1e36 then overflow no earlier than the result.
constexpr float kStreamDown = 1.0f / 16384.0f, kStreamUp = 16384.0f;

#ifdef __CUDACC__

// EPI: kTwin; Params; State (of a draining thread, across the CTA's tiles); tile<NT>(p, e, state, z, c0, cols, t): z[row * kStreamPitch + c] the
// sums over 2^14, but for the row's scale, of the tile's columns c0 + c < c0 + cols (twin: the second matrix's at 64 + c), t the thread of 128; finish<NT>(p, e, state, t).
template <class EPI, int NT>
__global__ void __launch_bounds__(kStreamThreads, 1)
    stream_kernel(const __grid_constant__ StreamMaps maps, const __grid_constant__ Stream p, const __grid_constant__ typename EPI::Params e) {
    constexpr int TILE = EPI::kTwin ? 64 : 128, SLOT = kStreamSlot<NT>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bar_full[kStreamSlots], bar_empty[kStreamSlots], bar_scale[4], bar_acc_full[2], bar_acc_empty[2], bar_done;
    __shared__ uint32_t tmem_base_slot;
    __shared__ int abort_flag_s;
    __shared__ float scale_s[4][128]; // inverse scales of a stage's columns; a converting warp is at most four stages ahead of the draining ones
    volatile int *abort_flag = &abort_flag_s;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    griddep_launch_dependents();
    if (threadIdx.x == 0)
        abort_flag_s = *reinterpret_cast<volatile uint32_t *>(p.flags + FLAG_TIMEOUT) != 0 ? 1 : 0;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t *smem            = smem_raw + (smem_base - smem_u32(smem_raw));
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStreamSlots; ++s) {
            mbar_init(smem_u32(&bar_full[s]), 9); // eight converting warps, and x
            mbar_init(smem_u32(&bar_empty[s]), 1);
        }
        for (int s = 0; s < 4; ++s)
            mbar_init(smem_u32(&bar_scale[s]), 8);
        for (int s = 0; s < 2; ++s) {
            mbar_init(smem_u32(&bar_acc_full[s]), 1);
            mbar_init(smem_u32(&bar_acc_empty[s]), 4);
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
    const int64_t begin = (int64_t)blockIdx.x * p.per, end = min(p.n, begin + p.per);
    const int tiles = (int)((end - begin + TILE - 1) / TILE), total = tiles * p.stages; // stages numbered across tiles

    if (failed) {
    } else if (warp == 0) {
        // ===== x =====
        if (elect_one()) {
            int issued = 0;
            for (int tile = 0, s = 0; tile < tiles && !*abort_flag; ++tile)
                for (int kb = 0; kb < p.stages; ++kb, ++s) {
                    const int slot = s % kStreamSlots;
                    if (!mbar_wait(smem_u32(&bar_empty[slot]), (uint32_t)(s / kStreamSlots + 1) & 1u, abort_flag))
                        break;
                    const uint32_t full = smem_u32(&bar_full[slot]), dst = smem_base + slot * SLOT + 2 * kTile;
                    mbar_expect_tx(full, 2 * NT * 128);
                    tma_load_2d(dst, &maps.x_hi, full, kb * 64, 0);
                    tma_load_2d(dst + NT * 128, &maps.x_lo, full, kb * 64, 0);
                    issued = s + 1;
                }
            if (*abort_flag) {
                // unwind: copies land on their own, but the barrier that counts them counts converting warps too: give them the
                // time that a wait has
                const uint64_t t0 = globaltimer_ns();
                while (issued > 0 && globaltimer_ns() - t0 < 1000000ull) {
                }
            }
        }
    } else if (warp == 1) {
        // ===== MMA =====
        if (elect_one()) {
            constexpr uint32_t idesc = make_idesc(0u, 128, NT) | 1u << 15; // the weights are MN-major
            bool ok = true;
            for (int s = 0; s < total && ok; ++s) {
                const int slot = s % kStreamSlots, set = s & 1;
                ok = mbar_wait(smem_u32(&bar_full[slot]), (uint32_t)(s / kStreamSlots) & 1u, abort_flag) &&
                     mbar_wait(smem_u32(&bar_acc_empty[set]), (uint32_t)((s >> 1) + 1) & 1u, abort_flag);
                if (!ok)
                    break;
                tc_fence_after_sync();
                const uint32_t at    = smem_base + slot * SLOT;
                const uint64_t w_hi = desc_mn(at), w_lo = desc_mn(at + kTile);
                const uint64_t x_hi = smem_desc_k<128>(at + 2 * kTile), x_lo = smem_desc_k<128>(at + 2 * kTile + NT * 128);
                const uint32_t d_main = tmem_base + set * 256, d_cross = d_main + 128;
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    mma_f16(d_cross, w_lo + 128 * kk, x_hi + 2 * kk, idesc, kk > 0);
                    mma_f16(d_cross, w_hi + 128 * kk, x_lo + 2 * kk, idesc, 1u);
                    mma_f16(d_main, w_hi + 128 * kk, x_hi + 2 * kk, idesc, kk > 0);
                }
                tc_commit(smem_u32(&bar_empty[slot]));
                tc_commit(smem_u32(&bar_acc_full[set]));
            }
            if (!ok || *abort_flag) {
                tc_commit(smem_u32(&bar_done));
                const uint64_t t0 = globaltimer_ns();
                while (!mbar_try_wait(smem_u32(&bar_done), 0) && globaltimer_ns() - t0 < kWaitBudgetNs) {
                }
            }
        }
    } else if (warp < 6) {
        // ===== draining =====
        const int quarter = warp & 3, t = (warp - 2) * 32 + lane, row = quarter * 32 + lane; // a thread's row: a column of the tile
        float *z = reinterpret_cast<float *>(smem + kStreamSlots * SLOT);
        typename EPI::State state;
        EPI::init(state);
        bool ok = true;
        for (int tile = 0, s = 0; tile < tiles; ++tile) { // all warps take all tiles' barriers, also after a failed wait
            float acc[NT];
#pragma unroll
            for (int j = 0; j < NT; ++j)
                acc[j] = 0.0f;
#pragma unroll 1
            for (int kb = 0; kb < p.stages; ++kb, ++s) {
                const int set = s & 1;
                if (ok)
                    ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_acc_full[set]), (uint32_t)(s >> 1) & 1u, abort_flag) &&
                                                     mbar_wait(smem_u32(&bar_scale[s & 3]), (uint32_t)(s >> 2) & 1u, abort_flag)) != 0;
                if (!ok)
                    continue;
                tc_fence_after_sync();
                const float by = scale_s[s & 3][row];
                const uint32_t at = tmem_base + ((uint32_t)(quarter * 32) << 16) + set * 256;
#pragma unroll
                for (int g = 0; g < NT / 16; ++g) {
                    uint32_t a[16], b[16];
                    tmem_ld_32x16(at + g * 16, a);
                    tmem_ld_32x16(at + 128 + g * 16, b);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 16; ++j)
                        acc[g * 16 + j] = __fmaf_rn(__fmaf_rn(__uint_as_float(b[j]), kLoInv, __uint_as_float(a[j])), by, acc[g * 16 + j]);
                }
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(smem_u32(&bar_acc_empty[set]));
            }
            asm volatile("bar.sync 1, 128;" ::: "memory"); // the last tile's sums have been read
#pragma unroll
            for (int j = 0; j < NT; ++j)
                z[j * kStreamPitch + row] = acc[j];
            asm volatile("bar.sync 1, 128;" ::: "memory");
            const int64_t c0 = begin + (int64_t)tile * TILE;
            if (ok)
                EPI::template tile<NT>(p, e, state, z, c0, (int)(end - c0 < TILE ? end - c0 : TILE), t);
        }
        if (ok)
            EPI::template finish<NT>(p, e, state, t);
    } else {
        // ===== converting =====
        // A warp has 16 columns, a lane two of them and of each eight values of k two at 2 g: with the 128-byte swizzle the four rows that a store
        // touches then lie in different banks.
        const int who = warp - 6, g = lane >> 3, pair = lane & 7;
        const int local = who * 16 + pair * 2; // row of the accumulator
        const float *w  = EPI::kTwin && who >= 4 ? p.w2 : p.w;
        float2 v[3][16];
        auto load = [&](float2 (&to)[16], int s) {
            const int tile = s / p.stages, kb = s - tile * p.stages;
            const int64_t col  = begin + (int64_t)tile * TILE + (EPI::kTwin ? local & 63 : local);
            const int64_t k0   = (int64_t)kb * 64 + 2 * g;
            const float *src   = w + k0 * p.ld + col;
            const bool first   = s < total && col < end, second = first && col + 1 < end;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int64_t k = (i >> 1) * 8 + (i & 1);
                to[i]           = make_float2(0.0f, 0.0f);
                if (first && k0 + k < p.k) {
                    if (p.pairs && second) {
                        to[i] = __ldcs(reinterpret_cast<const float2 *>(src + k * p.ld));
                    } else {
                        to[i].x = __ldcs(src + k * p.ld);
                        if (second)
                            to[i].y = __ldcs(src + k * p.ld + 1);
                    }
                }
            }
        };
        auto convert = [&](const float2 (&x)[16], int s) {
            const int slot = s % kStreamSlots;
            uint32_t m0 = 0, m1 = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i)
                m0 = max(m0, finite_bits(x[i].x)), m1 = max(m1, finite_bits(x[i].y));
            m0 = max(m0, __shfl_xor_sync(0xffffffffu, m0, 8)), m1 = max(m1, __shfl_xor_sync(0xffffffffu, m1, 8));
            m0 = max(m0, __shfl_xor_sync(0xffffffffu, m0, 16)), m1 = max(m1, __shfl_xor_sync(0xffffffffu, m1, 16));
            const float s0 = line_scale(m0), s1 = line_scale(m1);
            if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&bar_empty[slot]), (uint32_t)(s / kStreamSlots + 1) & 1u, abort_flag)))
                return false;
            uint8_t *plane = smem + slot * SLOT + (local >> 6) * 8192 + (local & 7) * 2;
            const int chunk = (local & 63) >> 3;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int k = (i >> 1) * 8 + 2 * g + (i & 1);
                __half2 hi, lo;
                split2(x[i].x * s0, x[i].y * s1, hi, lo);
                *reinterpret_cast<__half2 *>(plane + k * 128 + ((chunk ^ (k & 7)) << 4))         = hi;
                *reinterpret_cast<__half2 *>(plane + kTile + k * 128 + ((chunk ^ (k & 7)) << 4)) = lo;
            }
            if (g == 0)
                *reinterpret_cast<float2 *>(&scale_s[s & 3][local]) = make_float2(line_inverse(m0) * kStreamDown, line_inverse(m1) * kStreamDown);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); // written here, read by the tensor core
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(smem_u32(&bar_scale[s & 3]));
                mbar_arrive(smem_u32(&bar_full[slot]));
            }
            return true;
        };
        load(v[0], 0);
        load(v[1], 1);
        for (int s = 0; s < total; s += 3) {
            load(v[2], s + 2);
            if (!convert(v[0], s))
                break;
            if (s + 1 >= total)
                break;
            load(v[0], s + 3);
            if (!convert(v[1], s + 1))
                break;
            if (s + 2 >= total)
                break;
            load(v[1], s + 4);
            if (!convert(v[2], s + 2))
                break;
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
    auto whole = [](const void *q) { return (reinterpret_cast<uintptr_t>(q) & 7u) == 0; };
    p.pairs  = (p.ld & 1) == 0 && whole(p.w) && whole(p.w2) ? 1 : 0;
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
// Rows of x as planes [m][k], m <= kStreamRows.  rows_from(e, r): the parameters for the rows from r on.
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
// Threads that share a row in an epilogue that gives each thread a row.
inline int stream_shares(int64_t m) { return m <= 32 ? 4 : 2; }

#endif // __CUDACC__

} // namespace fused
} // namespace ct
