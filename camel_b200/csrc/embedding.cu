// Embedding lookup, and the gradient of its table.
//
//   out[i] = scale table[ids[i]];   dtable[v] = scale (sum of dout[i] over the i with ids[i] = v)
//
// Both are bound by memory: a lookup reads a row and writes one, the gradient reads dout once and writes every row of the table.
// Gradient: the tokens are sorted by id (stable, so that sums have one order), then warps walk the tokens and the rows together.  Rows
// without a token are as many as there are stores of zeros, rows with thousands as many as there are loads, so what is cut into equal slices is
// the merged list of both: each token, and behind its last token the end of each row.  A row that lies across slices leaves a partial
// sum in each, which a third kernel adds up.  Few tokens are found by each block for its own rows, in one launch.  Sums are kept in 64 bits and rounded once; their
// order follows from the ids, the sizes and the device, and not from when a block runs.
// Measured (L2 flushed): 32768 rows of 50257 x 2048 59 to 61 us (348 MB, 0.88 to 0.90 of a copy); gradient of 16384 tokens in the same table 111 us (546 MB,
// 0.75: sorting 15, sums 91, joining the rest), of 1537 in 2050 x 771 12 us in one (11 MB; each block's chain of loads), of 1000 in 100 x 64 5 in line.
// Times at the rules below are of a lone call between two events, L2 flushed, with the events' own 4 us or so, unless in line is said: call behind call.
#include "common.cuh"
#include "tc_ptx.cuh"

#include <algorithm>
#include <cfloat>
#include <cmath>

namespace ct {
namespace {

using namespace ptx;

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ---- lookup -------------------------------------------------------------------------------------

// TPR threads to a piece of a row, 16 values each: float4 j of thread t is at 4 (j TPR + t), or value j of it at j TPR + t.
constexpr int kLookupValues = 16;
template <int TPR, bool VEC>
__global__ void __launch_bounds__(256) embedding_kernel(
    const float *__restrict__ table, const int64_t *__restrict__ ids, int64_t m, int64_t n, int64_t k, int64_t pieces, float scale,
    float *__restrict__ out, int early) {
    griddep_wait();
    if (early)
        griddep_launch_dependents();
    const int t = threadIdx.x % TPR;
    const int64_t units = m * pieces;
    for (int64_t u = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR; u < units; u += (int64_t)gridDim.x * (256 / TPR)) {
        const int64_t i = pieces == 1 ? u : u / pieces, c0 = (u - i * pieces) * (TPR * kLookupValues);
        const int64_t id = ids[i], left = k - c0;
        const bool has   = id >= 0 && id < n;
        const float *src = table + (has ? id : 0) * k + c0;
        float *dst       = out + i * k + c0;
        if (VEC) {
            float4 v[kLookupValues / 4];
#pragma unroll
            for (int j = 0; j < kLookupValues / 4; ++j) {
                const int c = (j * TPR + t) * 4;
                v[j]        = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (has && c < left) {
                    v[j] = *reinterpret_cast<const float4 *>(src + c);
                    v[j] = make_float4(__fmul_rn(v[j].x, scale), __fmul_rn(v[j].y, scale), __fmul_rn(v[j].z, scale), __fmul_rn(v[j].w, scale));
                }
            }
#pragma unroll
            for (int j = 0; j < kLookupValues / 4; ++j) {
                const int c = (j * TPR + t) * 4;
                if (c < left)
                    __stcs(reinterpret_cast<float4 *>(dst + c), v[j]);
            }
        } else {
            float v[kLookupValues];
#pragma unroll
            for (int j = 0; j < kLookupValues; ++j)
                v[j] = has && j * TPR + t < left ? __fmul_rn(src[j * TPR + t], scale) : 0.0f;
#pragma unroll
            for (int j = 0; j < kLookupValues; ++j)
                if (j * TPR + t < left)
                    __stcs(dst + j * TPR + t, v[j]);
        }
    }
}

// ---- tokens by id -------------------------------------------------------------------------------

// One cluster sorts: each CTA has a range of the tokens, each of its warps a range of that.  A pass over `bits` bits of the ids counts each
// warp's digits, adds up the counts in the order of warps and CTAs, and puts every token behind those of smaller digits and those before it.
// ROUNDS: tokens of a lane, which stay in its registers from the count to the end of a pass; 0: any number, read twice.
constexpr int kSortWarps = 32, kSortBits = 10;
struct Sorted {
    uint32_t *ids[2], *at[2]; // two places each: a pass goes from one to the other
    uint32_t *counts;         // [0] tokens with an id of the table; [1] rows across slices (of the kernel behind)
};

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa(addr, rank)) : "memory");
    return v;
}

template <int CTAS, int ROUNDS>
__global__ void __launch_bounds__(kSortWarps * 32) embedding_sort_kernel(
    const int64_t *__restrict__ ids, uint32_t m, uint32_t n, int passes, int bits, Sorted s) {
    extern __shared__ uint32_t smem[];
    const int bins   = 1 << bits;
    uint32_t *counts = smem;                      // [warp][bin]
    uint32_t *totals = counts + kSortWarps * bins; // of this CTA, and behind them its tokens without a row
    uint32_t *base   = totals + bins + 1;
    __shared__ uint32_t warp_sums[kSortWarps];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const uint32_t rank = cluster_rank();
    const uint32_t each = ((m + CTAS * kSortWarps - 1) / (CTAS * kSortWarps) + 31) & ~31u; // tokens of a warp
    const uint64_t lo64 = (uint64_t)(rank * kSortWarps + warp) * each;
    const uint32_t lo = (uint32_t)min(lo64, (uint64_t)m), hi = (uint32_t)min(lo64 + each, (uint64_t)m);
    const uint32_t totals_at = static_cast<uint32_t>(__cvta_generic_to_shared(totals));
    uint32_t *mine           = counts + warp * bins;
    griddep_wait();
    griddep_launch_dependents(); // the sums' kernel reads what this one writes from L2
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * bits, from = pass & 1, to = from ^ 1;
        auto id_of      = [&](uint32_t i) -> uint32_t {
            if (pass)
                return __ldcg(s.ids[from] + i);
            const int64_t id = ids[i];
            return id >= 0 && id < (int64_t)n ? (uint32_t)id : n;
        };
        // Counts a round of the warp, and says how many tokens of its digit a lane's has before it.
        auto count = [&](uint32_t id, bool here) -> uint32_t {
            // lanes of the same digit, bit by bit (__match_any_sync takes 250 clocks, these 30)
            const uint32_t d = (id >> shift) & (bins - 1);
            uint32_t alike   = __ballot_sync(0xffffffffu, here);
            for (int b = 0; b < bits; ++b) {
                const uint32_t set = __ballot_sync(0xffffffffu, (d >> b) & 1);
                alike &= (d >> b) & 1 ? set : ~set;
            }
            const uint32_t ahead = __popc(alike & ((1u << lane) - 1));
            const uint32_t place = here ? mine[d] + ahead : 0;
            __syncwarp();
            if (here && ahead == 0)
                mine[d] += __popc(alike);
            __syncwarp();
            return place;
        };
        uint32_t id[ROUNDS ? ROUNDS : 1], at[ROUNDS ? ROUNDS : 1], place[ROUNDS ? ROUNDS : 1];
        if (ROUNDS) {
#pragma unroll
            for (int r = 0; r < ROUNDS; ++r) {
                const uint32_t i = lo + r * 32 + lane;
                // (without conditions: each load would wait for the one before)
                id[r] = id_of(min(i, m - 1)), at[r] = pass ? __ldcg(s.at[from] + min(i, m - 1)) : i;
            }
        }
        for (int i = lane; i < bins; i += 32)
            mine[i] = 0;
        if (t == 0)
            totals[bins] = 0;
        __syncthreads();
        uint32_t none = 0;
        if (ROUNDS) {
#pragma unroll
            for (int r = 0; r < ROUNDS; ++r) {
                const bool here = lo + r * 32 + lane < hi;
                none += here && id[r] == n;
                place[r] = count(id[r], here);
            }
        } else {
#pragma unroll 4
            for (uint32_t i = lo + lane; i < hi; i += 32) {
                const uint32_t v = id_of(i);
                none += v == n;
                atomicAdd(&mine[(v >> shift) & (bins - 1)], 1u);
            }
        }
        none = __reduce_add_sync(0xffffffffu, none);
        if (none && lane == 0)
            atomicAdd(&totals[bins], none);
        __syncthreads();
        for (int d = t; d < bins; d += kSortWarps * 32) {
            uint32_t sum = 0, c[kSortWarps];
#pragma unroll
            for (int w = 0; w < kSortWarps; ++w)
                c[w] = counts[w * bins + d];
#pragma unroll
            for (int w = 0; w < kSortWarps; ++w) {
                counts[w * bins + d] = sum;
                sum += c[w];
            }
            totals[d] = sum;
        }
        cluster_sync();
        uint32_t before = 0, all = 0; // of this thread's digit (bins <= threads)
        if (t < bins) {
            uint32_t c[CTAS];
#pragma unroll
            for (int r = 0; r < CTAS; ++r)
                c[r] = ld_cluster_u32(totals_at + t * 4, r);
#pragma unroll
            for (int r = 0; r < CTAS; ++r) {
                before += r < (int)rank ? c[r] : 0;
                all += c[r];
            }
        }
        if (pass == 0 && rank == 0 && warp == kSortWarps - 1) {
            const uint32_t none_of = lane < CTAS ? ld_cluster_u32(totals_at + bins * 4, lane) : 0;
            const uint32_t without = __reduce_add_sync(0xffffffffu, none_of);
            if (lane == 0)
                s.counts[0] = m - without, s.counts[1] = 0;
        }
        cluster_arrive(); // this CTA has read the others' totals
        uint32_t upto = all; // over digits, this one included
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
            upto += lane >= o ? v : 0;
        }
        if (lane == 31)
            warp_sums[warp] = upto;
        __syncthreads();
        const uint32_t digits = __reduce_add_sync(0xffffffffu, lane < warp ? warp_sums[lane] : 0);
        if (t < bins)
            base[t] = digits + upto - all + before;
        __syncthreads();
        auto put = [&](uint32_t id, uint32_t at, uint32_t place) {
            s.ids[to][place] = id;
            s.at[to][place]  = at;
        };
        if (ROUNDS) {
#pragma unroll
            for (int r = 0; r < ROUNDS; ++r) {
                const uint32_t d = (id[r] >> shift) & (bins - 1);
                if (lo + r * 32 + lane < hi)
                    put(id[r], at[r], base[d] + mine[d] + place[r]);
            }
            // (mine holds the counts of the warps before: a lane's place is by its own warp's, taken before they were replaced)
        } else {
            for (uint32_t i0 = lo; i0 < hi; i0 += 32) {
                const uint32_t i = i0 + lane;
                const bool here  = i < hi;
                const uint32_t v = here ? id_of(i) : 0, a = here && pass ? __ldcg(s.at[from] + i) : i;
                const uint32_t p = count(v, here); // from the counts of the warps before on
                if (here)
                    put(v, a, base[(v >> shift) & (bins - 1)] + p);
            }
        }
        cluster_wait();
        if (pass + 1 < passes)
            cluster_sync(); // the next pass reads what the others wrote
    }
}

// ---- sums ---------------------------------------------------------------------------------------

// Where a slice begins: its first token, and the row that that is in or before.
struct Begin {
    uint32_t token, row;
};
// Of two slices' beginnings, d[0] and d[1] places behind that of the merged list, in which token i is number i + ids[i].  A row that lies across, but by
// fewer than about `near` tokens (32 at most, or a multiple of 32), belongs to the slice before.
__device__ __forceinline__ void beginnings(
    const uint32_t *__restrict__ ids, uint32_t tokens, uint32_t n, uint32_t near, const uint64_t (&d)[2], int lane, Begin (&b)[2], bool (&goes_on)[2]) {
    uint32_t lo[2], hi[2];
#pragma unroll
    for (int q = 0; q < 2; ++q)
        lo[q] = d[q] > n ? (uint32_t)(d[q] - n) : 0, hi[q] = (uint32_t)min(d[q], (uint64_t)tokens);
    while (lo[0] < hi[0] || lo[1] < hi[1]) {
        uint32_t step[2], id[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            step[q]          = (hi[q] - lo[q] + 31) / 32;
            const uint32_t i = lo[q] + lane * step[q];
            id[q]            = __ldcg(ids + min(i, tokens - 1)); // (tokens > 0: there is something to look for)
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const uint32_t i = lo[q] + lane * step[q];
            const int before = __popc(__ballot_sync(0xffffffffu, i < hi[q] && (uint64_t)i + id[q] < d[q]));
            if (before == 0)
                hi[q] = lo[q];
            else
                hi[q] = min(hi[q], lo[q] + before * step[q]), lo[q] = lo[q] + (before - 1) * step[q] + 1;
        }
    }
    // the row's tokens from there on, up to `near`: every step-th of them, and those behind the last one that is its
    const uint32_t step = max(near / 32, 1u), probes = min(near, 32u);
    uint32_t last[2], next[2], more[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        last[q] = __ldcg(ids + max(lo[q], 1u) - 1), next[q] = __ldcg(ids + min(lo[q] + lane * step, max(tokens, 1u) - 1));
        b[q]       = {lo[q], (uint32_t)(d[q] - lo[q])};
        goes_on[q] = lo[q] > 0 && last[q] == b[q].row && d[q] < (uint64_t)n + tokens; // the row has tokens in slices before
        hi[q]      = __popc(__ballot_sync(0xffffffffu, lane < probes && lo[q] + lane * step < tokens && next[q] == b[q].row));
        lo[q] += hi[q] ? (hi[q] - 1) * step + 1 : 0;
    }
#pragma unroll
    for (int q = 0; q < 2; ++q)
        more[q] = __ldcg(ids + min(lo[q] + lane, max(tokens, 1u) - 1));
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int beyond = __popc(__ballot_sync(0xffffffffu, lo[q] + lane < tokens && lane < (int)step - 1 && more[q] == b[q].row));
        if (goes_on[q] && hi[q] < probes)
            b[q].token = lo[q] + (hi[q] ? beyond : 0), ++b[q].row, goes_on[q] = false;
    }
}

enum SliceState : uint8_t { SLICE_THROUGH = 1 }; // all of it belongs to a row that began before and ends behind

// A warp to a slice and 128 V columns.
template <int V, int AT_ONCE, int FIT, bool VEC>
__global__ void __launch_bounds__(256, FIT) embedding_grad_kernel(
    const uint32_t *__restrict__ ids, const uint32_t *__restrict__ at, uint32_t *__restrict__ counts, const float *__restrict__ dout, uint32_t n,
    int64_t k, float scale, uint32_t slices, uint32_t strips, float *__restrict__ dtable, double *__restrict__ head, double *__restrict__ tail,
    uint8_t *__restrict__ states, uint2 *__restrict__ across) {
    griddep_wait();
    const int lane       = threadIdx.x & 31;
    const uint64_t unit  = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const uint32_t slice = (uint32_t)(unit / strips), strip = (uint32_t)(unit - (uint64_t)slice * strips);
    if (slice >= slices)
        return;
    const int64_t c0 = (int64_t)strip * 128 * V;
    auto column      = [&](int j, int q) -> int64_t { return c0 + (VEC ? (j * 32 + lane) * 4 + q : (j * 4 + q) * 32 + lane); };
    const uint32_t tokens = __ldcg(counts);
    const uint64_t total  = (uint64_t)n + tokens, each = (total + slices - 1) / slices;
    const uint64_t d[2]   = {min((uint64_t)slice * each, total), min((uint64_t)(slice + 1) * each, total)};
    // half a slice, at least 8
    const uint32_t near = each >= 64 ? (uint32_t)min(each / 2, (uint64_t)1024) & ~31u : max((uint32_t)each / 2, 8u);
    Begin bounds[2];
    bool goes_on[2];
    beginnings(ids, tokens, n, near, d, lane, bounds, goes_on);
    const uint32_t i0 = bounds[0].token, i1 = bounds[1].token, r0 = bounds[0].row, r1 = bounds[1].row;
    double sum[4 * V];
#pragma unroll
    for (int j = 0; j < 4 * V; ++j)
        sum[j] = 0.0;
    auto leave = [&](double *to) {
        to += (int64_t)slice * k;
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (column(j, q) < k)
                    to[column(j, q)] = sum[4 * j + q];
    };
    auto finish = [&](uint32_t row) {
        if (row == r0 && goes_on[0]) {
            leave(head);
        } else {
            float *to = dtable + (int64_t)row * k;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                if (VEC) {
                    if (column(j, 0) < k)
                        __stcs(reinterpret_cast<float4 *>(to + column(j, 0)),
                               make_float4((float)(sum[4 * j] * scale), (float)(sum[4 * j + 1] * scale), (float)(sum[4 * j + 2] * scale),
                                           (float)(sum[4 * j + 3] * scale)));
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (column(j, q) < k)
                            __stcs(to + column(j, q), (float)(sum[4 * j + q] * scale));
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 4 * V; ++j)
            sum[j] = 0.0;
    };
    // Rows without a token.  Those that begin anywhere are cleared as what they are together, a stretch of which each strip has a part (16384 x 50257 x 2047 120 us
    // so, 125 row by row).
    auto clear = [&](uint32_t first, uint32_t last) {
        float *to = dtable + (int64_t)first * k;
        if (VEC) {
            for (uint32_t row = first; row < last; ++row, to += k)
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (column(j, 0) < k)
                        __stcs(reinterpret_cast<float4 *>(to + column(j, 0)), make_float4(0.0f, 0.0f, 0.0f, 0.0f));
            return;
        }
        int64_t count = (int64_t)(last - first) * k;
        if (strips > 1) {
            const int64_t part = count < (int64_t)1 << 32 ? (uint32_t)count / strips + 1 : count / strips + 1, begin = min(part * strip, count);
            count              = min(part, count - begin);
            to += begin;
        }
        const int ahead      = (int)min((int64_t)(-(reinterpret_cast<uintptr_t>(to) >> 2) & 3), count);
        const int64_t pieces = (count - ahead) / 4;
        if (lane < ahead)
            to[lane] = 0.0f;
        to += ahead;
        for (int64_t i = lane; i < pieces; i += 32)
            __stcs(reinterpret_cast<float4 *>(to) + i, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
        if (lane < count - ahead - 4 * pieces)
            to[4 * pieces + lane] = 0.0f;
    };
    uint32_t row = r0;
    bool open    = goes_on[0]; // whether the row has tokens
    auto go_to   = [&](uint32_t next) {
        if (row < next) {
            if (open)
                finish(row);
            clear(row + open, next);
            row = next, open = false;
        }
    };
    constexpr int kAtOnce = AT_ONCE;
    for (uint32_t i = i0; i < i1; i += 32) {
        const uint32_t mine = __ldcg(ids + min(i + lane, i1 - 1)), mine_at = __ldcg(at + min(i + lane, i1 - 1));
        const int count = min(32u, i1 - i);
        for (int g = 0; g < count; g += kAtOnce) {
            float v[kAtOnce][4 * V];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                // without conditions, which would make each load wait for the one before: the last token or column again
                const float *src = dout + (int64_t)__shfl_sync(0xffffffffu, mine_at, min(g + u, count - 1)) * k;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (VEC) {
                        const float4 f = *reinterpret_cast<const float4 *>(src + min(column(j, 0), k - 4));
                        v[u][4 * j] = f.x, v[u][4 * j + 1] = f.y, v[u][4 * j + 2] = f.z, v[u][4 * j + 3] = f.w;
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            v[u][4 * j + q] = src[min(column(j, q), k - 1)];
                    }
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const uint32_t id = __shfl_sync(0xffffffffu, mine, (g + u) & 31);
                if (g + u < count) {
                    go_to(id);
                    open = true;
#pragma unroll
                    for (int j = 0; j < 4 * V; ++j)
                        sum[j] += (double)v[u][j];
                }
            }
        }
    }
    go_to(r1);
    const bool through = goes_on[0] && r0 == r1;
    if (goes_on[1]) // row r1 ends in a later slice
        leave(tail);
    if (strip == 0 && lane == 0) {
        states[slice] = through ? SLICE_THROUGH : 0;
        if (goes_on[0] && r0 < r1)
            across[atomicAdd(counts + 1, 1u)] = make_uint2(slice, r0); // in any order: each is a row of its own
    }
}

// The rows that lie across slices: what each slice left of it, the last one's first.  A block has 32 columns of a row, and eight parts of its slices.
__global__ void __launch_bounds__(256) embedding_join_kernel(
    const uint32_t *__restrict__ counts, int64_t k, float scale, uint32_t column_blocks, const double *__restrict__ head, const double *__restrict__ tail,
    const uint8_t *__restrict__ states, const uint2 *__restrict__ across, float *__restrict__ dtable) {
    __shared__ double part[8][32];
    griddep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t units = (uint64_t)__ldcg(counts + 1) * column_blocks;
    for (uint64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const uint2 last     = __ldcg(across + u / column_blocks); // the slice in which the row ends, and the row
        const int64_t c      = (int64_t)(u % column_blocks) * 32 + lane;
        uint32_t first       = last.x - 1; // the slice in which it begins, 32 of them looked at together
        for (;;) {
            const bool through    = lane <= first && (__ldcg(states + first - lane) & SLICE_THROUGH);
            const uint32_t beyond = __ballot_sync(0xffffffffu, !through);
            if (beyond) {
                first -= __ffs(beyond) - 1;
                break;
            }
            first -= 32;
        }
        double sum = 0.0;
        if (c < k) {
#pragma unroll 8
            for (uint32_t s = first + warp; s < last.x; s += 8)
                sum += __ldcg(tail + (int64_t)s * k + c);
        }
        part[warp][lane] = sum;
        __syncthreads();
        if (warp == 0 && c < k) {
            sum = __ldcg(head + (int64_t)last.x * k + c);
#pragma unroll
            for (int w = 0; w < 8; ++w)
                sum += part[w][lane];
            dtable[(int64_t)last.y * k + c] = (float)(sum * scale);
        }
        __syncthreads();
    }
}

// ---- few tokens -----------------------------------------------------------------------------------

// A block has 128 columns of every apart-th row, since those that follow one another may be the words that come most often (1000 x 3000 x 1000 15 us with rows that do,
// 8 so).  It looks through all ids for those of its rows, ranks them by row as the sorting kernel does, in shared memory, and adds up: a warp to a row, or all of
// them, each a part of its tokens, to a row of more than kAloneTokens.
constexpr uint32_t kNoRow  = 0xffffffffu;
constexpr int kAloneTokens = 48, kFewRows = 512; // (with 16 more rows are taken one after the other)
template <int TOKENS, bool VEC>
__global__ void __launch_bounds__(256) embedding_grad_few_kernel(
    const int64_t *__restrict__ ids, const float *__restrict__ dout, int m, int64_t n, int64_t k, int rows, uint32_t apart, int strips, float scale,
    float *__restrict__ dtable) {
    constexpr int TURNS = TOKENS / 256, AT_ONCE = 8;
    __shared__ uint32_t counts[8][kFewRows], begins[kFewRows + 1], warp_sums[8];
    __shared__ uint16_t order[TOKENS], many[kFewRows];
    __shared__ double part[8][128];
    __shared__ int many_count;
    griddep_wait();
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const uint32_t range = blockIdx.x / strips;
    const int64_t c0     = (int64_t)(blockIdx.x - range * strips) * 128;
    const int here = (int)((n - 1 - range) / apart) + 1; // row range + r apart is its row r
    uint32_t place[TURNS]; // the token's row of the block, and behind the 16th bit its place among the warp's tokens of that row
#pragma unroll
    for (int i = 0; i < TURNS; ++i) { // (without conditions: each load would wait for the one before)
        const int64_t id = ids[min((warp * TURNS + i) * 32 + lane, m - 1)];
        const bool is    = (warp * TURNS + i) * 32 + lane < m && id >= 0 && id < n;
        const uint32_t r = (uint32_t)id / apart;
        place[i]         = is && (uint32_t)id - r * apart == range ? r : kNoRow;
    }
    for (int r = t; r < rows; r += 256)
#pragma unroll
        for (int w = 0; w < 8; ++w)
            counts[w][r] = 0;
    if (t == 0)
        many_count = 0;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
        const uint32_t row = place[i];
        uint32_t alike     = __ballot_sync(0xffffffffu, row != kNoRow);
        if (alike) {
            for (int b = 0; (rows - 1) >> b; ++b) {
                const uint32_t set = __ballot_sync(0xffffffffu, (row >> b) & 1);
                alike &= (row >> b) & 1 ? set : ~set;
            }
            const int ahead = __popc(alike & ((1u << lane) - 1));
            if (row != kNoRow)
                place[i] |= (counts[warp][row] + ahead) << 16;
            __syncwarp();
            if (row != kNoRow && ahead == 0)
                counts[warp][row] += __popc(alike);
            __syncwarp();
        }
    }
    __syncthreads();
    // where each row's tokens begin, and each warp's of it: two rows to a thread
    uint32_t sum[2], upto;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        sum[q] = 0;
        if (2 * t + q < rows) {
            uint32_t c[8];
#pragma unroll
            for (int w = 0; w < 8; ++w)
                c[w] = counts[w][2 * t + q];
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                counts[w][2 * t + q] = sum[q];
                sum[q] += c[w];
            }
        }
    }
    upto = sum[0] + sum[1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
        upto += lane >= o ? v : 0;
    }
    if (lane == 31)
        warp_sums[warp] = upto;
    __syncthreads();
    upto += __reduce_add_sync(0xffffffffu, lane < warp ? warp_sums[lane] : 0);
    begins[2 * t + 1] = upto - sum[1], begins[2 * t + 2] = upto;
    if (t == 0)
        begins[0] = 0;
#pragma unroll
    for (int q = 0; q < 2; ++q)
        if (sum[q] > kAloneTokens)
            many[atomicAdd(&many_count, 1)] = (uint16_t)(2 * t + q); // in any order: each is a row of its own
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TURNS; ++i)
        if (place[i] != kNoRow)
            order[begins[place[i] & 0xffff] + counts[warp][place[i] & 0xffff] + (place[i] >> 16)] = (uint16_t)((warp * TURNS + i) * 32 + lane);
    __syncthreads();
    auto in_strip = [&](int q) { return VEC ? lane * 4 + q : q * 32 + lane; };
    auto add      = [&](uint32_t first, uint32_t last, double (&to)[4]) {
        for (uint32_t i = first; i < last; i += AT_ONCE) {
            float v[AT_ONCE][4];
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u) {
                const float *src = dout + (int64_t)order[min(i + u, last - 1)] * k;
                if (VEC) {
                    const float4 f = *reinterpret_cast<const float4 *>(src + min(c0 + in_strip(0), k - 4));
                    v[u][0] = f.x, v[u][1] = f.y, v[u][2] = f.z, v[u][3] = f.w;
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        v[u][q] = src[min(c0 + in_strip(q), k - 1)];
                }
            }
#pragma unroll
            for (int u = 0; u < AT_ONCE; ++u)
                if (i + u < last)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        to[q] += (double)v[u][q];
        }
    };
    for (int r = warp; r < here; r += 8) {
        const uint32_t first = begins[r], last = begins[r + 1];
        if (last - first > kAloneTokens)
            continue;
        float *to = dtable + (range + (int64_t)r * apart) * k + c0;
        if (first == last) {
            if (VEC) {
                if (c0 + in_strip(0) < k)
                    __stcs(reinterpret_cast<float4 *>(to + in_strip(0)), make_float4(0.0f, 0.0f, 0.0f, 0.0f));
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (c0 + in_strip(q) < k)
                        __stcs(to + in_strip(q), 0.0f);
            }
            continue;
        }
        double all[4] = {};
        add(first, last, all);
        if (VEC) {
            if (c0 + in_strip(0) < k)
                __stcs(reinterpret_cast<float4 *>(to + in_strip(0)),
                       make_float4((float)(all[0] * scale), (float)(all[1] * scale), (float)(all[2] * scale), (float)(all[3] * scale)));
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (c0 + in_strip(q) < k)
                    __stcs(to + in_strip(q), (float)(all[q] * scale));
        }
    }
    for (int i = 0; i < many_count; ++i) {
        const int r          = many[i];
        const uint32_t first = begins[r], count = begins[r + 1] - first;
        double all[4]        = {};
        add(first + count * warp / 8, first + count * (warp + 1) / 8, all);
#pragma unroll
        for (int q = 0; q < 4; ++q)
            part[warp][in_strip(q)] = all[q];
        __syncthreads();
        if (t < 128 && c0 + t < k) {
            double whole = 0.0;
#pragma unroll
            for (int w = 0; w < 8; ++w)
                whole += part[w][t];
            dtable[(range + (int64_t)r * apart) * k + c0 + t] = (float)(whole * scale);
        }
        __syncthreads();
    }
}

constexpr int kSortMemory = ((kSortWarps + 2) * (1 << kSortBits) + 1) * 4;
// Whether a cluster of 16 sorting blocks, an SM to each, can run here: not where a part of the device is all that the process has, or no group of SMs has 16.  With 8
// the gradient of 16384 x 50257 x 2048 takes 116 us instead of 111, 131072 x 50000 x 256 105 instead of 88.
ct_status sort_by_sixteen(const DeviceState *st, bool *possible) {
    static int known[16] = {}; // by device: 1 no, 2 yes.  Under the entry points' lock
    int &mine            = known[st->device & 15];
    if (mine == 0) {
        auto kernel = embedding_sort_kernel<16, 0>;
        CT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortMemory));
        CT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        cudaLaunchAttribute attr{};
        attr.id               = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 16, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(16), cfg.blockDim = dim3(kSortWarps * 32), cfg.dynamicSmemBytes = kSortMemory;
        cfg.attrs = &attr, cfg.numAttrs = 1;
        int clusters = 0;
        if (cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess) {
            cudaGetLastError();
            clusters = 0;
        }
        mine = clusters > 0 && cluster_limit() >= 16 ? 2 : 1;
    }
    *possible = mine == 2;
    return CT_OK;
}

constexpr int64_t kMostTokens = 1 << 29;

ct_status check_embedding(const char *name, int64_t m, int64_t n, int64_t k, double scale) {
    if (m < 0 || n < 0 || k < 0)
        return fail(CT_ERR_INVALID, "%s: negative dimension", name);
    if (m > kMostTokens || n > kMostTokens || k > kMostTokens)
        return fail(CT_ERR_TOO_LARGE, "%s: dimension too large", name);
    if (!(std::fabs((float)scale) <= FLT_MAX))
        return fail(CT_ERR_INVALID, "%s: scale must be finite", name);
    return CT_OK;
}

} // namespace
} // namespace ct

using namespace ct;

extern "C" {

ct_status ct_embedding(const float *table, const int64_t *ids, int64_t m, int64_t n, int64_t k, double scale, float *out) {
    OpLock op_lock;
    DeviceState *st;
    CT_TRY(current(&st));
    CT_TRY(check_embedding("embedding", m, n, k, scale));
    if (m == 0 || k == 0)
        return CT_OK;
    if (!ids || !out || (n > 0 && !table))
        return fail(CT_ERR_INVALID, "embedding: null pointer");
    ProfScope prof("embedding");
    const bool vec = (k & 3) == 0 && aligned16(table) && aligned16(out);
    const int early = lines_apart(out, m * k * 4, table, n * k * 4) && lines_apart(out, m * k * 4, ids, m * 8);
    auto launch     = [&](auto kernel, int tpr) -> ct_status {
        const int64_t pieces = (k + tpr * kLookupValues - 1) / (tpr * kLookupValues), per_block = 256 / tpr;
        const int64_t blocks = std::min<int64_t>((m * pieces + per_block - 1) / per_block, INT32_MAX);
        CT_CUDA(launch_dependent(kernel, dim3((unsigned)blocks), dim3(256), 0, stream(), table, ids, m, n, k, pieces, (float)scale, out, early));
        CT_LAUNCH_CHECK("embedding");
        return CT_OK;
    };
#define CT_LOOKUP(TPR) return vec ? launch(embedding_kernel<TPR, true>, TPR) : launch(embedding_kernel<TPR, false>, TPR)
    // measured (us, 65536 rows of 50000; 4, 8, 16 and 32 threads): 16 columns 8, 10, 12, 18; 64 12, 10, 14, 18; 128 16, 14, 14, 20; 256 23, 21, 21, 23;
    // 512 37, 35, 35, 33; 2048 125, 117, 121, 117
    if (k <= 32)
        CT_LOOKUP(4);
    if (k <= 128)
        CT_LOOKUP(8);
    if (k <= 256)
        CT_LOOKUP(16);
    CT_LOOKUP(32);
#undef CT_LOOKUP
}

ct_status ct_embedding_grad(const int64_t *ids, const float *dout, int64_t m, int64_t n, int64_t k, double scale, float *dtable) {
    OpLock op_lock;
    DeviceState *st;
    CT_TRY(current(&st));
    CT_TRY(check_embedding("embedding_grad", m, n, k, scale));
    if (n == 0 || k == 0)
        return CT_OK;
    if (!dtable || (m > 0 && (!ids || !dout)))
        return fail(CT_ERR_INVALID, "embedding_grad: null pointer");
    if (m == 0) {
        CT_CUDA(cudaMemsetAsync(dtable, 0, (size_t)n * k * 4, stream()));
        return CT_OK;
    }
    ProfScope prof("embedding_grad");
    const bool vec = (k & 3) == 0 && aligned16(dout) && aligned16(dtable);
    // In one launch, where that is sooner than sorting, adding up and joining in three (us in line, three launches and one; tokens x rows x columns):
    // 1000 x 3000 x 1000 22 and 8, 1000 x 50000 x 1000 56 and 37, 8 x 131072 x 768 77 and 65, 1537 x 2050 x 771 21 and 13, 4000 x 4000 x 100 20 and 12,
    // 4000 x 50000 x 300 32 and 26, 4000 x 50000 x 1000 58 and 52; but 8000 x 58000 x 266 39 and 52, 8000 x 20000 x 1000 39 and 52.  Rows of many tokens keep one
    // block busy, for words of a text the first with every second to fifth token of few rows: 2000 x 10 x 2000 18 and 10, 4000 x 10 x 2000 19 and 17 (behind other work
    // 29 and 35), 4000 x 3 x 64 17 and 22, 4000 x 1 x 500 22 and 39
    const int64_t columns = (k + 127) / 128;
    // 4 blocks to an SM run at once; large tables take 12 (us with 4 and 12; 500 x 50000 x 1000 46 and 37, 16 x 32003 x 1024 24 and 23, 1000 x 20000 x 400 13 and 14,
    // 1537 x 2050 x 771 13 and 18)
    const int64_t blocks = st->sm_count * (n * k > 1 << 24 ? 12 : 4);
    const int rows       = (int)std::max<int64_t>(1, std::min<int64_t>(kFewRows, (n * columns + blocks - 1) / blocks));
    const int64_t apart  = (n + rows - 1) / rows;
    if ((m <= 1024 || (m <= 4096 && m <= 256 * n)) && apart * columns <= INT32_MAX) {
        auto few = [&](auto kernel) -> ct_status {
            CT_CUDA(launch_dependent(kernel, dim3((unsigned)(apart * columns)), dim3(256), 0, stream(), ids, dout, (int)m, n, k, rows,
                                     (uint32_t)apart, (int)columns, (float)scale, dtable));
            CT_LAUNCH_CHECK("embedding_grad_few");
            return CT_OK;
        };
        if (m <= 1024)
            return vec ? few(embedding_grad_few_kernel<1024, true>) : few(embedding_grad_few_kernel<1024, false>);
        if (m <= 2048)
            return vec ? few(embedding_grad_few_kernel<2048, true>) : few(embedding_grad_few_kernel<2048, false>);
        return vec ? few(embedding_grad_few_kernel<4096, true>) : few(embedding_grad_few_kernel<4096, false>);
    }
    const int v    = k <= 64 ? 1 : 2; // 16384 x 50000 x 32 33 us by 128 columns, 38 by 256; 64 36 and 39; 128 42 and 40; 256 46 and 44
    const int64_t strips = (k + 128 * v - 1) / (128 * v);
    // Slices: as many as run at once, of 8 items at least; where that is more than 64 items each, four times as many, since their ends come apart
    // (16384 x 50257 x 2048: 149 us with one for each warp that runs, 125 with four);
    // up to twice as many of rows without tokens, which take less time than those with (6913 x 58582 x 266 40 and 34, 8666 x 575 x 2393 41 and 50)
    const int64_t wave = std::max<int64_t>(1, (int64_t)st->sm_count * 16 / strips), items = n + m;
    const int64_t once = std::max<int64_t>(1, std::min(wave, items / 8));
    const int64_t slices = wave == 1           ? 1 // of rows so long, whose partial sums would take more memory than they save time
                           : items >= wave * 64 ? std::min(wave * 4 + 1, items / 64)
                           : n > 2 * m          ? std::max(once, std::min(wave * 2, items / 32))
                                                : once;

    int bits = 1; // of the ids and of n, which stands for none
    while ((n >> bits) > 0)
        ++bits;
    const int passes = (bits + kSortBits - 1) / kSortBits;
    bits             = (bits + passes - 1) / passes;

    auto up              = [](int64_t bytes) { return (bytes + 255) & ~(int64_t)255; };
    const int64_t words  = up(m * 4), partial = up(slices * k * 8);
    Scratch scratch;
    CT_TRY(scratch.get((size_t)(4 * words + 2 * partial + 256 + up(slices) + up(slices * 8))));
    Sorted s;
    for (int i = 0; i < 2; ++i)
        s.ids[i] = scratch.as<uint32_t>(2 * i * words), s.at[i] = scratch.as<uint32_t>((2 * i + 1) * words);
    double *head = scratch.as<double>(4 * words), *tail = scratch.as<double>(4 * words + partial);
    s.counts        = scratch.as<uint32_t>(4 * words + 2 * partial);
    uint2 *across   = scratch.as<uint2>(4 * words + 2 * partial + 256);
    uint8_t *states = scratch.as<uint8_t>(4 * words + 2 * partial + 256 + up(slices * 8));

    bool wide = m > 8 * 1024;
    if (wide)
        CT_TRY(sort_by_sixteen(st, &wide));
    auto sort = [&](auto kernel, int ctas) -> ct_status {
        CT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortMemory));
        CT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        CT_CUDA(launch_dependent_cluster(kernel, ctas, dim3((unsigned)ctas), dim3(kSortWarps * 32), ((size_t)(kSortWarps + 2) * (1 << bits) + 1) * 4, stream(), ids,
                                         (uint32_t)m, (uint32_t)n, passes, bits, s));
        CT_LAUNCH_CHECK("embedding_sort");
        return CT_OK;
    };
    CT_TRY(m <= 8 * 1024    ? sort(embedding_sort_kernel<8, 1>, 8)
           : !wide          ? sort(embedding_sort_kernel<8, 0>, 8)
           : m <= 16 * 1024 ? sort(embedding_sort_kernel<16, 1>, 16)
           : m <= 32 * 1024 ? sort(embedding_sort_kernel<16, 2>, 16)
           : m <= 64 * 1024 ? sort(embedding_sort_kernel<16, 4>, 16)
           : m <= 128 * 1024 ? sort(embedding_sort_kernel<16, 8>, 16)
                             : sort(embedding_sort_kernel<16, 0>, 16));
    const uint32_t *sorted_ids = s.ids[passes & 1], *sorted_at = s.at[passes & 1];
    auto launch = [&](auto kernel) -> ct_status {
        CT_CUDA(launch_dependent(kernel, dim3((unsigned)((slices * strips + 7) / 8)), dim3(256), 0, stream(), sorted_ids, sorted_at, s.counts, dout, (uint32_t)n,
                                 k, (float)scale, (uint32_t)slices, (uint32_t)strips, dtable, head, tail, states, across));
        CT_LAUNCH_CHECK("embedding_grad");
        return CT_OK;
    };
    if (v == 1)
        CT_TRY(vec ? launch(embedding_grad_kernel<1, 8, 3, true>) : launch(embedding_grad_kernel<1, 8, 3, false>));
    else
        CT_TRY(vec ? launch(embedding_grad_kernel<2, 4, 2, true>) : launch(embedding_grad_kernel<2, 4, 2, false>));
    if (slices > 1) {
        CT_CUDA(launch_dependent(embedding_join_kernel, dim3((unsigned)(8 * st->sm_count)), dim3(256), 0, stream(), static_cast<const uint32_t *>(s.counts), k,
                                 (float)scale, (uint32_t)((k + 31) / 32), static_cast<const double *>(head), static_cast<const double *>(tail),
                                 static_cast<const uint8_t *>(states), static_cast<const uint2 *>(across), dtable));
        CT_LAUNCH_CHECK("embedding_join");
    }
    return CT_OK;
}

} // extern "C"
