// Embedding lookup, and the gradient of its table.
//
//   out[i] = scale table[ids[i]];   dtable[v] = scale (sum of dout[i] over the i with ids[i] = v), in the order of i
//
// Both are bound by memory: a lookup reads a row and writes one, the gradient reads dout once and writes every row of the table.
// Gradient: the tokens are sorted by id (stable, so that sums have one order), then warps walk the tokens and the rows together.  Rows
// without a token are as many as there are stores of zeros, rows with thousands as many as there are loads, so what is cut into equal slices is
// the merged list of both: each token, and behind its last token the end of each row.  A row that lies across slices leaves a partial
// sum in each, which a third kernel adds up.  Sums are kept in 64 bits and rounded once.
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
    float *__restrict__ out) {
    griddep_wait();
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
constexpr int kSortWarps = 32, kSortBits = 10, kSortCtas = 8;
struct Sorted {
    uint32_t *ids[2], *at[2]; // two places each: a pass goes from one to the other
    uint32_t *counts;         // [0] tokens with an id of the table; [1] rows across slices (of the kernel behind)
};

__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa(addr, rank)) : "memory");
    return v;
}

__global__ void __launch_bounds__(kSortWarps * 32) embedding_sort_kernel(
    const int64_t *__restrict__ ids, uint32_t m, uint32_t n, int passes, int bits, Sorted s, uint32_t ctas) {
    extern __shared__ uint32_t smem[];
    const int bins   = 1 << bits;
    uint32_t *counts = smem;                      // [warp][bin]
    uint32_t *totals = counts + kSortWarps * bins; // of this CTA, and behind them its tokens without a row
    uint32_t *base   = totals + bins + 1;
    __shared__ uint32_t warp_sums[kSortWarps];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const uint32_t rank = cluster_rank();
    const uint32_t each = ((m + ctas * kSortWarps - 1) / (ctas * kSortWarps) + 31) & ~31u; // tokens of a warp
    const uint64_t lo64 = (uint64_t)(rank * kSortWarps + warp) * each;
    const uint32_t lo = (uint32_t)min(lo64, (uint64_t)m), hi = (uint32_t)min(lo64 + each, (uint64_t)m);
    const uint32_t totals_at = static_cast<uint32_t>(__cvta_generic_to_shared(totals));
    griddep_wait();
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * bits, from = pass & 1, to = from ^ 1;
        auto id_of      = [&](uint32_t i) -> uint32_t {
            if (pass)
                return __ldcg(s.ids[from] + i);
            const int64_t id = ids[i];
            return id >= 0 && id < (int64_t)n ? (uint32_t)id : n;
        };
        for (int i = t; i < kSortWarps * bins; i += kSortWarps * 32)
            counts[i] = 0;
        if (t == 0)
            totals[bins] = 0;
        __syncthreads();
        uint32_t none = 0;
#pragma unroll 4
        for (uint32_t i = lo + lane; i < hi; i += 32) {
            const uint32_t id = id_of(i);
            none += id == n;
            atomicAdd(&counts[warp * bins + ((id >> shift) & (bins - 1))], 1u);
        }
        if (none)
            atomicAdd(&totals[bins], none);
        __syncthreads();
        for (int d = t; d < bins; d += kSortWarps * 32) {
            uint32_t sum = 0;
#pragma unroll
            for (int w = 0; w < kSortWarps; ++w) {
                const uint32_t c      = counts[w * bins + d];
                counts[w * bins + d]  = sum;
                sum                  += c;
            }
            totals[d] = sum;
        }
        cluster_sync();
        uint32_t before = 0, all = 0; // of this thread's digit (bins <= threads)
        if (t < bins)
            for (uint32_t r = 0; r < ctas; ++r) {
                const uint32_t c = ld_cluster_u32(totals_at + t * 4, r);
                before += r < rank ? c : 0;
                all += c;
            }
        uint32_t upto = all; // over digits, this one included
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
            upto += lane >= o ? v : 0;
        }
        if (lane == 31)
            warp_sums[warp] = upto;
        if (pass == 0 && rank == 0 && t == 0) {
            uint32_t without = 0;
            for (uint32_t r = 0; r < ctas; ++r)
                without += ld_cluster_u32(totals_at + bins * 4, r);
            s.counts[0] = m - without;
            s.counts[1] = 0;
        }
        __syncthreads();
        uint32_t digits = 0;
        for (int w = 0; w < warp; ++w)
            digits += warp_sums[w];
        if (t < bins)
            base[t] = digits + upto - all + before;
        __syncthreads();
        for (uint32_t i0 = lo; i0 < hi; i0 += 32) {
            const uint32_t i  = i0 + lane;
            const bool here   = i < hi;
            const uint32_t id = here ? id_of(i) : 0, at = here ? (pass ? __ldcg(s.at[from] + i) : i) : 0;
            const uint32_t d     = here ? (id >> shift) & (bins - 1) : 0xffffffffu;
            const uint32_t alike = __match_any_sync(0xffffffffu, d);
            const uint32_t ahead = __popc(alike & ((1u << lane) - 1));
            uint32_t *count      = &counts[warp * bins + (here ? d : 0)];
            const uint32_t place = here ? base[d] + *count + ahead : 0;
            __syncwarp();
            if (here && ahead == 0)
                *count += __popc(alike);
            __syncwarp();
            if (here) {
                s.ids[to][place] = id;
                s.at[to][place]  = at;
            }
        }
        cluster_sync(); // the next pass reads what the others wrote; their totals have been read
    }
}

// ---- sums ---------------------------------------------------------------------------------------

// How many tokens stand among the first d of the merged list: token i is number i + ids[i] of it.
__device__ __forceinline__ uint32_t tokens_before(const uint32_t *__restrict__ ids, uint32_t tokens, uint32_t n, uint64_t d, int lane) {
    uint32_t lo = d > n ? (uint32_t)(d - n) : 0, hi = (uint32_t)min(d, (uint64_t)tokens);
    while (lo < hi) {
        const uint32_t step = (hi - lo + 31) / 32, i = lo + lane * step;
        const bool is_before = i < hi && (uint64_t)i + __ldcg(ids + i) < d;
        const int before     = __popc(__ballot_sync(0xffffffffu, is_before));
        if (before == 0)
            break;
        hi = min(hi, lo + before * step);
        lo = lo + (before - 1) * step + 1;
    }
    return lo;
}

enum SliceState : uint8_t { SLICE_THROUGH = 1 }; // all of it belongs to a row that began before and ends behind

// A warp to a slice and 128 V columns.
template <int V, bool VEC>
__global__ void __launch_bounds__(256) embedding_grad_kernel(
    const uint32_t *__restrict__ ids, const uint32_t *__restrict__ at, uint32_t *__restrict__ counts, const float *__restrict__ dout, uint32_t n,
    int64_t k, float scale, uint32_t slices, uint32_t strips, float *__restrict__ dtable, double *__restrict__ head, double *__restrict__ tail,
    uint8_t *__restrict__ states, uint32_t *__restrict__ across) {
    griddep_wait();
    const int lane       = threadIdx.x & 31;
    const uint64_t unit  = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const uint32_t slice = (uint32_t)(unit / strips), strip = (uint32_t)(unit - (uint64_t)slice * strips);
    if (slice >= slices)
        return;
    const int64_t c0 = (int64_t)strip * 128 * V;
    auto column      = [&](int j, int q) -> int64_t { return c0 + (VEC ? (j * 32 + lane) * 4 + q : (j * 4 + q) * 32 + lane); };
    const uint32_t tokens = __ldcg(counts);
    const uint64_t total  = (uint64_t)n + tokens;
    const uint64_t each   = (total + slices - 1) / slices;
    const uint64_t d0 = min((uint64_t)slice * each, total), d1 = min(d0 + each, total);
    const uint32_t i0 = tokens_before(ids, tokens, n, d0, lane), i1 = tokens_before(ids, tokens, n, d1, lane);
    const uint32_t r0 = (uint32_t)(d0 - i0), r1 = (uint32_t)(d1 - i1);
    const bool goes_on = d0 < d1 && i0 > 0 && __ldcg(ids + i0 - 1) == r0; // row r0 has tokens in slices before
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
        if (row == r0 && goes_on) {
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
    uint32_t row = r0;
    constexpr int kAtOnce = 4;
    for (uint32_t i = i0; i < i1; i += 32) {
        const uint32_t mine = i + lane < i1 ? __ldcg(ids + i + lane) : 0, mine_at = i + lane < i1 ? __ldcg(at + i + lane) : 0;
        const int count = min(32u, i1 - i);
        for (int g = 0; g < count; g += kAtOnce) {
            float v[kAtOnce][4 * V];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const float *src = dout + (int64_t)__shfl_sync(0xffffffffu, mine_at, (g + u) & 31) * k;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    if (VEC) {
                        float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                        if (g + u < count && column(j, 0) < k)
                            f = __ldcs(reinterpret_cast<const float4 *>(src + column(j, 0)));
                        v[u][4 * j] = f.x, v[u][4 * j + 1] = f.y, v[u][4 * j + 2] = f.z, v[u][4 * j + 3] = f.w;
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            v[u][4 * j + q] = g + u < count && column(j, q) < k ? __ldcs(src + column(j, q)) : 0.0f;
                    }
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
                const uint32_t id = __shfl_sync(0xffffffffu, mine, (g + u) & 31);
                if (g + u < count) {
                    for (; row < id; ++row)
                        finish(row);
#pragma unroll
                    for (int j = 0; j < 4 * V; ++j)
                        sum[j] += (double)v[u][j];
                }
            }
        }
    }
    for (; row < r1; ++row)
        finish(row);
    const bool through = goes_on && r0 == r1;
    if (through || (i1 > i0 && __ldcg(ids + i1 - 1) == r1)) // row r1 ends in a later slice
        leave(tail);
    if (strip == 0 && lane == 0) {
        states[slice] = through ? SLICE_THROUGH : 0;
        if (goes_on && r0 < r1)
            across[atomicAdd(counts + 1, 1u)] = slice; // in any order: each is a row of its own
    }
}

// The rows that lie across slices: what each slice left of it, the last one's first.  A block has 32 columns of a row, and eight parts of its slices.
__global__ void __launch_bounds__(256) embedding_join_kernel(
    const uint32_t *__restrict__ ids, const uint32_t *__restrict__ counts, uint32_t n, int64_t k, float scale, uint32_t slices, uint32_t column_blocks,
    const double *__restrict__ head, const double *__restrict__ tail, const uint8_t *__restrict__ states, const uint32_t *__restrict__ across,
    float *__restrict__ dtable) {
    __shared__ double part[8][32];
    griddep_wait();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t tokens = __ldcg(counts);
    const uint64_t total = (uint64_t)n + tokens, each = (total + slices - 1) / slices, units = (uint64_t)__ldcg(counts + 1) * column_blocks;
    for (uint64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const uint32_t slice = __ldcg(across + u / column_blocks);
        const int64_t c      = (int64_t)(u % column_blocks) * 32 + lane;
        const uint64_t d     = (uint64_t)slice * each;
        const uint32_t row   = (uint32_t)(d - tokens_before(ids, tokens, n, d, lane));
        uint32_t first       = slice - 1; // the slice in which the row begins, 32 of them looked at together
        for (;;) {
            const bool through     = lane <= first && (__ldcg(states + first - lane) & SLICE_THROUGH);
            const uint32_t beyond = __ballot_sync(0xffffffffu, !through);
            if (beyond) {
                first -= __ffs(beyond) - 1;
                break;
            }
            first -= 32;
        }
        double sum = 0.0;
        if (c < k)
            for (uint32_t s = first + warp; s < slice; s += 8)
                sum += __ldcg(tail + (int64_t)s * k + c);
        part[warp][lane] = sum;
        __syncthreads();
        if (warp == 0 && c < k) {
            sum = __ldcg(head + (int64_t)slice * k + c);
#pragma unroll
            for (int w = 0; w < 8; ++w)
                sum += part[w][lane];
            dtable[(int64_t)row * k + c] = (float)(sum * scale);
        }
        __syncthreads();
    }
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
    auto launch    = [&](auto kernel, int tpr) -> ct_status {
        const int64_t pieces = (k + tpr * kLookupValues - 1) / (tpr * kLookupValues), per_block = 256 / tpr;
        const int64_t blocks = std::min<int64_t>((m * pieces + per_block - 1) / per_block, INT32_MAX);
        CT_CUDA(launch_dependent(kernel, dim3((unsigned)blocks), dim3(256), 0, stream(), table, ids, m, n, k, pieces, (float)scale, out));
        CT_LAUNCH_CHECK("embedding");
        return CT_OK;
    };
#define CT_LOOKUP(TPR) return vec ? launch(embedding_kernel<TPR, true>, TPR) : launch(embedding_kernel<TPR, false>, TPR)
    if (k <= 4 * kLookupValues)
        CT_LOOKUP(4);
    if (k <= 16 * kLookupValues)
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
    const int v    = k <= 128 ? 1 : 2;
    const int64_t strips = (k + 128 * v - 1) / (128 * v);
    const int64_t slices = std::max<int64_t>(1, std::min<int64_t>((int64_t)st->sm_count * 32 / strips, (n + m + 7) / 8));

    int bits = 1; // of the ids and of n, which stands for none
    while ((n >> bits) > 0)
        ++bits;
    const int passes = (bits + kSortBits - 1) / kSortBits;
    bits             = (bits + passes - 1) / passes;
    int ctas         = 1;
    while (ctas < kSortCtas && m > (int64_t)ctas * kSortWarps * 32)
        ctas *= 2;

    auto up              = [](int64_t bytes) { return (bytes + 255) & ~(int64_t)255; };
    const int64_t words  = up(m * 4), partial = up(slices * k * 8);
    Scratch scratch;
    CT_TRY(scratch.get((size_t)(4 * words + 2 * partial + 256 + up(slices) + up(slices * 4))));
    Sorted s;
    for (int i = 0; i < 2; ++i)
        s.ids[i] = scratch.as<uint32_t>(2 * i * words), s.at[i] = scratch.as<uint32_t>((2 * i + 1) * words);
    double *head = scratch.as<double>(4 * words), *tail = scratch.as<double>(4 * words + partial);
    s.counts        = scratch.as<uint32_t>(4 * words + 2 * partial);
    uint32_t *across = scratch.as<uint32_t>(4 * words + 2 * partial + 256);
    uint8_t *states  = scratch.as<uint8_t>(4 * words + 2 * partial + 256 + up(slices * 4));

    const size_t smem = ((size_t)(kSortWarps + 2) * (1 << bits) + 1) * 4;
    CT_CUDA(cudaFuncSetAttribute(embedding_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, ((kSortWarps + 2) * (1 << kSortBits) + 1) * 4));
    CT_CUDA(launch_dependent_cluster(embedding_sort_kernel, ctas, dim3((unsigned)ctas), dim3(kSortWarps * 32), smem, stream(), ids, (uint32_t)m, (uint32_t)n,
                                     passes, bits, s, (uint32_t)ctas));
    CT_LAUNCH_CHECK("embedding_sort");
    const uint32_t *sorted_ids = s.ids[passes & 1], *sorted_at = s.at[passes & 1];
    auto launch = [&](auto kernel) -> ct_status {
        CT_CUDA(launch_dependent(kernel, dim3((unsigned)((slices * strips + 7) / 8)), dim3(256), 0, stream(), sorted_ids, sorted_at, s.counts, dout, (uint32_t)n,
                                 k, (float)scale, (uint32_t)slices, (uint32_t)strips, dtable, head, tail, states, across));
        CT_LAUNCH_CHECK("embedding_grad");
        return CT_OK;
    };
    if (v == 1)
        CT_TRY(vec ? launch(embedding_grad_kernel<1, true>) : launch(embedding_grad_kernel<1, false>));
    else
        CT_TRY(vec ? launch(embedding_grad_kernel<2, true>) : launch(embedding_grad_kernel<2, false>));
    if (slices > 1) {
        CT_CUDA(launch_dependent(embedding_join_kernel, dim3((unsigned)(2 * st->sm_count)), dim3(256), 0, stream(), sorted_ids,
                                 static_cast<const uint32_t *>(s.counts), (uint32_t)n, k, (float)scale, (uint32_t)slices, (uint32_t)((k + 31) / 32),
                                 static_cast<const double *>(head), static_cast<const double *>(tail), static_cast<const uint8_t *>(states),
                                 static_cast<const uint32_t *>(across), dtable));
        CT_LAUNCH_CHECK("embedding_join");
    }
    return CT_OK;
}

} // extern "C"
