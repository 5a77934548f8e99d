// Layer norm over the rows of a matrix, and its gradient.
//
//   mean = sum(x) / C,  var = sum((x - mean)^2) / C,  r = 1 / sqrt(var + eps),  h = (x - mean) r,  y = h gamma + beta
//   g = dy gamma,  dx = r (g - mean(g) - h mean(g h)),  dgamma = sum over rows of dy h,  dbeta = sum over rows of dy
//
// Both are bound by memory (8 and 12 bytes a value) if a row is read once, so a row stays in the registers of the threads that
// share it from the load to the store: a warp for short rows, a block for longer ones.  Only rows of more than 16384 values (8192 on the
// way back) are read again, three times in all and four.
//
// Sums along a row are float32, of at most 64 values before they meet in a tree (beyond 65536 columns: in 64 bits first).  Sums over rows are
// float32 over at most kChainRows rows of a thread (kChainRowsLong above 8192 columns) and the up to 32 rows that a block has at a time, then 64 bits.  The
// mean is taken twice: the sums of d = x - m and of d^2, about the first mean m, come from one exchange, and what d leaves of a mean corrects
// m and the variance.  Rows whose mean is large beside their spread keep the digits that float32 has of x - mean.
// The gradient takes them again from x, which it has in registers anyway, instead of reading them: one exchange more per row,
// no statistics to keep.
#include "common.cuh"

#include <algorithm>

namespace ct {
namespace {

// Values of a row that a thread of TPR holds, in groups of four: group j is columns 4 (j TPR + t) .. of aligned rows (VEC), and
// of others columns (4 j + q) TPR + t, which neighbours read together at any alignment.
template <int TPR, int V, bool VEC> struct Row {
    __device__ static __forceinline__ int64_t column(int t, int j, int q) {
        return VEC ? (int64_t)(j * TPR + t) * 4 + q : (int64_t)(j * 4 + q) * TPR + t;
    }
    __device__ static __forceinline__ void load(float (&v)[4 * V], const float *__restrict__ src, int64_t cols, int t) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (VEC) {
                float4 f = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (column(t, j, 0) < cols)
                    f = *reinterpret_cast<const float4 *>(src + column(t, j, 0));
                v[4 * j] = f.x, v[4 * j + 1] = f.y, v[4 * j + 2] = f.z, v[4 * j + 3] = f.w;
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    v[4 * j + q] = column(t, j, q) < cols ? src[column(t, j, q)] : 0.0f;
            }
    }
    __device__ static __forceinline__ void store(float *__restrict__ dst, const float (&v)[4 * V], int64_t cols, int t) {
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (VEC) {
                if (column(t, j, 0) < cols)
                    __stcs(reinterpret_cast<float4 *>(dst + column(t, j, 0)), make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
            } else {
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    if (column(t, j, q) < cols)
                        __stcs(dst + column(t, j, q), v[4 * j + q]);
            }
    }
};

// The sums of N values over the TPR threads of a row; all threads of the block call it.  Two calls in turn need words of their own: a
// warp that is through the second call's barrier has seen every warp through the first.
template <int TPR, int N> __device__ __forceinline__ void row_sums(float (&s)[N], float (&words)[N][32]) {
#pragma unroll
    for (int o = (TPR < 32 ? TPR : 32) / 2; o; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i)
            s[i] = __fadd_rn(s[i], __shfl_xor_sync(0xffffffffu, s[i], o));
    if (TPR > 32) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < N; ++i)
                words[i][warp] = s[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s[i] = lane < TPR / 32 ? words[i][lane] : 0.0f;
#pragma unroll
            for (int o = TPR / 64; o; o >>= 1)
                s[i] = __fadd_rn(s[i], __shfl_xor_sync(0xffffffffu, s[i], o));
            if (TPR < 1024)
                s[i] = __shfl_sync(0xffffffffu, s[i], 0);
        }
    }
}

// The sums of N float32 terms over a thread's columns first, first + 1024, ...: add(c, s) puts the terms of column c into s.  CHAINED: they meet
// 64 bits every 64 columns; 1000 x 100000 takes 307 us so, 291 in one chain, 1 x 100000 45 and 43.
constexpr int64_t kChainColumns = 64 * 1024; // of a row, where one chain has 64 values
template <bool CHAINED, int N, typename F> __device__ __forceinline__ void column_sums(float (&sums)[N], int64_t first, int64_t last, F &&add) {
    float s[N] = {};
    int64_t c  = first;
    if (CHAINED) {
        double all[N] = {};
        while (last - c > kChainColumns) {
#pragma unroll 8
            for (int q = 0; q < 64; ++q, c += 1024)
                add(c, s);
#pragma unroll
            for (int j = 0; j < N; ++j)
                all[j] += (double)s[j], s[j] = 0.0f;
        }
        for (; c < last; c += 1024)
            add(c, s);
#pragma unroll
        for (int j = 0; j < N; ++j)
            s[j] = (float)(all[j] + (double)s[j]);
    } else {
        for (; c < last; c += 1024)
            add(c, s);
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
        sums[j] = s[j];
}

// 1 / sqrt(var + eps) from the sums of d and d^2, and what d lacks of the mean.
__device__ __forceinline__ float spread(float sum_d, float sum_dd, float inv_cols, float eps, float &rest) {
    rest            = __fmul_rn(sum_d, inv_cols);
    const float var = __fsub_rn(__fmul_rn(sum_dd, inv_cols), __fmul_rn(rest, rest));
    return __fdiv_rn(1.0f, __fsqrt_rn(__fadd_rn(var < 0.0f ? 0.0f : var, eps)));
}

template <int TPR> constexpr int kBlock = TPR <= 32 ? 256 : TPR; // several rows, or one

// early: whether the next kernel may be launched meanwhile.  Not in place: a block's loads bring what lies beside its rows into the SM's first-level
// cache, which the next kernel would find there as it was.

template <int TPR, int V, bool VEC>
__global__ void __launch_bounds__(kBlock<TPR>) layer_norm_kernel(
    const float *__restrict__ x, const float *__restrict__ gamma, const float *__restrict__ beta, int64_t rows, int64_t cols, float eps,
    float *__restrict__ out, int early) {
    using R = Row<TPR, V, VEC>;
    __shared__ float words1[1][32], words2[2][32];
    griddep_wait();
    if (early)
        griddep_launch_dependents();
    const int t       = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (kBlock<TPR> / TPR) + threadIdx.x / TPR;
    const int64_t mine = row < rows ? cols : 0; // a warp's last rows may not be there
    if (TPR == 32 && row >= rows)
        return;
    const float inv_cols = __fdiv_rn(1.0f, (float)cols);
    float v[4 * V];
    R::load(v, x + row * cols, mine, t);
    float sum[1] = {0.0f};
#pragma unroll
    for (int i = 0; i < 4 * V; ++i)
        sum[0] = __fadd_rn(sum[0], v[i]);
    row_sums<TPR>(sum, words1);
    const float mean = __fmul_rn(sum[0], inv_cols);
    float s[2]       = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < V; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const float d = R::column(t, j, q) < cols ? __fsub_rn(v[4 * j + q], mean) : 0.0f;
            v[4 * j + q]  = d;
            s[0]          = __fadd_rn(s[0], d);
            s[1]          = __fmaf_rn(d, d, s[1]);
        }
    row_sums<TPR>(s, words2);
    float rest;
    const float r = spread(s[0], s[1], inv_cols, eps, rest);
    float g[4 * V], b[4 * V];
    if (gamma)
        R::load(g, gamma, cols, t);
    if (beta)
        R::load(b, beta, cols, t);
#pragma unroll
    for (int i = 0; i < 4 * V; ++i) {
        float y = __fmul_rn(__fsub_rn(v[i], rest), r);
        if (gamma)
            y = __fmul_rn(y, g[i]);
        if (beta)
            y = __fadd_rn(y, b[i]);
        v[i] = y;
    }
    R::store(out + row * cols, v, mine, t);
}

// Rows of any length, a block to a row, which is read three times.
template <bool CHAINED>
__global__ void __launch_bounds__(1024) layer_norm_long_kernel(
    const float *__restrict__ x, const float *__restrict__ gamma, const float *__restrict__ beta, int64_t cols, float eps, float *__restrict__ out,
    int early) {
    __shared__ float words1[1][32], words2[2][32];
    griddep_wait();
    if (early)
        griddep_launch_dependents();
    const float *src     = x + (int64_t)blockIdx.x * cols;
    const float inv_cols = __fdiv_rn(1.0f, (float)cols);
    float sum[1];
    column_sums<CHAINED>(sum, threadIdx.x, cols, [&](int64_t c, float (&s)[1]) { s[0] = __fadd_rn(s[0], src[c]); });
    row_sums<1024>(sum, words1);
    const float mean = __fmul_rn(sum[0], inv_cols);
    float s[2];
    column_sums<CHAINED>(s, threadIdx.x, cols, [&](int64_t c, float (&s)[2]) {
        const float d = __fsub_rn(src[c], mean);
        s[0]          = __fadd_rn(s[0], d);
        s[1]          = __fmaf_rn(d, d, s[1]);
    });
    row_sums<1024>(s, words2);
    float rest;
    const float r = spread(s[0], s[1], inv_cols, eps, rest);
    for (int64_t c = threadIdx.x; c < cols; c += 1024) {
        float y = __fmul_rn(__fsub_rn(__fsub_rn(src[c], mean), rest), r);
        if (gamma)
            y = __fmul_rn(y, gamma[c]);
        if (beta)
            y = __fadd_rn(y, beta[c]);
        out[(int64_t)blockIdx.x * cols + c] = y;
    }
}

// A row on its way to shared memory, column c at slot + 4 c: aligned rows 16 bytes at a time, each thread what it will read (only its own
// copies are waited for); other rows of an aligned matrix as the 16-byte pieces that they touch, from slot - 4 skew on, where skew is the row's
// distance from a 16-byte boundary; else value by value, which is four times the instructions (60000 x 785: 161 us).
template <int TPR, int V, bool VEC>
__device__ __forceinline__ void row_copy(uint32_t slot, const float *__restrict__ src, int64_t cols, int skew, bool pieces, int t) {
    using R = Row<TPR, V, VEC>;
    if (VEC) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int64_t c = R::column(t, j, 0);
            const int bytes = c < cols ? 16 : 0; // none: zeros, and nothing is read
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(slot + (int)c * 4), "l"(src + (bytes ? c : 0)), "r"(bytes) : "memory");
        }
    } else if (pieces) {
        const int end = skew + (int)cols;
        for (int c = 4 * t; c < end; c += 4 * TPR) {
            const int bytes = end - c < 4 ? (end - c) * 4 : 16; // not past the last row's end
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(slot + (c - skew) * 4), "l"(src + (c - skew)), "r"(bytes) : "memory");
        }
    } else {
        for (int c = t; c < (int)cols; c += TPR)
            asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(slot + c * 4), "l"(src + c) : "memory");
    }
}
// A thread's values of it; columns that the row does not have are zero (VEC: in the slot as well).
template <int TPR, int V, bool VEC> __device__ __forceinline__ void row_read(float (&v)[4 * V], const float *slot, int64_t cols, int t) {
    using R = Row<TPR, V, VEC>;
#pragma unroll
    for (int j = 0; j < V; ++j)
        if (VEC) {
            const float4 f = *reinterpret_cast<const float4 *>(slot + R::column(t, j, 0));
            v[4 * j] = f.x, v[4 * j + 1] = f.y, v[4 * j + 2] = f.z, v[4 * j + 3] = f.w;
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                v[4 * j + q] = R::column(t, j, q) < cols ? slot[R::column(t, j, q)] : 0.0f;
        }
}
template <int TPR> __device__ __forceinline__ void row_sync() {
    if (TPR <= 32)
        __syncwarp();
    else
        __syncthreads();
}

// The gradient.  A block (of one row at a time, or a row per warp) walks rows; a thread has the same columns of each, and keeps their sums
// over its rows, which go to partial[block][2][cols] (dgamma, dbeta) for norm_columns_kernel.  Between a row's loads and its stores stand two
// exchanges, so the next two rows are on their way meanwhile: with the loads of a row issued when it was its turn, 16384 x 4096 took 177 us
// and 60000 x 785 208.
constexpr int kAhead = 3; // rows in shared memory, the one at work among them
// Rows of a thread whose sums are one float32 chain: with more rows there are more blocks, as many turns of the machine as it takes.
constexpr int64_t kChainRows = 256, kChainRowsLong = 64; // up to 8192 columns, and beyond
// Values of a slot: a row, with what lies before and behind it in its 16-byte pieces.  Slots begin on 128-byte boundaries: 16 bytes off, 2048
// aligned columns took 165 us for 140.
template <int TPR, int V, bool VEC> constexpr int kSlot = 4 * V * TPR + (VEC ? 0 : 32);
template <int TPR, int V, bool VEC> constexpr int kGradSmem = (kAhead * 2 * kSlot<TPR, V, VEC> * (kBlock<TPR> / TPR) + 4 * V * TPR) * 4;
template <int TPR, int V, bool VEC>
__global__ void __launch_bounds__(kBlock<TPR>) layer_norm_grad_kernel(
    const float *__restrict__ x, const float *__restrict__ gamma, const float *__restrict__ dout, int64_t rows, int64_t cols, float eps,
    float *__restrict__ dx, float *__restrict__ partial, int pieces, int early) {
    using R               = Row<TPR, V, VEC>;
    constexpr int THREADS = kBlock<TPR>, RPB = THREADS / TPR, SLOT = kSlot<TPR, V, VEC>;
    extern __shared__ __align__(128) float smem[];
    __shared__ float words1[1][32], words2[4][32];
    griddep_wait();
    if (early)
        griddep_launch_dependents();
    const int t = threadIdx.x % TPR, group = threadIdx.x / TPR;
    float *ring    = smem + group * kAhead * 2 * SLOT; // [row][x, dout], column 0 up to three values behind the beginning
    float *gamma_s = smem + RPB * kAhead * 2 * SLOT;
    const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
    const int64_t step = (int64_t)gridDim.x * RPB, row0 = (int64_t)blockIdx.x * RPB + group;
    auto skew_of = [&](int64_t row) { return VEC || !pieces ? 0 : (int)((row * cols) & 3); };
    auto fetch   = [&](int64_t row, int at) {
        if (row < rows) {
            const int skew = skew_of(row);
            row_copy<TPR, V, VEC>(ring_at + (at * 2 * SLOT + skew) * 4, x + row * cols, cols, skew, pieces != 0, t);
            row_copy<TPR, V, VEC>(ring_at + ((at * 2 + 1) * SLOT + skew) * 4, dout + row * cols, cols, skew, pieces != 0, t);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < kAhead - 1; ++i)
        fetch(row0 + i * step, i);
    for (int c = threadIdx.x; c < 4 * V * TPR; c += THREADS)
        gamma_s[c] = c < cols ? (gamma ? gamma[c] : 1.0f) : 0.0f;
    __syncthreads();
    const float inv_cols = __fdiv_rn(1.0f, (float)cols);
    float sum_g[4 * V], sum_b[4 * V];
#pragma unroll
    for (int i = 0; i < 4 * V; ++i)
        sum_g[i] = sum_b[i] = 0.0f;
    int at = 0;
    const int64_t warp_row = TPR < 32 ? (int64_t)blockIdx.x * RPB + (threadIdx.x >> 5) * (32 / (TPR < 32 ? TPR : 32)) : row0; // the warp's first
    for (int64_t row = row0; row - row0 + warp_row < rows; row += step) { // whole warps, or the whole block
        if (!VEC && TPR <= 32)
            __syncwarp(); // the slot's last row has been read (a block's exchanges come behind its reads)
        fetch(row + (kAhead - 1) * step, at == 0 ? kAhead - 1 : at - 1);
        asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
        if (!VEC)
            row_sync<TPR>(); // the others' copies
        float v[4 * V], dy[4 * V];
        row_read<TPR, V, VEC>(v, ring + at * 2 * SLOT + skew_of(row), cols, t);
        row_read<TPR, V, VEC>(dy, ring + (at * 2 + 1) * SLOT + skew_of(row), cols, t);
        const bool here = TPR >= 32 || row < rows; // a warp's last rows may not be: what their slots hold is not used
        if (!here)
#pragma unroll
            for (int i = 0; i < 4 * V; ++i)
                v[i] = dy[i] = 0.0f;
        at = at == kAhead - 1 ? 0 : at + 1;
        float sum[1] = {0.0f};
#pragma unroll
        for (int i = 0; i < 4 * V; ++i)
            sum[0] = __fadd_rn(sum[0], v[i]);
        row_sums<TPR>(sum, words1);
        const float mean = __fmul_rn(sum[0], inv_cols);
        float s[4]       = {0.0f, 0.0f, 0.0f, 0.0f}; // of d, d^2, g, g d
        float g[4 * V];
        row_read<TPR, V, VEC>(g, gamma_s, cols, t);
#pragma unroll
        for (int j = 0; j < V; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int i   = 4 * j + q;
                const float d = R::column(t, j, q) < cols ? __fsub_rn(v[i], mean) : 0.0f;
                g[i]          = __fmul_rn(dy[i], g[i]);
                v[i]          = d;
                s[0]          = __fadd_rn(s[0], d);
                s[1]          = __fmaf_rn(d, d, s[1]);
                s[2]          = __fadd_rn(s[2], g[i]);
                s[3]          = __fmaf_rn(g[i], d, s[3]);
            }
        row_sums<TPR>(s, words2);
        float rest;
        const float r  = spread(s[0], s[1], inv_cols, eps, rest);
        const float mg = __fmul_rn(s[2], inv_cols);                                                            // mean of g
        const float mh = __fmul_rn(__fmul_rn(__fsub_rn(s[3], __fmul_rn(rest, s[2])), r), inv_cols); // mean of g h
#pragma unroll
        for (int i = 0; i < 4 * V; ++i) {
            const float h = here ? __fmul_rn(__fsub_rn(v[i], rest), r) : 0.0f;
            sum_g[i]      = __fmaf_rn(dy[i], h, sum_g[i]);
            sum_b[i]      = __fadd_rn(sum_b[i], dy[i]);
            v[i]          = __fmul_rn(r, __fsub_rn(__fsub_rn(g[i], mg), __fmul_rn(h, mh)));
        }
        if (dx && here)
            R::store(dx + row * cols, v, cols, t);
    }
    if (!partial)
        return;
    float *mine = partial + (int64_t)blockIdx.x * 2 * cols;
    if (RPB > 1) { // the warps' sums, one after the other
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncthreads(); // no row is at work any more
        float *sums = smem; // [2][4 V TPR]
        for (int who = 0; who < RPB; ++who) {
            if (group == who)
#pragma unroll
                for (int i = 0; i < 4 * V; ++i) {
                    const int64_t c = R::column(t, i >> 2, i & 3);
                    sums[c]               = who ? __fadd_rn(sums[c], sum_g[i]) : sum_g[i];
                    sums[4 * V * TPR + c] = who ? __fadd_rn(sums[4 * V * TPR + c], sum_b[i]) : sum_b[i];
                }
            __syncthreads();
        }
        for (int64_t c = threadIdx.x; c < cols; c += THREADS)
            mine[c] = sums[c], mine[cols + c] = sums[4 * V * TPR + c];
    } else {
        R::store(mine, sum_g, cols, t);
        R::store(mine + cols, sum_b, cols, t); // VEC: cols is a multiple of four, aligned like the first half
    }
}

// Longer rows: the statistics and dx, a block to a row, then the columns' sums from both matrices again.
template <bool CHAINED>
__global__ void __launch_bounds__(1024) layer_norm_grad_long_kernel(
    const float *__restrict__ x, const float *__restrict__ gamma, const float *__restrict__ dout, int64_t cols, float eps, float *__restrict__ dx,
    float2 *__restrict__ stats, int early) {
    __shared__ float words1[1][32], words2[4][32];
    griddep_wait();
    if (early)
        griddep_launch_dependents();
    const int64_t row    = blockIdx.x;
    const float *src     = x + row * cols, *dy = dout + row * cols;
    const float inv_cols = __fdiv_rn(1.0f, (float)cols);
    float sum[1];
    column_sums<CHAINED>(sum, threadIdx.x, cols, [&](int64_t c, float (&s)[1]) { s[0] = __fadd_rn(s[0], src[c]); });
    row_sums<1024>(sum, words1);
    const float mean = __fmul_rn(sum[0], inv_cols);
    float s[4];
    column_sums<CHAINED>(s, threadIdx.x, cols, [&](int64_t c, float (&s)[4]) {
        const float d = __fsub_rn(src[c], mean), g = gamma ? __fmul_rn(dy[c], gamma[c]) : dy[c];
        s[0] = __fadd_rn(s[0], d);
        s[1] = __fmaf_rn(d, d, s[1]);
        s[2] = __fadd_rn(s[2], g);
        s[3] = __fmaf_rn(g, d, s[3]);
    });
    row_sums<1024>(s, words2);
    float rest;
    const float r  = spread(s[0], s[1], inv_cols, eps, rest);
    const float mg = __fmul_rn(s[2], inv_cols);
    const float mh = __fmul_rn(__fmul_rn(__fsub_rn(s[3], __fmul_rn(rest, s[2])), r), inv_cols);
    if (stats && threadIdx.x == 0) // two numbers: their sum would be rounded to float32
        stats[2 * row] = make_float2(mean, rest), stats[2 * row + 1] = make_float2(r, 0.0f);
    if (dx)
        for (int64_t c = threadIdx.x; c < cols; c += 1024) {
            const float g = gamma ? __fmul_rn(dy[c], gamma[c]) : dy[c];
            const float h = __fmul_rn(__fsub_rn(__fsub_rn(src[c], mean), rest), r);
            dx[row * cols + c] = __fmul_rn(r, __fsub_rn(__fsub_rn(g, mg), __fmul_rn(h, mh)));
        }
}

__global__ void __launch_bounds__(256) layer_norm_grad_long_columns_kernel(
    const float *__restrict__ x, const float *__restrict__ dout, const float2 *__restrict__ stats, int64_t rows, int64_t cols, int64_t rows_each,
    float *__restrict__ partial) {
    griddep_wait();
    griddep_launch_dependents();
    const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (c >= cols)
        return;
    const int64_t r1 = min(rows, ((int64_t)blockIdx.y + 1) * rows_each);
    float sum_g = 0.0f, sum_b = 0.0f;
    for (int64_t r = (int64_t)blockIdx.y * rows_each; r < r1; ++r) {
        const float2 m = stats[2 * r], q = stats[2 * r + 1];
        const float dy = dout[r * cols + c];
        sum_g = __fmaf_rn(dy, __fmul_rn(__fsub_rn(__fsub_rn(x[r * cols + c], m.x), m.y), q.x), sum_g);
        sum_b = __fadd_rn(sum_b, dy);
    }
    partial[(int64_t)blockIdx.y * 2 * cols + c]        = sum_g;
    partial[((int64_t)blockIdx.y * 2 + 1) * cols + c] = sum_b;
}

// out0[c] = sum over `parts` of partial[part][c], out1[c] of partial[part][cols + c]: 32 columns to a block, a warp takes every eighth part.
__global__ void __launch_bounds__(256) norm_columns_kernel(
    const float *__restrict__ partial, int parts, int64_t cols, float *__restrict__ out0, float *__restrict__ out1) {
    __shared__ double sums[8][32];
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    double s        = 0.0;
    if (c < 2 * cols)
#pragma unroll 8
        for (int p = warp; p < parts; p += 8)
            s += (double)partial[(int64_t)p * 2 * cols + c];
    sums[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c < 2 * cols) {
#pragma unroll
        for (int w = 1; w < 8; ++w)
            s += sums[w][lane];
        float *out = c < cols ? out0 : out1;
        if (out)
            out[c < cols ? c : c - cols] = (float)s;
    }
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <int TPR, int V>
ct_status launch_norm(const float *x, const float *gamma, const float *beta, int64_t rows, int64_t cols, float eps, float *out, bool vec) {
    constexpr int RPB   = kBlock<TPR> / TPR;
    const dim3 grid((unsigned)((rows + RPB - 1) / RPB));
    if (vec)
        CT_CUDA(launch_dependent(layer_norm_kernel<TPR, V, true>, grid, dim3(kBlock<TPR>), 0, stream(), x, gamma, beta, rows, cols, eps, out, out != x));
    else
        CT_CUDA(launch_dependent(layer_norm_kernel<TPR, V, false>, grid, dim3(kBlock<TPR>), 0, stream(), x, gamma, beta, rows, cols, eps, out, out != x));
    CT_LAUNCH_CHECK("layer_norm");
    return CT_OK;
}

template <int TPR, int V, bool VEC>
ct_status launch_norm_grad(
    const DeviceState *st, const float *x, const float *gamma, const float *dout, int64_t rows, int64_t cols, float eps, float *dx, bool sums, Scratch &partial,
    int64_t *blocks) {
    constexpr int SMEM = kGradSmem<TPR, V, VEC>, RPB = kBlock<TPR> / TPR;
    auto kernel        = layer_norm_grad_kernel<TPR, V, VEC>;
    static int resident[16] = {}; // blocks to an SM, per device; under the entry points' lock
    int &fit                = resident[st->device & 15];
    if (fit == 0) {
        CT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM));
        CT_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&fit, kernel, kBlock<TPR>, SMEM));
        fit = std::max(fit, 1);
    }
    *blocks = blocks_for((rows + RPB - 1) / RPB, (int64_t)st->sm_count * fit, kChainRows);
    if (sums)
        CT_TRY(partial.get((size_t)*blocks * 8 * cols));
    CT_CUDA(launch_dependent(kernel, dim3((unsigned)*blocks), dim3(kBlock<TPR>), SMEM, stream(), x, gamma, dout, rows, cols, eps, dx,
                             sums ? partial.as<float>() : nullptr, aligned16(x) && aligned16(dout) ? 1 : 0, dx != x && dx != dout));
    CT_LAUNCH_CHECK("layer_norm_grad");
    return CT_OK;
}

ct_status check_norm(const char *name, const void *x, const void *second, int64_t rows, int64_t cols, double eps) {
    if (rows < 0 || cols < 0)
        return fail(CT_ERR_INVALID, "%s: negative dimension", name);
    if (!(eps >= 0.0))
        return fail(CT_ERR_INVALID, "%s: eps must not be negative", name);
    if (rows > 1 << 29 || cols > 1 << 29)
        return fail(CT_ERR_TOO_LARGE, "%s: dimension too large", name);
    if (rows > 0 && cols > 0 && (!x || !second))
        return fail(CT_ERR_INVALID, "%s: null pointer", name);
    return CT_OK;
}

} // namespace
} // namespace ct

using namespace ct;

extern "C" {

ct_status ct_layer_norm(
    const float *x, const float *gamma, const float *beta, int64_t rows, int64_t cols, double eps, float *out) {
    OpLock op_lock;
    DeviceState *st;
    CT_TRY(current(&st));
    CT_TRY(check_norm("layer_norm", x, out, rows, cols, eps));
    if (rows == 0 || cols == 0)
        return CT_OK;
    ProfScope prof("layer_norm");
    const bool vec = (cols & 3) == 0 && aligned16(x) && aligned16(out) && (!gamma || aligned16(gamma)) && (!beta || aligned16(beta));
    const float e  = (float)eps;
    // Threads to a row and float4 to a thread, measured (us; 200 calls in line, or many rows with L2 flushed):
    //   512 columns: a warp 1.7, 256 threads 1.9 (1 row), 2.1 and 2.3 (500), 18 and 37 (16384)
    //   1024: a warp 2.9, 256 threads 2.0 (16 rows), 3.0 and 2.5 (500), 31 and 41 (16384); 768: 2.6 and 2.0 (16 rows), 2.8 and 2.4 (500)
    //   785: 7 float4 88, 8 94 (60000 rows); 896: 84 and 86; 640: 6 float4 59, 7 75
    //   2048: 128 threads 2.0, 256 2.1, 1024 2.4 (1 row), 2.9, 3.0, 6.1 (500), 49, 53, 155 (16384)
    //   4095: 128 threads 57, 256 68, 1024 107 (8000 rows); 4096: 2.4, 2.4, 2.6 (1 row), 51, 52, 88 (8000)
    //   8192: 256 threads 3.1, 512 3.1, 1024 3.4 (1 row), 7.5, 7.7, 9.7 (500), 58, 59, 66 (4000)
    //   16384: in registers 8, read three times 12 (50 rows), 105 and 104 (3000); 24576: 16 and 14 (50), 125 and 84 (1500)
#define CT_NORM(TPR, V) launch_norm<TPR, V>(x, gamma, beta, rows, cols, e, out, vec)
    if (cols <= 32)
        return CT_NORM(8, 1);
    if (cols <= 64)
        return CT_NORM(8, 2);
    if (cols <= 128)
        return CT_NORM(16, 2);
    if (cols <= 256)
        return CT_NORM(32, 2);
    if (cols <= 512)
        return CT_NORM(32, 4);
    if (cols <= 1024 && rows < st->sm_count * 4)
        return CT_NORM(256, 1);
    if (cols <= 768)
        return CT_NORM(32, 6);
    if (cols <= 896)
        return CT_NORM(32, 7);
    if (cols <= 1024)
        return CT_NORM(32, 8);
    if (cols <= 2048)
        return CT_NORM(128, 4);
    if (cols <= 4096)
        return CT_NORM(128, 8);
    if (cols <= 8192)
        return CT_NORM(256, 8);
    if (cols <= 16384)
        return CT_NORM(1024, 4);
#undef CT_NORM
    auto kernel = cols <= kChainColumns ? layer_norm_long_kernel<false> : layer_norm_long_kernel<true>;
    CT_CUDA(launch_dependent(kernel, dim3((unsigned)rows), dim3(1024), 0, stream(), x, gamma, beta, cols, e, out, out != x));
    CT_LAUNCH_CHECK("layer_norm_long");
    return CT_OK;
}

ct_status ct_layer_norm_grad(
    const float *x, const float *gamma, const float *dout, int64_t rows, int64_t cols, double eps, float *dx, float *dgamma, float *dbeta) {
    OpLock op_lock;
    DeviceState *st;
    CT_TRY(current(&st));
    CT_TRY(check_norm("layer_norm_grad", x, dout, rows, cols, eps));
    if (cols == 0)
        return CT_OK;
    if (rows == 0) { // sums of nothing
        if (dgamma)
            CT_CUDA(cudaMemsetAsync(dgamma, 0, (size_t)cols * 4, stream()));
        if (dbeta)
            CT_CUDA(cudaMemsetAsync(dbeta, 0, (size_t)cols * 4, stream()));
        return CT_OK;
    }
    ProfScope prof("layer_norm_grad");
    const float e   = (float)eps;
    const bool sums = dgamma || dbeta;
    Scratch scratch;
    int64_t parts = 0;
    if (cols <= 8192) {
        const bool vec = (cols & 3) == 0 && aligned16(x) && aligned16(dout) && (!dx || aligned16(dx)) && (!gamma || aligned16(gamma));
        // measured (us, L2 flushed): 512 columns a warp 31, 256 threads 62 (16384 rows), 17 and 21 (1000), 15 and 15 (300); 1024: 51 and 64 (16384
        // rows), 22 and 24 (1300), 19 and 17 (300); 785: 7 float4 to a lane 127, 8 138 (60000 rows), 896: 125 and 123; 640: 6 88, 7 97; 2048: 256
        // threads 86, 512 113 (16384 rows); 4096: 256 threads 80, 512 88 (8000 rows); 8192: 512 threads 88, 1024 92 (4000 rows)
#define CT_NORM_GRAD(TPR, V)                                                                                                      \
    CT_TRY(vec ? (launch_norm_grad<TPR, V, true>(st, x, gamma, dout, rows, cols, e, dx, sums, scratch, &parts))                  \
               : (launch_norm_grad<TPR, V, false>(st, x, gamma, dout, rows, cols, e, dx, sums, scratch, &parts)))
        if (cols <= 32)
            CT_NORM_GRAD(8, 1);
        else if (cols <= 64)
            CT_NORM_GRAD(8, 2);
        else if (cols <= 128)
            CT_NORM_GRAD(16, 2);
        else if (cols <= 256)
            CT_NORM_GRAD(32, 2);
        else if (cols <= 512)
            CT_NORM_GRAD(32, 4);
        else if (cols <= 768 && rows >= st->sm_count * 8)
            CT_NORM_GRAD(32, 6);
        else if (cols <= 896 && rows >= st->sm_count * 8)
            CT_NORM_GRAD(32, 7);
        else if (cols <= 1024 && rows >= st->sm_count * 8)
            CT_NORM_GRAD(32, 8);
        else if (cols <= 1024)
            CT_NORM_GRAD(256, 1);
        else if (cols <= 2048)
            CT_NORM_GRAD(256, 2);
        else if (cols <= 4096)
            CT_NORM_GRAD(256, 4);
        else
            CT_NORM_GRAD(512, 4);
#undef CT_NORM_GRAD
    } else {
        const int64_t strips = (cols + 255) / 256;
        // parts for eight blocks to an SM, of 8 rows at least and kChainRowsLong at most, or as many as a grid has
        const int64_t fill = (rows * strips + st->sm_count * 8 - 1) / (st->sm_count * 8);
        const int64_t each = std::max(std::min(std::max<int64_t>(8, fill), kChainRowsLong), (rows + 65534) / 65535);
        parts              = (rows + each - 1) / each;
        const size_t stats_bytes = ((size_t)rows * 16 + 255) & ~(size_t)255;
        if (sums)
            CT_TRY(scratch.get(stats_bytes + (size_t)parts * 8 * cols));
        float2 *stats  = sums ? scratch.as<float2>() : nullptr;
        float *partial = sums ? scratch.as<float>(stats_bytes) : nullptr;
        auto rows_pass = [&](float *dx_to, float2 *stats_to) -> ct_status {
            auto kernel = cols <= kChainColumns ? layer_norm_grad_long_kernel<false> : layer_norm_grad_long_kernel<true>;
            CT_CUDA(launch_dependent(kernel, dim3((unsigned)rows), dim3(1024), 0, stream(), x, gamma, dout, cols, e, dx_to, stats_to, dx_to != x && dx_to != dout));
            CT_LAUNCH_CHECK("layer_norm_grad_long");
            return CT_OK;
        };
        // dx in the place of x or dout, which the columns' sums read: it is written behind them, by a second pass
        const bool behind = sums && (dx == x || dx == dout);
        CT_TRY(rows_pass(behind ? nullptr : dx, stats));
        if (sums) {
            CT_CUDA(launch_dependent(layer_norm_grad_long_columns_kernel, dim3((unsigned)strips, (unsigned)parts), dim3(256), 0, stream(), x, dout,
                                     static_cast<const float2 *>(stats), rows, cols, each, partial));
            CT_LAUNCH_CHECK("layer_norm_grad_long_columns");
            CT_CUDA(launch_dependent(norm_columns_kernel, dim3((unsigned)((2 * cols + 31) / 32)), dim3(256), 0, stream(),
                                     static_cast<const float *>(partial), (int)parts, cols, dgamma, dbeta));
            CT_LAUNCH_CHECK("norm_columns");
        }
        if (behind)
            CT_TRY(rows_pass(dx, nullptr));
        return CT_OK;
    }
    if (sums) {
        CT_CUDA(launch_dependent(norm_columns_kernel, dim3((unsigned)((2 * cols + 31) / 32)), dim3(256), 0, stream(),
                                 scratch.as<const float>(), (int)parts, cols, dgamma, dbeta));
        CT_LAUNCH_CHECK("norm_columns");
    }
    return CT_OK;
}

} // extern "C"
