// Operand planes of the fused products (fused_product.cuh), and the product that is simply stored.
//
// The pre-passes are bound by memory: 4 bytes read and 4 written a value.  A scale is found and used while its line is in registers: rows of up to
// 8192 values, a warp or a block to each, and columns of up to 1024, a block to 16 of them.  Longer lines are read twice, the second
// time from L2 where that holds them; rows of up to 65536 by clusters, once.  All operands of a product whose columns are short are split in one launch.
#include "fused_product.cuh"

namespace ct {
namespace fused {
namespace {

// Two matrices side by side, the second from column ld on; zeros between cols and ld.
struct Source {
    const float *in, *in2, *col_factor;
    int64_t rows, cols, ld;
    int vec; // rows of both are whole and aligned float4
    __device__ __forceinline__ float4 quad(int64_t r, int64_t c) const {
        float4 q = plain_quad(r, c);
        if (col_factor) { // of columns that there are
            const float4 f = *reinterpret_cast<const float4 *>(col_factor + c);
            q.x = q.x != 0.0f ? q.x * f.x : 0.0f, q.y = q.y != 0.0f ? q.y * f.y : 0.0f;
            q.z = q.z != 0.0f ? q.z * f.z : 0.0f, q.w = q.w != 0.0f ? q.w * f.w : 0.0f;
        }
        return q;
    }
    // Columns c .. c + 3, c a multiple of four.  Rows that are not aligned take a load for each: as aligned pieces, with what a lane lacks shuffled over
    // from the next one, columns of 1024 x 32003 took 160 us for 85, the selects and shuffles outweighing the loads.
    __device__ __forceinline__ float4 plain_quad(int64_t r, int64_t c) const {
        const float *src = in;
        if (c >= ld)
            src = in2, c -= ld;
        src += r * cols + c;
        if (vec && c + 3 < cols)
            return *reinterpret_cast<const float4 *>(src);
        float4 q;
        q.x = c < cols ? src[0] : 0.0f;
        q.y = c + 1 < cols ? src[1] : 0.0f;
        q.z = c + 2 < cols ? src[2] : 0.0f;
        q.w = c + 3 < cols ? src[3] : 0.0f;
        return q;
    }
};

__device__ __forceinline__ uint32_t quad_bits(const float4 &q) {
    return max(max(finite_bits(q.x), finite_bits(q.y)), max(finite_bits(q.z), finite_bits(q.w)));
}
__device__ __forceinline__ void put_quad(const Planes &to, int64_t at, float a, float b, float c, float d) {
    __half2 hi[2], lo[2];
    split2(a, b, hi[0], lo[0]);
    split2(c, d, hi[1], lo[1]);
    *reinterpret_cast<uint2 *>(to.hi + at) = *reinterpret_cast<uint2 *>(hi);
    *reinterpret_cast<uint2 *>(to.lo + at) = *reinterpret_cast<uint2 *>(lo);
}

__device__ __forceinline__ float4 factored(float4 q, const float *row_factor, int64_t r) {
    if (row_factor) {
        const float f = row_factor[r];
        q = __float_as_uint(f) == kNoPart ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : make_float4(q.x * f, q.y * f, q.z * f, q.w * f);
    }
    return q;
}

// TPR threads to a row, which they hold in V float4 each if it is that short.
template <int TPR, int V>
__device__ __forceinline__ void split_rows(const Source &src, int64_t width, const Planes &to, float *inverse, int64_t block, uint32_t (&words)[8]) {
    const int t       = threadIdx.x % TPR;
    const int64_t row = block * (256 / TPR) + threadIdx.x / TPR;
    if (row >= src.rows) // whole warps, or the whole block
        return;
    const bool fits = width <= TPR * V * 4;
    float4 v[V];
    uint32_t mx = 0;
    if (fits) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int64_t c = (int64_t)(j * TPR + t) * 4;
            v[j]            = c < width ? src.quad(row, c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (int j = 0; j < V; ++j)
            mx = max(mx, quad_bits(v[j]));
    } else {
#pragma unroll 8
        for (int64_t c = t * 4; c < width; c += TPR * 4)
            mx = max(mx, quad_bits(src.quad(row, c)));
    }
    mx = __reduce_max_sync(0xffffffffu, mx);
    if (TPR > 32) {
        if ((threadIdx.x & 31) == 0)
            words[threadIdx.x >> 5] = mx;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; ++w)
            mx = max(mx, words[w]);
    }
    const float s = line_scale(mx);
    if (fits) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int64_t c = (int64_t)(j * TPR + t) * 4;
            if (c < width)
                put_quad(to, row * to.ld + c, v[j].x * s, v[j].y * s, v[j].z * s, v[j].w * s);
        }
    } else {
#pragma unroll 8
        for (int64_t c = t * 4; c < width; c += TPR * 4) {
            const float4 q = src.quad(row, c);
            put_quad(to, row * to.ld + c, q.x * s, q.y * s, q.z * s, q.w * s);
        }
    }
    if (t == 0)
        inverse[row] = line_inverse(mx);
}

// 16 columns to the block, four lanes to a row; at most kShort rows of 64 to a thread.
constexpr int kShort = 16;
// Values that split_small_kernel takes: gated 1024 x 1024 x 500 (2.1 M) 32 us so, 33 by two launches, 1500 x 600 x 300 (1.3 M) 27 and 29, 1024 x 1024 x
// 1000 (3.1 M) 39 and 36, but both products' operands of a gradient of 2^21 21 and 14.
constexpr int64_t kFewValues = 1 << 20;
__device__ __forceinline__ void split_short_cols(
    const Source &src, int64_t width, const float *row_factor, const Planes &to, float *inverse, int64_t block, uint32_t (&words)[8][16]) {
    constexpr int L = 4, RP = 256 / L;
    const int t = threadIdx.x, quad = t % L;
    const int64_t c = block * (4 * L) + quad * 4;
    float4 v[kShort];
    uint32_t mx[4] = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < kShort; ++i) {
        const int64_t r = i * RP + t / L;
        v[i]            = r < src.rows && c < width ? src.quad(r, c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
#pragma unroll
    for (int i = 0; i < kShort; ++i) {
        const int64_t r = i * RP + t / L;
        if (row_factor && r < src.rows)
            v[i] = factored(v[i], row_factor, r);
        mx[0] = max(mx[0], finite_bits(v[i].x)), mx[1] = max(mx[1], finite_bits(v[i].y));
        mx[2] = max(mx[2], finite_bits(v[i].z)), mx[3] = max(mx[3], finite_bits(v[i].w));
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
        for (int o = 16; o >= L; o >>= 1)
            mx[q] = max(mx[q], __shfl_xor_sync(0xffffffffu, mx[q], o));
    if ((t & 31) < L)
#pragma unroll
        for (int q = 0; q < 4; ++q)
            words[t >> 5][quad * 4 + q] = mx[q];
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        mx[q] = words[0][quad * 4 + q];
#pragma unroll
        for (int w = 1; w < 8; ++w)
            mx[q] = max(mx[q], words[w][quad * 4 + q]);
    }
    if (c >= width)
        return;
    const float s0 = line_scale(mx[0]), s1 = line_scale(mx[1]), s2 = line_scale(mx[2]), s3 = line_scale(mx[3]);
#pragma unroll
    for (int i = 0; i < kShort; ++i) {
        const int64_t r = i * RP + t / L;
        if (r < src.rows)
            put_quad(to, r * to.ld + c, v[i].x * s0, v[i].y * s1, v[i].z * s2, v[i].w * s3);
    }
    if (t < L)
        *reinterpret_cast<float4 *>(inverse + c) = make_float4(line_inverse(mx[0]), line_inverse(mx[1]), line_inverse(mx[2]), line_inverse(mx[3]));
}

// Up to four matrices, each with its range of blocks.
enum Form : int { kRowsWarp, kCols16, kCols4 };
struct SplitJobs {
    struct Job {
        Source src;
        int64_t width;
        const float *row_factor;
        Planes to;
        float *inverse;
        int form;
        int64_t first; // block
    } job[6];
    int count;
};
__global__ void __launch_bounds__(256, 2) split_short_cols_kernel(const __grid_constant__ SplitJobs jobs) {
    __shared__ uint32_t many[8][16];
    griddep_wait();
    griddep_launch_dependents();
    int j = 0;
    while (j + 1 < jobs.count && (int64_t)blockIdx.x >= jobs.job[j + 1].first)
        ++j;
    const SplitJobs::Job &x = jobs.job[j];
    split_short_cols(x.src, x.width, x.row_factor, x.to, x.inverse, blockIdx.x - x.first, many);
}

// All of a small product's operands: a warp to a row, a block to 16 columns (4 of more than 256 rows, whose turns would take longer than the
// launch: 1569 x 247 23 us), read twice (the second time from L1).  In registers as above
// they are read once, but the code is ten times as long, and fetching it is what a launch of a few blocks then waits for (8 to 10 against
// 18 to 24 us with cold caches).
__global__ void __launch_bounds__(256) split_small_kernel(const __grid_constant__ SplitJobs jobs) {
    __shared__ uint32_t many[8][16];
    griddep_wait();
    griddep_launch_dependents();
    int j = 0;
    while (j + 1 < jobs.count && (int64_t)blockIdx.x >= jobs.job[j + 1].first)
        ++j;
    const SplitJobs::Job &x = jobs.job[j];
    const Source &src       = x.src;
    const int64_t block     = blockIdx.x - x.first;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (x.form == kRowsWarp) {
        const int64_t row = block * 8 + warp;
        if (row >= src.rows)
            return;
        uint32_t mx = 0;
#pragma unroll 4
        for (int64_t c = lane * 4; c < x.width; c += 128)
            mx = max(mx, quad_bits(src.quad(row, c)));
        mx            = __reduce_max_sync(0xffffffffu, mx);
        const float s = line_scale(mx);
#pragma unroll 4
        for (int64_t c = lane * 4; c < x.width; c += 128) {
            const float4 q = src.quad(row, c);
            put_quad(x.to, row * x.to.ld + c, q.x * s, q.y * s, q.z * s, q.w * s);
        }
        if (lane == 0)
            x.inverse[row] = line_inverse(mx);
    } else {
        const int t = threadIdx.x, lanes = x.form == kCols16 ? 4 : 1, quad = t & (lanes - 1), step = 256 / lanes, first = t / lanes;
        const int64_t c = (block * lanes + quad) * 4;
        uint32_t mx[4] = {0, 0, 0, 0};
        if (c < x.width)
#pragma unroll 4
            for (int64_t r = first; r < src.rows; r += step) {
                const float4 q = factored(src.quad(r, c), x.row_factor, r);
                mx[0] = max(mx[0], finite_bits(q.x)), mx[1] = max(mx[1], finite_bits(q.y));
                mx[2] = max(mx[2], finite_bits(q.z)), mx[3] = max(mx[3], finite_bits(q.w));
            }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            for (int o = 16; o >= lanes; o >>= 1)
                mx[q] = max(mx[q], __shfl_xor_sync(0xffffffffu, mx[q], o));
            if (lane < lanes)
                many[warp][quad * 4 + q] = mx[q];
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int w = 0; w < 8; ++w)
                mx[q] = max(mx[q], many[w][quad * 4 + q]);
        if (c >= x.width)
            return;
        const float s0 = line_scale(mx[0]), s1 = line_scale(mx[1]), s2 = line_scale(mx[2]), s3 = line_scale(mx[3]);
#pragma unroll 4
        for (int64_t r = first; r < src.rows; r += step) {
            const float4 q = factored(src.quad(r, c), x.row_factor, r);
            put_quad(x.to, r * x.to.ld + c, q.x * s0, q.y * s1, q.z * s2, q.w * s3);
        }
        if (t < lanes)
            *reinterpret_cast<float4 *>(x.inverse + c) = make_float4(line_inverse(mx[0]), line_inverse(mx[1]), line_inverse(mx[2]), line_inverse(mx[3]));
    }
}
template <int TPR, int V>
__global__ void __launch_bounds__(256) split_rows_kernel(const Source src, int64_t width, const Planes to, float *__restrict__ inverse) {
    __shared__ uint32_t words[8];
    griddep_wait();
    griddep_launch_dependents();
    split_rows<TPR, V>(src, width, to, inverse, blockIdx.x, words);
}

// Longer rows, a cluster of CTAs to each, 8192 values to a CTA.  Read twice, as rows beyond that are, 1024 x 50257 took 183 us: all rows are under
// way at once, and L2 does not hold them.
constexpr int kLongQuads = 8;
__global__ void __launch_bounds__(256) split_long_rows_kernel(
    const Source src, int64_t width, int ranks, int64_t each, const Planes to, float *__restrict__ inverse) {
    __shared__ uint32_t words[8], most;
    griddep_wait();
    griddep_launch_dependents();
    const int t = threadIdx.x, rank = (int)(blockIdx.x % ranks);
    const int64_t row = blockIdx.x / ranks, first = rank * each, last = min(width, first + each);
    float4 v[kLongQuads];
    uint32_t mx = 0;
#pragma unroll
    for (int j = 0; j < kLongQuads; ++j) {
        const int64_t c = first + (int64_t)(j * 256 + t) * 4;
        v[j]            = c < last ? src.quad(row, c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
#pragma unroll
    for (int j = 0; j < kLongQuads; ++j)
        mx = max(mx, quad_bits(v[j]));
    mx = __reduce_max_sync(0xffffffffu, mx);
    if ((t & 31) == 0)
        words[t >> 5] = mx;
    __syncthreads();
    if (t == 0) {
        for (int w = 0; w < 8; ++w)
            mx = max(mx, words[w]);
        most = mx;
    }
    ptx::cluster_sync();
    for (int q = 0; q < ranks; ++q) {
        uint32_t other;
        asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(other) : "r"(ptx::mapa(ptx::smem_u32(&most), (uint32_t)q)) : "memory");
        mx = max(mx, other);
    }
    const float s = line_scale(mx);
#pragma unroll
    for (int j = 0; j < kLongQuads; ++j) {
        const int64_t c = first + (int64_t)(j * 256 + t) * 4;
        if (c < last)
            put_quad(to, row * to.ld + c, v[j].x * s, v[j].y * s, v[j].z * s, v[j].w * s);
    }
    if (t == 0 && rank == 0)
        inverse[row] = line_inverse(mx);
    ptx::cluster_sync(); // a CTA's word stays until the others have read it
}

// Largest finite magnitude of each column into col_max (zeroed before): a lane has four columns, the block's warps the rows in turn.
__global__ void __launch_bounds__(256) col_max_kernel(
    const Source src, int64_t width, const float *__restrict__ row_factor, int64_t rows_each, uint32_t *__restrict__ col_max) {
    __shared__ uint32_t max_s[8][128];
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 128 + lane * 4;
    const int64_t r0 = (int64_t)blockIdx.y * rows_each, r1 = min(src.rows, r0 + rows_each);
    uint32_t mx[4] = {0, 0, 0, 0};
    if (!src.vec) { // the order is all the same to a maximum: neighbours
        const float *in[4];
        bool here[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int64_t at = (int64_t)blockIdx.x * 128 + lane + 32 * i;
            in[i]      = at >= src.ld ? src.in2 : src.in;
            at -= at >= src.ld ? src.ld : 0;
            here[i] = in[i] && at < src.cols;
            in[i] += at;
        }
#pragma unroll 8
        for (int64_t r = r0 + warp; r < r1; r += 8) {
            float4 q = make_float4(here[0] ? in[0][r * src.cols] : 0.0f, here[1] ? in[1][r * src.cols] : 0.0f, here[2] ? in[2][r * src.cols] : 0.0f,
                                   here[3] ? in[3][r * src.cols] : 0.0f);
            q = factored(q, row_factor, r);
            mx[0] = max(mx[0], finite_bits(q.x)), mx[1] = max(mx[1], finite_bits(q.y));
            mx[2] = max(mx[2], finite_bits(q.z)), mx[3] = max(mx[3], finite_bits(q.w));
        }
    } else if (c < width) {
#pragma unroll 8
        for (int64_t r = r0 + warp; r < r1; r += 8) {
            const float4 q = factored(src.quad(r, c), row_factor, r);
            mx[0] = max(mx[0], finite_bits(q.x)), mx[1] = max(mx[1], finite_bits(q.y));
            mx[2] = max(mx[2], finite_bits(q.z)), mx[3] = max(mx[3], finite_bits(q.w));
        }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q)
        max_s[warp][src.vec ? lane * 4 + q : lane + 32 * q] = mx[q];
    __syncthreads();
    const int64_t mine = (int64_t)blockIdx.x * 128 + threadIdx.x;
    if (threadIdx.x < 128 && mine < width) {
        uint32_t all = max_s[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < 8; ++w)
            all = max(all, max_s[w][threadIdx.x]);
        if (all)
            atomicMax(col_max + mine, all); // the same whatever the order
    }
}

__global__ void __launch_bounds__(256) split_cols_kernel(
    const Source src, int64_t width, const float *__restrict__ row_factor, int64_t rows_each, const uint32_t *__restrict__ col_max, const Planes to,
    float *__restrict__ inverse) {
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 128 + lane * 4;
    if (c >= width)
        return;
    const int64_t r0 = (int64_t)blockIdx.y * rows_each, r1 = min(src.rows, r0 + rows_each);
    const uint4 mx = *reinterpret_cast<const uint4 *>(col_max + c);
    const float s0 = line_scale(mx.x), s1 = line_scale(mx.y), s2 = line_scale(mx.z), s3 = line_scale(mx.w);
    if (blockIdx.y == 0 && warp == 0)
        *reinterpret_cast<float4 *>(inverse + c) = make_float4(line_inverse(mx.x), line_inverse(mx.y), line_inverse(mx.z), line_inverse(mx.w));
#pragma unroll 4
    for (int64_t r = r0 + warp; r < r1; r += 8) {
        const float4 q = factored(src.quad(r, c), row_factor, r);
        put_quad(to, r * to.ld + c, q.x * s0, q.y * s1, q.z * s2, q.w * s3);
    }
}

// out = the slices' sums, in order (and what out held); columns from `second` (a multiple of eight) on to out2.  The slices' rows are whole float4,
// what out's may not be: with a division for each value and one value to a thread 8192 x 2048 of two slices took 66 us, so 29.
struct Joins {
    struct Job {
        const float *partial;
        int slices, shift; // 2^shift threads to a row
        int64_t m, n, pitch, strips, first; // blocks: strips to each turn of the rows; the first block
        float *out, *out2;
        int64_t cols, stride, second;
        int vec, add;
    } job[2];
    int64_t blocks; // of both
    int count;
};
__global__ void __launch_bounds__(256) join_slices_kernel(const __grid_constant__ Joins joins, const uint32_t *__restrict__ flags) {
    griddep_wait();
    griddep_launch_dependents();
    if (*reinterpret_cast<const volatile uint32_t *>(flags + FLAG_TIMEOUT) != 0) // the slices were not computed
        return;
    const int which     = joins.count > 1 && (int64_t)blockIdx.x >= joins.job[1].first ? 1 : 0;
    const Joins::Job &x = joins.job[which];
    const int64_t block = blockIdx.x - x.first, turns = ((which + 1 < joins.count ? joins.job[1].first : joins.blocks) - x.first) / x.strips;
    const int64_t total = x.m * x.pitch, c0 = ((block % x.strips << x.shift) + (threadIdx.x & ((1 << x.shift) - 1))) * 4;
    if (c0 >= x.n)
        return;
    const int rows = 256 >> x.shift; // at a time
    for (int64_t r = block / x.strips * rows + (threadIdx.x >> x.shift); r < x.m; r += turns * rows) {
        const float *src = x.partial + r * x.pitch + c0;
        float4 s         = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
        for (int z = 0; z < x.slices; ++z) {
            const float4 q = __ldcs(reinterpret_cast<const float4 *>(src + z * total));
            s = make_float4(__fadd_rn(s.x, q.x), __fadd_rn(s.y, q.y), __fadd_rn(s.z, q.z), __fadd_rn(s.w, q.w));
        }
        int64_t c = c0;
        float *to = x.out;
        if (x.out2 && c >= x.second)
            to = x.out2, c -= x.second;
        to += r * x.stride + c;
        if (x.vec && c + 3 < x.cols) {
            if (x.add) {
                const float4 o = *reinterpret_cast<const float4 *>(to);
                s = make_float4(__fadd_rn(o.x, s.x), __fadd_rn(o.y, s.y), __fadd_rn(o.z, s.z), __fadd_rn(o.w, s.w));
            }
            *reinterpret_cast<float4 *>(to) = s;
        } else {
            const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (c + q < x.cols)
                    to[q] = x.add ? __fadd_rn(to[q], v[q]) : v[q];
        }
    }
}

Source source_of(const float *in, const float *in2, int64_t rows, int64_t cols, const float *col_factor = nullptr) {
    const bool vec = (cols & 3) == 0 && (reinterpret_cast<uintptr_t>(in) & 15u) == 0 && (reinterpret_cast<uintptr_t>(in2) & 15u) == 0;
    return Source{in, in2, col_factor, rows, cols, padded(cols), vec ? 1 : 0};
}

// A K-major and an MN-major product over the same machine.
__global__ void __launch_bounds__(kThreads, 1) two_products_kernel(
    const __grid_constant__ Maps maps, const __grid_constant__ Product p, const __grid_constant__ Store::Params e, const __grid_constant__ Maps maps_mn,
    const __grid_constant__ Product p_mn, const __grid_constant__ Store::Params e_mn, int longer, int turns) {
    product_body<Store, 128, 1, false, false>(
        maps, p, e, maps_mn, p_mn, e_mn,
        TilesOfTwo{(int)blockIdx.x, (int)gridDim.x, longer, longer ? p_mn.total : p.total, longer ? p.total : p_mn.total, turns});
}

} // namespace

// Long columns: their maxima, then the planes.
static ct_status split_long_cols(DeviceState *st, const Split &x) {
    const Source src     = source_of(x.in, x.in2, x.rows, x.cols);
    const int64_t width  = x.in2 ? 2 * src.ld : src.ld;
    const int64_t strips = (width + 127) / 128;
    // a few blocks to an SM, of at least 32 rows
    const int64_t slices = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>((x.rows + 31) / 32, 65535), (int64_t)st->sm_count * 6 / strips));
    const int64_t each   = (x.rows + slices - 1) / slices;
    const dim3 grid((unsigned)strips, (unsigned)((x.rows + each - 1) / each));
    Scratch words;
    CT_TRY(words.get((size_t)width * 4));
    uint32_t *col_max = words.as<uint32_t>();
    CT_CUDA(cudaMemsetAsync(col_max, 0, (size_t)width * 4, stream()));
    CT_CUDA(launch_dependent(col_max_kernel, grid, dim3(256), 0, stream(), src, width, x.row_factor, each, col_max));
    CT_LAUNCH_CHECK("col_max");
    CT_CUDA(launch_dependent(split_cols_kernel, grid, dim3(256), 0, stream(), src, width, x.row_factor, each, (const uint32_t *)col_max, x.to, x.inverse));
    CT_LAUNCH_CHECK("split_cols");
    return CT_OK;
}

ct_status split(DeviceState *st, const Split *what, int count) {
    auto blocks_of = [](int form, int64_t rows, int64_t width) {
        return form == kRowsWarp ? (rows + 7) / 8 : form == kCols16 ? (width + 15) / 16 : (width + 3) / 4;
    };
    auto add = [&](SplitJobs &jobs, int64_t &blocks, const Split &x, const float *in, const float *in2, int64_t at, int form) {
        const Source src    = source_of(in, in2, x.rows, x.cols, x.col_factor);
        const int64_t width = in2 ? 2 * src.ld : src.ld;
        Planes to           = x.to;
        to.hi += at, to.lo += at;
        jobs.job[jobs.count++] = SplitJobs::Job{src, width, x.row_factor, to, x.by_column ? x.inverse + at : x.inverse, form, blocks};
        blocks += blocks_of(form, x.rows, width);
    };
    // a column job to each matrix, since its columns are its own
    auto add_cols = [&](SplitJobs &jobs, int64_t &blocks, const Split &x, int form) {
        add(jobs, blocks, x, x.in, nullptr, 0, form);
        if (x.in2)
            add(jobs, blocks, x, x.in2, nullptr, padded(x.cols), form);
    };
    // One launch while there is little to do, and it is the launches that count.
    int64_t values = 0, longest = 0;
    for (int i = 0; i < count; ++i) {
        values += what[i].rows * what[i].cols * (what[i].in2 ? 2 : 1);
        longest = std::max(longest, what[i].by_column ? what[i].rows : what[i].cols);
    }
    if (values <= kFewValues && longest <= 4096) {
        SplitJobs jobs{};
        int64_t blocks = 0;
        for (int i = 0; i < count; ++i)
            if (what[i].by_column)
                add_cols(jobs, blocks, what[i], what[i].rows > 256 ? kCols4 : kCols16);
            else
                add(jobs, blocks, what[i], what[i].in, what[i].in2, 0, kRowsWarp);
        if (blocks > 0) {
            CT_CUDA(launch_dependent(split_small_kernel, dim3((unsigned)blocks), dim3(256), 0, stream(), jobs));
            CT_LAUNCH_CHECK("split_small");
        }
        return CT_OK;
    }
    SplitJobs cols{};
    int64_t col_blocks = 0;
    for (int i = 0; i < count; ++i) {
        const Split &x = what[i];
        if (!x.by_column)
            continue;
        if (x.rows <= kShort * 64)
            add_cols(cols, col_blocks, x, kCols16);
        else
            CT_TRY(split_long_cols(st, x));
    }
    if (col_blocks > 0) { // of 16 columns each: a grid holds kMostSize of two matrices
        CT_CUDA(launch_dependent(split_short_cols_kernel, dim3((unsigned)col_blocks), dim3(256), 0, stream(), cols));
        CT_LAUNCH_CHECK("split_short_cols");
    }
    for (int i = 0; i < count; ++i) {
        const Split &x = what[i];
        if (x.by_column)
            continue;
        const Source src    = source_of(x.in, x.in2, x.rows, x.cols, x.col_factor);
        const int64_t width = x.in2 ? 2 * src.ld : src.ld;
        auto run = [&](auto kernel, int per_block) {
            return launch_dependent(kernel, dim3((unsigned)((x.rows + per_block - 1) / per_block)), dim3(256), 0, stream(), src, width, x.to, x.inverse);
        };
        if (width <= 256)
            CT_CUDA(run(split_rows_kernel<32, 2>, 8));
        else if (width <= 512)
            CT_CUDA(run(split_rows_kernel<32, 4>, 8));
        else if (width <= 1024)
            CT_CUDA(run(split_rows_kernel<32, 8>, 8));
        else if (width <= 2048)
            CT_CUDA(run(split_rows_kernel<256, 2>, 1));
        else if (width <= 4096)
            CT_CUDA(run(split_rows_kernel<256, 4>, 1));
        else if (width <= 8192)
            CT_CUDA(run(split_rows_kernel<256, 8>, 1));
        else if (width <= 8 * kLongQuads * 1024) {
            const int ranks    = width <= 2 * kLongQuads * 1024 ? 2 : width <= 4 * kLongQuads * 1024 ? 4 : 8;
            const int64_t each = (width + 4 * ranks - 1) / (4 * ranks) * 4;
            CT_CUDA(launch_dependent_cluster(split_long_rows_kernel, ranks, dim3((unsigned)(x.rows * ranks)), dim3(256), 0, stream(), src, width, ranks, each,
                                             x.to, x.inverse));
        } else
            CT_CUDA(run(split_rows_kernel<256, 8>, 1)); // read twice
        CT_LAUNCH_CHECK("split_rows");
    }
    return CT_OK;
}

namespace {

// Tile and slices of a product by what they take, in microseconds: a stage of a pair's 256 x 256 tile ~ 0.95, of a single CTA's 128 x 128 ~ 0.6;
// filling and draining a tile as much as four stages; the slices' sums written, read and a launch.
struct Plan {
    bool pair  = false;
    int splits = 1;
    double cost = 1e300;
};
int64_t stages_of(const Wanted &x) { return ((x.mn ? x.a.rows : x.a.cols) + 63) / 64; }
int64_t tiles_of(const Wanted &x, int64_t side) { return ((x.m + side - 1) / side) * ((x.n + side - 1) / side); }
double cost_of(const Wanted &x, int splits, int64_t waves, bool pair) {
    return (double)waves * (double)((stages_of(x) + splits - 1) / splits + 4) * (pair ? 0.95 : 0.6);
}
double join_cost(const Wanted &x, int splits) { return splits > 1 ? 3.0 + 0.1 * splits + (double)(x.m * x.n) * (splits + 1) * 4 / 5e6 : 0.0; }
bool may_split(const Wanted &x, int splits) { return splits == 1 || stages_of(x) >= 4 * splits; }
int whole_slices(const Wanted &x, int splits) { // no empty slice
    const int64_t stages = stages_of(x), each = (stages + splits - 1) / splits;
    return splits > 1 ? (int)((stages + each - 1) / each) : 1;
}
Plan plan_of(const DeviceState *st, const Wanted &x) {
    Plan best;
    for (int kind = 0; kind < 2; ++kind) {
        const int64_t units = kind ? st->sm_count / 2 : st->sm_count, tiles = tiles_of(x, kind ? 256 : 128);
        for (int s = 1; s <= 32 && may_split(x, s); ++s) {
            const double cost = cost_of(x, s, (tiles * s + units - 1) / units, kind != 0) + join_cost(x, s);
            if (cost < best.cost)
                best.cost = cost, best.pair = kind != 0, best.splits = s;
        }
    }
    best.splits = whole_slices(x, best.splits);
    return best;
}
// Both at once, on single CTAs, and their joins at once: TilesOfTwo, where the longer tiles are no more than the CTAs.  Gated gradient of
// 404 x 322 x 177 30 us one after the other, so 19, of 1315 x 118 x 773 41 and 32, of 1537 x 771 x 2050 120 and 103.
struct Shared {
    bool use   = false;
    int longer = 0, turns = 0;
};
Shared plan_both(const DeviceState *st, const Wanted *x, Plan *plan) {
    constexpr int kSplits[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32};
    const int64_t units = st->sm_count;
    double best         = plan[0].cost + plan[1].cost + 3.0; // a launch
    Shared how;
    for (int s : kSplits)
        for (int t : kSplits) {
            if (!may_split(x[0], s) || !may_split(x[1], t))
                break;
            const int splits[2]     = {s, t};
            const int64_t tiles[2]  = {tiles_of(x[0], 128) * s, tiles_of(x[1], 128) * t};
            const double of_tile[2] = {cost_of(x[0], s, 1, false), cost_of(x[1], t, 1, false)};
            const int longer        = of_tile[0] >= of_tile[1] ? 0 : 1;
            const int64_t spare = units - tiles[longer], others = tiles[1 - longer];
            const double lt = of_tile[longer], ot = of_tile[1 - longer], join = std::max(join_cost(x[0], s), join_cost(x[1], t));
            if (spare < 0 || others > 0x3fffffff)
                continue;
            for (int turns = (int)(lt / ot); turns <= (int)(lt / ot) + 1; ++turns) {
                const int64_t first = spare > 0 ? std::min<int64_t>(turns, (others + spare - 1) / spare) : 0, left = std::max<int64_t>(0, others - turns * spare);
                const double cost = std::max(lt, (double)first * ot) + (double)((left + units - 1) / units) * ot + join;
                if (cost < best) {
                    best = cost, how.use = true, how.longer = longer, how.turns = turns;
                    plan[0].splits = splits[0], plan[1].splits = splits[1], plan[0].pair = plan[1].pair = false;
                }
            }
        }
    if (how.use)
        for (int i = 0; i < 2; ++i)
            plan[i].splits = whole_slices(x[i], plan[i].splits);
    return how;
}

bool whole(const void *q) { return (reinterpret_cast<uintptr_t>(q) & 15u) == 0; }

} // namespace

ct_status products(DeviceState *st, const Wanted *what, int count) {
    const char *name = "fused_product";
    Plan plan[2]     = {plan_of(st, what[0]), {}};
    Shared both;
    if (count == 2) {
        plan[1] = plan_of(st, what[1]);
        both    = plan_both(st, what, plan);
    }
    Scratch partial[2];
    Product p[2]{};
    Store::Params e[2]{};
    Joins joins{};
    auto join = [&]() -> ct_status {
        if (joins.count) {
            CT_CUDA(launch_dependent(join_slices_kernel, dim3((unsigned)joins.blocks), dim3(256), 0, stream(), joins, (const uint32_t *)st->flags_dev));
            CT_LAUNCH_CHECK("join_slices");
        }
        joins = Joins{};
        return CT_OK;
    };
    for (int i = 0; i < count; ++i) {
        const Wanted &x  = what[i];
        const Result &to = x.to;
        p[i].m = x.m, p[i].n = x.n, p[i].row_scale = x.row_scale, p[i].col_scale = x.col_scale;
        const int vec = (to.stride & 3) == 0 && whole(to.out) && whole(to.out2) ? 1 : 0;
        e[i].out = to.out, e[i].out2 = to.out2, e[i].n = to.cols, e[i].stride = to.stride, e[i].second = to.second, e[i].add = to.add ? 1 : 0;
        e[i].vec = vec;
        if (plan[i].splits > 1) {
            const int64_t pitch = (x.n + 3) / 4 * 4;
            CT_TRY(partial[i].get((size_t)plan[i].splits * x.m * pitch * 4));
            e[i].out = partial[i].as<float>(), e[i].out2 = nullptr, e[i].n = e[i].stride = pitch, e[i].second = 0, e[i].slice = x.m * pitch, e[i].add = 0;
            e[i].vec = 1;
            int shift = 3;
            while (shift < 8 && (4 << shift) < x.n)
                ++shift;
            const int64_t strips = (x.n + (4 << shift) - 1) / (4 << shift), turns = (x.m + (256 >> shift) - 1) / (256 >> shift);
            joins.job[joins.count++] = Joins::Job{partial[i].as<const float>(), plan[i].splits, shift, x.m, x.n, pitch, strips, joins.blocks, to.out,
                                                  to.out2, to.cols, to.stride, to.second, vec, to.add ? 1 : 0};
            joins.blocks += strips * std::max<int64_t>(1, std::min<int64_t>(turns, (int64_t)st->sm_count * 16 / strips));
        }
        if (both.use)
            continue;
        if (x.mn)
            CT_TRY(plan[i].pair ? (launch<Store, 256, 2, true, true>(st, x.a, x.b, p[i], e[i], plan[i].splits, name))
                                : (launch<Store, 128, 1, true, true>(st, x.a, x.b, p[i], e[i], plan[i].splits, name)));
        else
            CT_TRY(plan[i].pair ? (launch<Store, 256, 2, false, false>(st, x.a, x.b, p[i], e[i], plan[i].splits, name))
                                : (launch<Store, 128, 1, false, false>(st, x.a, x.b, p[i], e[i], plan[i].splits, name)));
        CT_TRY(join()); // while the slices are in L2
    }
    if (both.use) {
        Maps maps[2];
        CT_TRY((prepare<Store, 128, 1, false, false>(st, what[0].a, what[0].b, plan[0].splits, maps[0], p[0], name)));
        CT_TRY((prepare<Store, 128, 1, true, true>(st, what[1].a, what[1].b, plan[1].splits, maps[1], p[1], name)));
        static bool set_dev[16] = {};
        CT_TRY(allow_shared(st, two_products_kernel, set_dev));
        const int grid = (int)std::min<int64_t>((int64_t)p[0].total + p[1].total, st->sm_count);
        p[0].chunk_first = p[1].chunk_first = p[0].total + p[1].total <= grid ? kChunk : kChunkFirst;
        CT_CUDA(launch_dependent(two_products_kernel, dim3((unsigned)grid), dim3(kThreads), (size_t)kSmem, stream(), maps[0], p[0], e[0], maps[1], p[1], e[1],
                                 both.longer, both.turns));
        CT_LAUNCH_CHECK(name);
        CT_TRY(join());
    }
    return CT_OK;
}

namespace {

// Sums of eight columns to a lane (16 bytes of each plane) over the block's rows, a row to each warp in turn.
__global__ void __launch_bounds__(256) plane_sums_kernel(
    const Planes x, const float *__restrict__ row_weight, int64_t rows_each, double *__restrict__ partial) {
    __shared__ float sums[8][256];
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c  = (int64_t)blockIdx.x * 256 + lane * 8, cols = x.cols;
    const int64_t r0 = (int64_t)blockIdx.y * rows_each, r1 = min(x.rows, r0 + rows_each);
    float s[8] = {};
    if (c < cols)
#pragma unroll 4
        for (int64_t r = r0 + warp; r < r1; r += 8) {
            const float w = row_weight[r];
            const uint4 h = *reinterpret_cast<const uint4 *>(x.hi + r * x.ld + c), l = *reinterpret_cast<const uint4 *>(x.lo + r * x.ld + c);
            const __half2 *hi = reinterpret_cast<const __half2 *>(&h), *lo = reinterpret_cast<const __half2 *>(&l);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                s[2 * q]     = __fmaf_rn(w, __fmaf_rn(__low2float(lo[q]), kLoInv, __low2float(hi[q])), s[2 * q]);
                s[2 * q + 1] = __fmaf_rn(w, __fmaf_rn(__high2float(lo[q]), kLoInv, __high2float(hi[q])), s[2 * q + 1]);
            }
        }
#pragma unroll
    for (int q = 0; q < 8; ++q)
        sums[warp][lane * 8 + q] = s[q];
    __syncthreads();
    const int64_t mine = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (mine < cols) {
        double all = 0.0;
#pragma unroll
        for (int w = 0; w < 8; ++w)
            all += (double)sums[w][threadIdx.x];
        partial[(int64_t)blockIdx.y * cols + mine] = all;
    }
}
// 32 columns to a block, a warp takes every 32nd part.
__global__ void __launch_bounds__(1024) join_columns_kernel(
    const double *__restrict__ partial, int64_t parts, int64_t n, int64_t width, float *__restrict__ first, float *__restrict__ second) {
    __shared__ double sums[32][33];
    griddep_wait();
    griddep_launch_dependents();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    double s = 0.0;
    if (c < width)
#pragma unroll 8
        for (int64_t p = warp; p < parts; p += 32)
            s += partial[p * width + c];
    sums[warp][lane] = s;
    __syncthreads();
    s = sums[lane][warp]; // column `warp` of the block, part `lane`
#pragma unroll
    for (int o = 16; o; o >>= 1)
        s += __shfl_xor_sync(0xffffffffu, s, o);
    const int64_t mine = (int64_t)blockIdx.x * 32 + warp;
    float *out         = mine < n ? first : second;
    if (lane == 0 && mine < width && out)
        out[mine < n ? mine : mine - n] = (float)s;
}

} // namespace

ct_status join_columns(const double *partial, int64_t parts, int64_t n, int64_t width, float *first, float *second) {
    CT_CUDA(launch_dependent(join_columns_kernel, dim3((unsigned)((width + 31) / 32)), dim3(1024), 0, stream(), partial, parts, n, width, first, second));
    CT_LAUNCH_CHECK("join_columns");
    return CT_OK;
}

ct_status column_sums(DeviceState *st, const Planes &x, const float *row_weight, float *out) {
    const int64_t strips = (x.cols + 255) / 256;
    const int64_t slices = row_slices(st, x.rows, strips);
    const int64_t each = (x.rows + slices - 1) / slices, parts = (x.rows + each - 1) / each;
    Scratch partial;
    CT_TRY(partial.get((size_t)(parts * x.cols) * 8));
    CT_CUDA(launch_dependent(plane_sums_kernel, dim3((unsigned)strips, (unsigned)parts), dim3(256), 0, stream(), x, row_weight, each, partial.as<double>()));
    CT_LAUNCH_CHECK("plane_sums");
    return join_columns(partial.as<const double>(), parts, x.cols, x.cols, out, nullptr);
}

} // namespace fused
} // namespace ct
