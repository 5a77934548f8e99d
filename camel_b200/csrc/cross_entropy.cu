// Softmax cross entropy of a dense layer's logits, and its gradient, without keeping the logits.
//
//   lse = log(sum exp z), loss = lse - z[target];  d = dloss (exp(z - lse) - [target]),  dx = d . w^T, dw = x^T . d, dbias = column sums of d
//
// Forward: a product whose tiles are not stored (fused_product.cuh).  A thread of the epilogue has a row and a quarter of the tile's columns in
// registers; it leaves their maximum, the sum of exponentials about it and, where it meets the target, that logit.  ce_join_kernel adds
// up a row's parts: 32 bytes for 256 logits.
// Gradient: the same product again, whose epilogue turns the logits into d / dloss = exp(z - lse) - [target], in [-1, 1], as planes of float16
// pairs under one scale.  A piece of the vocabulary at a time they are the left operand of dx += d . w^T as they lie (rows weighted by
// dloss at the end), and the right operand of dw = x'^T . d with their rows as k, x' being x with dloss in its rows.
// A pair holds d / dloss to 2^-23 of itself down to 2^-28, and to 2^-50 below: one scale for all, since a row's largest, 1 - p[target], is known
// only behind its last tile, and rows meet columns of any size in dw.
// Up to 16 rows have their logits written, and take few_rows.cu and few_rows_grad.cuh.
// Few classes (kFewClasses) take kernels of their own, whose logits are memory's smallest part; under the reduced precision the logits of a
// piece of the rows are written, by the library's products.
#include "fastmath.cuh"
#include "few_rows_grad.cuh"
#include "stream_product.cuh"

namespace ct {
namespace {

// One block per row of logits: running maximum and sum, then the loss.
__global__ void __launch_bounds__(256) ce_rows_kernel(
    const float *__restrict__ z, const int64_t *__restrict__ targets, int64_t n, float *__restrict__ loss, float *__restrict__ lse) {
    __shared__ float top_s[8], sum_s[8];
    griddep_wait();
    griddep_launch_dependents();
    const float *row = z + (int64_t)blockIdx.x * n;
    float top = -INFINITY, sum = 0.0f;
    for (int64_t c = threadIdx.x; c < n; c += 256)
        top = row[c] > top || row[c] != row[c] ? row[c] : top; // a NaN stays: nothing compares greater
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        const float other = __shfl_xor_sync(0xffffffffu, top, o);
        top               = other > top || other != other ? other : top;
    }
    if ((threadIdx.x & 31) == 0)
        top_s[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int w = 0; w < 8; ++w)
        top = top_s[w] > top || top_s[w] != top_s[w] ? top_s[w] : top;
    const float base = top == -INFINITY ? 0.0f : top; // all logits -inf: the sum is 0
    for (int64_t c = threadIdx.x; c < n; c += 256)
        sum = __fadd_rn(sum, expf(__fsub_rn(row[c], base)));
#pragma unroll
    for (int o = 16; o; o >>= 1)
        sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, o));
    if ((threadIdx.x & 31) == 0)
        sum_s[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.0f;
        for (int w = 0; w < 8; ++w)
            sum = __fadd_rn(sum, sum_s[w]);
        const float l   = __fadd_rn(base, logf(sum));
        const int64_t t = targets[blockIdx.x];
        if (lse)
            lse[blockIdx.x] = l;
        if (loss)
            loss[blockIdx.x] = t >= 0 && t < n ? __fsub_rn(l, row[t]) : 0.0f;
    }
}

// Long rows: the parts that ce_join_kernel adds up, 4096 logits to a block, read once.  By one block to a row 4 x 64 x 64000 took 30 us, so 11,
// 1 x 1024 x 131072 121 and 82.
constexpr int kPartLogits = 4096;
__global__ void __launch_bounds__(256) ce_parts_kernel(
    const float *__restrict__ z, const int64_t *__restrict__ targets, int64_t rows, int64_t n, float2 *__restrict__ part, float *__restrict__ at_target) {
    __shared__ float top_s[8], sum_s[8];
    griddep_wait();
    griddep_launch_dependents();
    const float *row = z + (int64_t)blockIdx.y * n;
    const int64_t c0 = (int64_t)blockIdx.x * kPartLogits;
    float v[kPartLogits / 256], top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kPartLogits / 256; ++i) {
        const int64_t c = c0 + i * 256 + threadIdx.x;
        v[i]            = c < n ? row[c] : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < kPartLogits / 256; ++i)
        top = fmaxf(top, v[i]); // a NaN shows in the sum
#pragma unroll
    for (int o = 16; o; o >>= 1)
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0)
        top_s[threadIdx.x >> 5] = top;
    __syncthreads();
    for (int w = 0; w < 8; ++w)
        top = fmaxf(top, top_s[w]);
    const float base = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for (int i = 0; i < kPartLogits / 256; ++i)
        sum = __fadd_rn(sum, expf(__fsub_rn(v[i], base)));
#pragma unroll
    for (int o = 16; o; o >>= 1)
        sum = __fadd_rn(sum, __shfl_xor_sync(0xffffffffu, sum, o));
    if ((threadIdx.x & 31) == 0)
        sum_s[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        sum = 0.0f;
        for (int w = 0; w < 8; ++w)
            sum = __fadd_rn(sum, sum_s[w]);
        part[(int64_t)blockIdx.x * rows + blockIdx.y] = make_float2(top, sum);
        const int64_t t = targets[blockIdx.y];
        if (t >= c0 && t < n && t < c0 + kPartLogits)
            at_target[blockIdx.y] = row[t];
    }
}

// x without the rows that have no target: 0 x anything of theirs is no term of dw.
__global__ void __launch_bounds__(256) ce_rows_with_target_kernel(
    const float *__restrict__ x, const int64_t *__restrict__ targets, int64_t count, int64_t k, int64_t n, float *__restrict__ out) {
    griddep_wait();
    griddep_launch_dependents();
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
        const int64_t t = targets[i / k];
        out[i]          = t >= 0 && t < n ? x[i] : 0.0f;
    }
}

// d in the place of the logits
__global__ void __launch_bounds__(256) ce_slopes_kernel(
    float *__restrict__ z, const int64_t *__restrict__ targets, const float *__restrict__ lse, const float *__restrict__ dloss, int64_t count, int64_t n) {
    griddep_wait();
    griddep_launch_dependents();
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / n, c = i - r * n, t = targets[r];
        const float p = expf(__fsub_rn(z[i], lse[r]));
        z[i]          = t >= 0 && t < n ? __fmul_rn(dloss ? dloss[r] : 1.0f, c == t ? __fsub_rn(p, 1.0f) : p) : 0.0f;
    }
}

// ---- logits that stay in the epilogue ----

// 2^x, to 2^-22 of itself; 0 below 2^-126.  Its argument is a rounded product with a rounded constant: three roundings of |z - lse| in all, about as
// many as the logit has of its own, so they are not taken back.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
constexpr float kLog2e = 1.44269504f;

// acc becomes the logits of the lane's row; columns past the last are -inf.  NC columns from col.
template <int NC>
__device__ __forceinline__ void logits_of(const fused::Product &p, const float *bias, float *acc, float rs, int64_t col) {
    const bool all = col + NC <= p.n;
#pragma unroll
    for (int j = 0; j < NC / 4; ++j) {
        const float4 s = fused::scales4(p.col_scale, col + 4 * j);
        acc[4 * j] = __fmul_rn(acc[4 * j], fused::weight(rs, s.x)), acc[4 * j + 1] = __fmul_rn(acc[4 * j + 1], fused::weight(rs, s.y));
        acc[4 * j + 2] = __fmul_rn(acc[4 * j + 2], fused::weight(rs, s.z)), acc[4 * j + 3] = __fmul_rn(acc[4 * j + 3], fused::weight(rs, s.w));
    }
    if (bias)
#pragma unroll
        for (int j = 0; j < NC; ++j)
            acc[j] = __fadd_rn(acc[j], col + j < p.n ? __ldg(bias + col + j) : 0.0f);
    if (!all)
#pragma unroll
        for (int j = 0; j < NC; ++j)
            acc[j] = col + j < p.n ? acc[j] : -INFINITY;
}

struct SumExp {
    static constexpr bool kTwin = false;
    struct Params {
        const float *bias;
        const int64_t *targets;
        float2 *part; // [4 tiles_n][m]: maximum, sum
        float *at_target;
    };
    template <int COLS>
    __device__ static __forceinline__ void store(
        const fused::Product &p, const Params &e, float (&z)[COLS], int64_t row0, int lane, int64_t col0, int, int slot, uint8_t *) {
        const int64_t row = row0 + lane;
        const bool mine   = row < p.m;
        logits_of<COLS>(p, e.bias, z, mine ? __ldg(p.row_scale + row) : 0.0f, col0);
        const int64_t t = mine ? e.targets[row] : -1, at = t >= 0 ? t - col0 : -1;
        if (__any_sync(0xffffffffu, at >= 0 && at < COLS)) { // one in n / COLS tiles for each row
            float found = 0.0f;
#pragma unroll
            for (int j = 0; j < COLS; ++j)
                found = at == j ? z[j] : found;
            if (at >= 0 && at < COLS && col0 + at < p.n)
                e.at_target[row] = found;
        }
        float top[4] = {z[0], z[1], z[2], z[3]};
#pragma unroll
        for (int j = 4; j < COLS; ++j)
            top[j & 3] = fmaxf(top[j & 3], z[j]);
        const float mx   = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
        const float base = mx == -INFINITY ? 0.0f : mx;
        float sum[4]     = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < COLS; ++j)
            sum[j & 3] = __fadd_rn(sum[j & 3], exp2_fast(__fmul_rn(__fsub_rn(z[j], base), kLog2e)));
        if (mine)
            e.part[(int64_t)slot * p.m + row] = make_float2(mx, __fadd_rn(__fadd_rn(sum[0], sum[1]), __fadd_rn(sum[2], sum[3])));
    }
};

// (maximum, sum of exponentials about it) of two sets of logits.
__device__ __forceinline__ float2 join_parts(float2 a, float2 b) {
    const float top  = fmaxf(a.x, b.x);
    const float base = top == -INFINITY ? 0.0f : top;
    const float x    = __fmul_rn(a.y, exp2_fast(__fmul_rn(__fsub_rn(a.x, base), kLog2e))), y = __fmul_rn(b.y, exp2_fast(__fmul_rn(__fsub_rn(b.x, base), kLog2e)));
    return make_float2(top, __fadd_rn(a.x == -INFINITY ? a.y : x, b.x == -INFINITY ? b.y : y)); // nothing but -inf: a sum of 0, or NaN
}

// A row's parts: eight rows to a block, a lane group of eight takes every 32nd part (with 32 rows to a block 64 rows of 500 parts took 23 us).
__global__ void __launch_bounds__(256) ce_join_kernel(
    const float2 *__restrict__ part, int slots, const float *__restrict__ at_target, const int64_t *__restrict__ targets, int64_t m, int64_t n,
    float *__restrict__ loss, float *__restrict__ lse, const uint32_t *__restrict__ flags) {
    __shared__ float2 words[32][8];
    griddep_wait();
    griddep_launch_dependents();
    if (*reinterpret_cast<const volatile uint32_t *>(flags + FLAG_TIMEOUT) != 0) // the parts were not computed
        return;
    const int at = threadIdx.x & 7, group = threadIdx.x >> 3;
    const int64_t row = (int64_t)blockIdx.x * 8 + at;
    float2 v = make_float2(-INFINITY, 0.0f);
    if (row < m)
#pragma unroll 4
        for (int s = group; s < slots; s += 32)
            v = join_parts(v, part[(int64_t)s * m + row]);
    words[group][at] = v;
    __syncthreads();
    if (group == 0 && row < m) {
        for (int w = 1; w < 32; ++w)
            v = join_parts(v, words[w][at]);
        const float l   = __fadd_rn(v.x == -INFINITY && v.y == v.y ? 0.0f : v.x, logf(v.y));
        const int64_t t = targets[row];
        if (lse)
            lse[row] = l;
        if (loss)
            loss[row] = t >= 0 && t < n ? __fsub_rn(l, at_target[row]) : 0.0f;
    }
}

// Streamed: a thread has every sixteenth of a row's logits, and keeps maximum and sum across the CTA's tiles.
struct SumExpStream {
    static constexpr bool kTwin  = false;
    static constexpr int kShares = fused::kStreamDrain * 32 / fused::kStreamPass;
    struct Params {
        const float *bias;
        const int64_t *targets;
        float2 *part; // [grid][rows]
        float *at_target;
        int64_t rows; // of all launches
    };
    struct State {
        float2 v[4]; // maximum, sum; of row t % 16 of each pass
    };
    __device__ static __forceinline__ void init(State &s) { s.v[0] = s.v[1] = s.v[2] = s.v[3] = make_float2(-INFINITY, 0.0f); }
    template <int Q>
    __device__ static __forceinline__ void tile(const fused::Stream &p, const Params &e, State &s, const float *z, int64_t c0, int cols, int t) {
        constexpr int S = kShares, N = 128 / S;
        const int r = 16 * Q + (t & 15), first = t >> 4;
        if (r >= p.m)
            return;
        const float rs   = p.row_scale[r] * fused::kStreamUp;
        const float *row = z + (t & 15) * fused::kStreamPitch + first;
        float v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = first + i * S;
            v[i]        = __fmul_rn(row[i * S], rs);
            if (e.bias && c < cols)
                v[i] = __fadd_rn(v[i], __ldg(e.bias + c0 + c));
            v[i] = c < cols ? v[i] : -INFINITY;
        }
        float top = s.v[Q].x;
#pragma unroll
        for (int i = 0; i < N; ++i)
            top = fmaxf(top, v[i]);
        const float base = top == -INFINITY ? 0.0f : top;
        float sum        = s.v[Q].x == -INFINITY ? s.v[Q].y : __fmul_rn(s.v[Q].y, exp2_fast(__fmul_rn(__fsub_rn(s.v[Q].x, base), kLog2e)));
#pragma unroll
        for (int i = 0; i < N; ++i)
            sum = __fadd_rn(sum, exp2_fast(__fmul_rn(__fsub_rn(v[i], base), kLog2e)));
        s.v[Q]           = make_float2(top, sum);
        const int64_t at = e.targets[r] >= 0 ? e.targets[r] - c0 : -1;
        if (at >= 0 && at < cols && (int)at % S == first)
#pragma unroll
            for (int i = 0; i < N; ++i)
                if ((int)at / S == i)
                    e.at_target[r] = v[i];
    }
    // The shares of each row, in order.
    __device__ static __forceinline__ void finish(const fused::Stream &p, const Params &e, State &s, float *z, int t) {
        float2 *words = reinterpret_cast<float2 *>(z); // [share][16]
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            fused::stream_epilogue_sync();
            words[t] = s.v[q];
            fused::stream_epilogue_sync();
            if (t < 16 && 16 * q + t < p.m) {
                float2 v = words[t];
                for (int i = 1; i < kShares; ++i)
                    v = join_parts(v, words[i * 16 + t]);
                e.part[(int64_t)blockIdx.x * e.rows + 16 * q + t] = v;
            }
        }
    }
};

ct_status ce_fused(
    DeviceState *st, const float *x, const float *w, const float *bias, const int64_t *targets, int64_t m, int64_t k, int64_t n, float *loss, float *lse) {
    using namespace fused;
    const int64_t lk = padded(k), ln = padded(n);
    const bool few = takes_stream(m, k, n), pair = !few && takes_pairs(st, m, n);
    int per;
    const int64_t slots = few ? (int64_t)stream_grid(st, n, &per) : pair ? (n + 255) / 256 * 4 : (n + 127) / 128 * 4;
    Parts parts;
    const size_t xp = parts.planes(m, lk), xi = parts.take((size_t)m * 4), wp = few ? 0 : parts.planes(k, ln),
                 wi = few ? 0 : parts.take((size_t)scales(ln) * 4),
                 pp = parts.take((size_t)(slots * m) * 8), tp = parts.take((size_t)m * 4);
    Scratch s;
    CT_TRY(s.get(parts.bytes));
    const Planes px = planes_at(s, xp, m, lk, lk), pw = planes_at(s, wp, k, ln, ln);
    const Split operands[2] = {{x, nullptr, m, k, false, nullptr, px, s.as<float>(xi)}, {w, nullptr, k, n, true, nullptr, pw, s.as<float>(wi)}};
    CT_TRY(split(st, operands, few ? 1 : 2));
    float2 *part     = s.as<float2>(pp);
    float *at_target = s.as<float>(tp);
    if (few) {
        Stream p{};
        p.w = w, p.k = k, p.n = p.ld = n, p.row_scale = s.as<float>(xi);
        const SumExpStream::Params e{bias, targets, part, at_target, m};
        CT_TRY(launch_stream<SumExpStream>(st, px, p, e, "cross_entropy", [](SumExpStream::Params f, int64_t r) {
            f.targets += r, f.part += r, f.at_target += r;
            return f;
        }));
    } else {
        Product p{};
        p.m = m, p.n = n, p.row_scale = s.as<float>(xi), p.col_scale = s.as<float>(wi);
        const SumExp::Params e{bias, targets, part, at_target};
        CT_TRY(pair ? (launch<SumExp, 256, 2, false, true>(st, px, pw, p, e, 1, "cross_entropy"))
                    : (launch<SumExp, 128, 1, false, true>(st, px, pw, p, e, 1, "cross_entropy")));
    }
    CT_CUDA(launch_dependent(ce_join_kernel, dim3((unsigned)((m + 7) / 8)), dim3(256), 0, stream(), (const float2 *)part, (int)slots,
                             (const float *)at_target, targets, m, n, loss, lse, (const uint32_t *)st->flags_dev));
    CT_LAUNCH_CHECK("ce_join");
    return CT_OK;
}

// ---- the gradient ----

constexpr float kSlopeScale = 16384.0f; // 2^14: d / dloss is at most 1, and representable up to 3.99

// Logits to the planes of (exp(z - lse) - [target]) 2^14.
struct Slopes {
    static constexpr bool kTwin = false;
    struct Params {
        const float *bias, *lse;
        const int64_t *targets;
        int64_t first, classes; // of the piece's columns
        __half *hi, *lo;
        int64_t ld;
    };
    template <int COLS>
    __device__ static __forceinline__ void store(
        const fused::Product &p, const Params &e, float (&z)[COLS], int64_t row0, int lane, int64_t col0, int, int, uint8_t *stage) {
        const int64_t row  = row0 + lane;
        const bool mine    = row < p.m;
        const float rs     = mine ? __ldg(p.row_scale + row) : 0.0f, l = mine ? __ldg(e.lse + row) : 0.0f;
        const int64_t t    = mine ? e.targets[row] : -1;
        const bool has     = t >= 0 && t < e.classes;
        const int64_t at   = has ? t - e.first - col0 : -1;
        const int64_t left = p.m - row0;
        const int rows     = left < 0 ? 0 : (left < 32 ? (int)left : 32);
        if (rows == 0)
            return;
#pragma unroll
        for (int g = 0; g < COLS / 16; ++g) {
            const int64_t col = col0 + g * 16;
            if (col >= p.n)
                break;
            float *d = z + g * 16;
            logits_of<16>(p, e.bias, d, rs, col);
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float v = exp2_fast(__fmul_rn(__fsub_rn(d[j], l), kLog2e));
                d[j]          = has ? __fmul_rn(at == g * 16 + j ? __fsub_rn(v, 1.0f) : v, kSlopeScale) : 0.0f;
            }
            // rows of 64 bytes, hi terms and lo terms: 16-byte slots XOR-swizzled by row
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                __half2 hi[4], lo[4];
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    fused::split2(d[8 * j + 2 * q], d[8 * j + 2 * q + 1], hi[q], lo[q]);
                *reinterpret_cast<uint4 *>(stage + fused::stage_slot(lane, j))     = *reinterpret_cast<uint4 *>(hi);
                *reinterpret_cast<uint4 *>(stage + fused::stage_slot(lane, j + 2)) = *reinterpret_cast<uint4 *>(lo);
            }
            __syncwarp();
            const int sub = lane & 3, rr = lane >> 2;
            __half *to = (sub < 2 ? e.hi : e.lo) + (row0 + rr) * e.ld + col + (sub & 1) * 8;
            if (col + (sub & 1) * 8 < p.n) // to the end of the slot, which ld covers
#pragma unroll
                for (int it = 0; it < 4; ++it) {
                    const int r = it * 8 + rr;
                    if (r < rows)
                        *reinterpret_cast<uint4 *>(to + (int64_t)it * 8 * e.ld) = *reinterpret_cast<const uint4 *>(stage + fused::stage_slot(r, sub));
                }
            __syncwarp();
        }
    }
};

// Streamed (without dx): a warp has a row of a tile at a time, a lane four of its columns.
struct SlopesStream {
    static constexpr bool kTwin = false;
    using Params = Slopes::Params;
    struct State {};
    __device__ static __forceinline__ void init(State &) {}
    template <int Q>
    __device__ static __forceinline__ void tile(const fused::Stream &p, const Params &e, State &, const float *z, int64_t c0, int cols, int t) {
        const int c = (t & 31) * 4, rows = p.m - 16 * Q < 16 ? p.m - 16 * Q : 16;
        if (c >= cols)
            return;
        for (int i = t >> 5; i < rows; i += fused::kStreamDrain) {
            const int r      = 16 * Q + i;
            const float rs   = p.row_scale[r] * fused::kStreamUp, l = e.lse[r];
            const int64_t tg = e.targets[r], at = tg - e.first - c0;
            const bool has   = tg >= 0 && tg < e.classes;
            float d[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float v = __fmul_rn(z[i * fused::kStreamPitch + c + q], rs);
                if (e.bias && c + q < cols)
                    v = __fadd_rn(v, __ldg(e.bias + c0 + c + q));
                v    = exp2_fast(__fmul_rn(__fsub_rn(v, l), kLog2e));
                d[q] = has && c + q < cols ? __fmul_rn(at == c + q ? __fsub_rn(v, 1.0f) : v, kSlopeScale) : 0.0f;
            }
            __half2 hi[2], lo[2];
            fused::split2(d[0], d[1], hi[0], lo[0]);
            fused::split2(d[2], d[3], hi[1], lo[1]);
            *reinterpret_cast<uint2 *>(e.hi + r * e.ld + c0 + c) = *reinterpret_cast<uint2 *>(hi); // ld covers it
            *reinterpret_cast<uint2 *>(e.lo + r * e.ld + c0 + c) = *reinterpret_cast<uint2 *>(lo);
        }
    }
    __device__ static __forceinline__ void finish(const fused::Stream &, const Params &, State &, float *, int) {}
};

// What the rows of d are weighted with behind the planes: dloss / 2^14 (never -0), and -0 for rows without a target, which take no part.
__global__ void __launch_bounds__(256) ce_weights_kernel(
    const float *__restrict__ dloss, const int64_t *__restrict__ targets, int64_t m, int64_t n, float *__restrict__ weight) {
    griddep_wait();
    griddep_launch_dependents();
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i < m)
        weight[i] = targets[i] >= 0 && targets[i] < n ? __fadd_rn(__fmul_rn(dloss ? dloss[i] : 1.0f, 1.0f / kSlopeScale), 0.0f) : __uint_as_float(fused::kNoPart);
}

ct_status ce_grad_fused(
    DeviceState *st, const float *x, const float *w, const float *bias, const int64_t *targets, const float *lse, const float *dloss, int64_t m, int64_t k,
    int64_t n, float *dx, float *dw, float *dbias) {
    using namespace fused;
    const int64_t lk = padded(k), ln = padded(n);
    // dx needs the weights' planes in any case, and with them tiles are sooner (20 x 1024 x 8192 78 us, streamed 89; 40 x 32000 205
    // and 219); without it 64 x 32000 takes 127 streamed, 186 by tiles.
    const bool few = !dx && takes_stream(m, k, n);
    // Pieces of the vocabulary: planes of d of up to 512 MB (more only above 2^19 rows, of 256 classes), alike in size and whole tiles.
    const int64_t most = std::max<int64_t>(256, (int64_t)(1u << 27) / m / 256 * 256);
    const int64_t pieces = (n + most - 1) / most;
    const int64_t piece = std::min<int64_t>(n, ((n + pieces - 1) / pieces + 255) / 256 * 256), ld = padded(piece);
    Parts parts;
    // The weights' planes for dx have a scale per row; with those folded into x they are the logits' as well, which saves a pre-pass over the
    // weights (1000 x 512 x 50257: 639 us, so 575) and keeps what features of different sizes meet.
    const size_t xp = parts.planes(m, lk), xi = parts.take((size_t)m * 4), dp = parts.planes(m, ld), rw = parts.take((size_t)m * 4);
    const bool weights = !few;
    const size_t wp = weights ? parts.planes(k, ln) : 0, wi = weights ? parts.take((size_t)scales(k) * 4) : 0;
    const size_t yp = dw ? parts.planes(m, lk) : 0, yi = dw ? parts.take((size_t)scales(lk) * 4) : 0;
    Scratch s;
    CT_TRY(s.get(parts.bytes));
    const Planes px = planes_at(s, xp, m, lk, lk), pw = planes_at(s, wp, k, ln, ln), py = planes_at(s, yp, m, lk, lk);
    float *weight = s.as<float>(rw);
    CT_CUDA(launch_dependent(ce_weights_kernel, dim3((unsigned)((m + 255) / 256)), dim3(256), 0, stream(), dloss, targets, m, n, weight));
    CT_LAUNCH_CHECK("ce_weights");
    Split operands[3];
    int operand_count = 0;
    if (weights)
        operands[operand_count++] = {w, nullptr, k, n, false, nullptr, pw, s.as<float>(wi)};
    if (dw)
        operands[operand_count++] = {x, nullptr, m, k, true, weight, py, s.as<float>(yi)};
    Split left = {x, nullptr, m, k, false, nullptr, px, s.as<float>(xi)};
    if (few) { // the logits' weights are read as they lie
        operands[operand_count++] = left;
    } else {
        left.col_factor = s.as<float>(wi);
    }
    CT_TRY(split(st, operands, operand_count));
    if (!few)
        CT_TRY(split(st, &left, 1));
    for (int64_t c = 0; c < n; c += piece) {
        const int64_t cols = std::min(piece, n - c);
        const Planes pd    = planes_at(s, dp, m, cols, ld);
        const Slopes::Params e{bias ? bias + c : nullptr, lse, targets, c, n, pd.hi, pd.lo, ld};
        if (few) {
            Stream p{};
            p.w = w + c, p.k = k, p.n = cols, p.ld = n, p.row_scale = s.as<float>(xi);
            CT_TRY(launch_stream<SlopesStream>(st, px, p, e, "cross_entropy_grad", [](Slopes::Params f, int64_t r) {
                f.lse += r, f.targets += r, f.hi += r * f.ld, f.lo += r * f.ld;
                return f;
            }));
        } else {
            Product p{};
            p.m = m, p.n = cols, p.row_scale = s.as<float>(xi);
            const Planes right = columns_of(pw, c, cols);
            const bool pair    = takes_pairs(st, m, cols);
            CT_TRY(pair ? (launch<Slopes, 256, 2, false, true>(st, px, right, p, e, 1, "cross_entropy_grad"))
                        : (launch<Slopes, 128, 1, false, true>(st, px, right, p, e, 1, "cross_entropy_grad")));
        }
        Wanted wanted[2];
        int count = 0;
        if (dx) {
            Result r{dx};
            r.cols = r.stride = k, r.add = c > 0;
            wanted[count++] = {pd, columns_of(pw, c, cols), false, m, k, weight, s.as<float>(wi), r};
        }
        if (dw) {
            Result r{dw + c};
            r.cols = cols, r.stride = n;
            wanted[count++] = {py, pd, true, k, cols, s.as<float>(yi), nullptr, r};
        }
        if (count)
            CT_TRY(products(st, wanted, count));
        if (dbias)
            CT_TRY(column_sums(st, pd, weight, dbias + c));
    }
    return CT_OK;
}

// ---- few classes: logits of up to kFewClasses columns, as the library's few-column products give them ----

// From 17 classes on the tiles of 128 win, empty as most of them is: gradient of 60000 x 785 x 17 494 us against 1626 (the library's products
// of more than 16 columns read x in many strips), of 2000 x 256 x 20 54 against 50.  At 10 classes the kernels below take 170 us, tiles as much as at 17.
constexpr int kFewClasses = 16;
// Rows of a block whose sums are one float32 chain, at most (60000 rows: 400).
constexpr int64_t kChainFew = 1024;

// A thread per row.
__global__ void __launch_bounds__(256) ce_few_kernel(
    const float *__restrict__ z, const int64_t *__restrict__ targets, int64_t m, int n, float *__restrict__ loss, float *__restrict__ lse) {
    griddep_wait();
    griddep_launch_dependents();
    const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (row >= m)
        return;
    const float *src = z + row * n;
    float top = -INFINITY, sum = 0.0f;
    for (int c = 0; c < n; ++c)
        top = fmaxf(top, src[c]);
    const float base = top == -INFINITY ? 0.0f : top;
    for (int c = 0; c < n; ++c)
        sum = __fadd_rn(sum, expf(__fsub_rn(src[c], base))); // a NaN shows here
    const float l   = __fadd_rn(base, logf(sum));
    const int64_t t = targets[row];
    if (lse)
        lse[row] = l;
    if (loss)
        loss[row] = t >= 0 && t < n ? __fsub_rn(l, src[t]) : 0.0f;
}

// d in the place of the logits, and the columns' sums over the block's 256 rows (partial may be null).
__global__ void __launch_bounds__(256) ce_few_slopes_kernel(
    float *__restrict__ z, const int64_t *__restrict__ targets, const float *__restrict__ lse, const float *__restrict__ dloss, int64_t m, int n,
    double *__restrict__ partial) {
    __shared__ float tile[256 * (kFewClasses + 1)];
    griddep_wait();
    griddep_launch_dependents();
    const int64_t row0 = (int64_t)blockIdx.x * 256;
    const int rows = (int)(m - row0 < 256 ? m - row0 : 256), pitch = n | 1;
    for (int i = threadIdx.x; i < rows * n; i += 256)
        tile[i / n * pitch + i % n] = z[row0 * n + i];
    __syncthreads();
    if ((int)threadIdx.x < rows) {
        const int64_t row = row0 + threadIdx.x, t = targets[row];
        const bool has = t >= 0 && t < n;
        const float l = lse[row], by = dloss ? dloss[row] : 1.0f;
        float *mine = tile + threadIdx.x * pitch;
        for (int c = 0; c < n; ++c) {
            const float p = expf(__fsub_rn(mine[c], l));
            mine[c]       = has ? __fmul_rn(by, c == t ? __fsub_rn(p, 1.0f) : p) : 0.0f;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < rows * n; i += 256)
        z[row0 * n + i] = tile[i / n * pitch + i % n];
    if (partial)
        for (int c = threadIdx.x >> 5; c < n; c += 8) {
            float s = 0.0f;
            for (int r = threadIdx.x & 31; r < rows; r += 32)
                s = __fadd_rn(s, tile[r * pitch + c]);
#pragma unroll
            for (int o = 16; o; o >>= 1)
                s = __fadd_rn(s, __shfl_xor_sync(0xffffffffu, s, o));
            if ((threadIdx.x & 31) == 0)
                partial[(int64_t)blockIdx.x * n + c] = (double)s;
        }
}

// dx = d . w^T and the parts of dw = x^T . d in one reading of x and d: a thread has a column of x, its weights and its sums in registers, 64
// rows of d come from shared memory at a time.  Blocks are strips x parts; a part has every parts-th 64 rows.  A row without a target takes
// no part, whatever x holds there.  Bound by issue, n FMAs of two values to a value of x.  Sums are chains of a part's rows, kChainFew at most, joined in 64 bits.
template <int N>
__global__ void __launch_bounds__(256) ce_few_back_kernel(
    const float *__restrict__ d, const float *__restrict__ x, const float *__restrict__ w, const int64_t *__restrict__ targets, int64_t m, int64_t k, int n,
    int64_t strips, int64_t parts, float *__restrict__ dx, double *__restrict__ partial) {
    constexpr int R = 64;
    __shared__ __align__(16) float tile[R][N];
    __shared__ int has_s[R];
    griddep_wait();
    griddep_launch_dependents();
    const int64_t part = blockIdx.x / strips, c = (blockIdx.x - part * strips) * 256 + threadIdx.x;
    f32x2 wc[N / 2], sum[N / 2];
#pragma unroll
    for (int j = 0; j < N / 2; ++j) {
        wc[j]  = pack2(c < k && 2 * j < n ? w[c * n + 2 * j] : 0.0f, c < k && 2 * j + 1 < n ? w[c * n + 2 * j + 1] : 0.0f);
        sum[j] = 0;
    }
    for (int64_t row0 = part * R; row0 < m; row0 += parts * R) {
        const int rows = (int)(m - row0 < R ? m - row0 : R);
        __syncthreads();
        for (int i = threadIdx.x; i < rows * N; i += 256)
            tile[i / N][i % N] = i % N < n ? d[(row0 + i / N) * n + i % N] : 0.0f;
        if ((int)threadIdx.x < rows) {
            const int64_t t   = targets[row0 + threadIdx.x];
            has_s[threadIdx.x] = t >= 0 && t < n;
        }
        __syncthreads();
        if (c >= k)
            continue;
        for (int r0 = 0; r0 < rows; r0 += 8) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                v[i] = partial && r0 + i < rows && has_s[r0 + i] ? x[(row0 + r0 + i) * k + c] : 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (r0 + i >= rows)
                    break;
                f32x2 back = 0, e[N / 2];
#pragma unroll
                for (int j = 0; j < N / 4; ++j) {
                    const float4 q = *reinterpret_cast<const float4 *>(&tile[r0 + i][4 * j]);
                    e[2 * j] = pack2(q.x, q.y), e[2 * j + 1] = pack2(q.z, q.w);
                }
#pragma unroll
                for (int j = 0; j < N / 2; ++j) {
                    sum[j] = fma2(pack2(v[i], v[i]), e[j], sum[j]);
                    back   = fma2(e[j], wc[j], back);
                }
                if (dx) {
                    float a, b;
                    unpack2(back, a, b);
                    dx[(row0 + r0 + i) * k + c] = __fadd_rn(a, b);
                }
            }
        }
    }
    if (partial && c < k)
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
            float a, b;
            unpack2(sum[j], a, b);
            if (2 * j < n)
                partial[(part * k + c) * n + 2 * j] = (double)a;
            if (2 * j + 1 < n)
                partial[(part * k + c) * n + 2 * j + 1] = (double)b;
        }
}

// The logits of few classes: of few rows by few_rows, whose cluster shares k.
ct_status few_logits(DeviceState *st, const float *x, const float *w, const float *bias, int64_t m, int64_t k, int64_t n, float *z) {
    if (m <= fused::kFewRows && k > 0 && ct_get_precision() == CT_PREC_3XTF32)
        return fused::few_rows(st, x, w, bias, nullptr, nullptr, m, k, n, 0, z, nullptr, nullptr);
    return ct_dense(x, w, bias, m, k, n, CT_ACT_NONE, z, nullptr);
}

// The whole gradient of up to 16 classes and 1024 columns of x in one reading of x, float32: a row of x for each warp of the block (8 or 16) in
// shared memory at a time, the next ones on their way.  Logits: a warp has four rows and a quarter of the columns of each 128, and its 4 N sums
// meet by halves; d: a thread to each; then half of the warps have the columns of dw as sums in registers, the other half those of w, for
// dx, and walk the rows.
// Bound by issue (half of the slots are busy, the FMAs of two values take a third) and by the phases' barriers.  60000 x 785 x 10: at the copy rate
// 58 us; as five kernels, each with its own reading of x or of d, 212; with columns of both w and dw in every thread 173; so 160.  dw's sums are
// chains of a block's rows, joined in 64 bits.
constexpr int kOneColumns = 1024;
// Between the rows of w in shared memory: an odd number of float4, so that eight of them lie in different banks (16 classes: 364 us at 16).
template <int P> constexpr int kOnePitch = (P / 4 | 1) * 4;
// Of shared memory: rows of x, parts of the logits, d, w.
constexpr int64_t one_words(int64_t k, int rows, int pitch, int ring) { return ring * rows * k + 4 * rows * pitch + rows * pitch + k * ((pitch / 4 | 1) * 4); }

template <int N, int RING, int THREADS>
__global__ void __launch_bounds__(THREADS, 512 / THREADS) ce_one_kernel(
    const float *__restrict__ x, const float *__restrict__ w, const float *__restrict__ bias, const int64_t *__restrict__ targets,
    const float *__restrict__ lse, const float *__restrict__ dloss, int64_t m, int k, int n, float *__restrict__ dx, double *__restrict__ partial) {
    constexpr int ROWS = THREADS / 32, HALF = THREADS / 2, SLOTS = kOneColumns / HALF, P = (N + 3) / 4 * 4, PW = kOnePitch<P>, GROUPS = ROWS / 4;
    constexpr int AT_ONCE = (SLOTS + 4) * N <= 100 ? 4 : 2; // rows whose logits a warp sums up at once: what the registers hold
    extern __shared__ __align__(16) float smem[];
    __shared__ int has_s[ROWS]; // a row without a target takes no part, whatever x holds there
    float *xs = smem, *parts = xs + RING * ROWS * k, *ds = parts + 4 * ROWS * P, *ws = ds + ROWS * P;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    griddep_wait();
    griddep_launch_dependents();
    const int64_t tiles = (m + ROWS - 1) / ROWS;
    auto fetch = [&](int64_t tile, int at) {
        if (tile < tiles) {
            const int64_t left = (m - tile * ROWS < ROWS ? m - tile * ROWS : ROWS) * k; // values; the rows are one piece
            const float *src   = x + tile * ROWS * k;
            const uint32_t to  = ptx::smem_u32(xs + at * ROWS * k);
            for (int64_t i = 4 * t; i < left; i += 4 * THREADS)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + (uint32_t)i * 4), "l"(src + i), "r"(left - i < 4 ? (int)(left - i) * 4 : 16)
                             : "memory");
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int i = 0; i < RING; ++i)
        fetch(blockIdx.x + (int64_t)i * gridDim.x, i);
    for (int i = t; i < k * PW; i += THREADS)
        ws[i] = i % PW < n ? w[(i / PW) * n + i % PW] : 0.0f;
    const bool back = t >= HALF; // dx, else dw
    const int mine  = t & (HALF - 1), turns = mine - lane >= k ? 0 : (k - (mine - lane) + HALF - 1) / HALF; // the warp's
    f32x2 reg[SLOTS][N / 2]; // of columns mine + HALF i: w, or sums
    float sum_b = 0.0f;
#pragma unroll
    for (int i = 0; i < SLOTS; ++i)
#pragma unroll
        for (int j = 0; j < N / 2; ++j) {
            const int c = mine + i * HALF;
            reg[i][j]   = back ? pack2(c < k && 2 * j < n ? w[(int64_t)c * n + 2 * j] : 0.0f, c < k && 2 * j + 1 < n ? w[(int64_t)c * n + 2 * j + 1] : 0.0f)
                               : (f32x2)0;
        }
    const int group = warp % GROUPS, quarter = warp / GROUPS;
    int at = 0;
    for (int64_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        asm volatile("cp.async.wait_group %0;" ::"n"(RING - 1) : "memory");
        __syncthreads();
        const float *rows_at = xs + at * ROWS * k;
        const int rows       = (int)(m - tile * ROWS < ROWS ? m - tile * ROWS : ROWS);
        // what d needs of this thread's row is on its way meanwhile
        const int64_t row = tile * ROWS + t / P;
        const bool slope  = t < ROWS * P && t / P < rows && t % P < n;
        const int64_t target = slope ? __ldg(targets + row) : -1;
        const float l = slope ? __ldg(lse + row) : 0.0f, by = slope && dloss ? __ldg(dloss + row) : 1.0f, add = slope && bias ? __ldg(bias + t % P) : 0.0f;
#pragma unroll 1
        for (int r0 = 0; r0 < 4; r0 += AT_ONCE) { // the logits' parts
            f32x2 acc[AT_ONCE][N / 2];
#pragma unroll
            for (int r = 0; r < AT_ONCE; ++r)
#pragma unroll
                for (int j = 0; j < N / 2; ++j)
                    acc[r][j] = 0;
            const float *from = rows_at + (group * 4 + r0) * k;
#pragma unroll 2
            for (int c = quarter * 32 + lane; c < k; c += 128) {
                f32x2 wv[P / 2];
#pragma unroll
                for (int j = 0; j < P / 4; ++j) {
                    const float4 q = *reinterpret_cast<const float4 *>(ws + c * PW + 4 * j);
                    wv[2 * j] = pack2(q.x, q.y), wv[2 * j + 1] = pack2(q.z, q.w);
                }
#pragma unroll
                for (int r = 0; r < AT_ONCE; ++r) {
                    const float v = from[r * k + c];
#pragma unroll
                    for (int j = 0; j < N / 2; ++j)
                        acc[r][j] = fma2(pack2(v, v), wv[j], acc[r][j]);
                }
            }
            constexpr int COUNT = (AT_ONCE * P + 15) / 16 * 16;
            float v[COUNT] = {};
#pragma unroll
            for (int r = 0; r < AT_ONCE; ++r)
#pragma unroll
                for (int j = 0; j < N / 2; ++j)
                    unpack2(acc[r][j], v[r * P + 2 * j], v[r * P + 2 * j + 1]);
            fused::sum_by_halves<COUNT>(v);
            if (!(lane & 1))
#pragma unroll
                for (int i = 0; i < COUNT / 16; ++i) {
                    const int which = (lane >> 1) * (COUNT / 16) + i;
                    if (which < AT_ONCE * P)
                        parts[(quarter * ROWS + group * 4 + r0) * P + which] = v[i];
                }
        }
        __syncthreads();
        if (t < ROWS * P) {
            const int j = t % P;
            float d     = 0.0f;
            if (slope) {
                float z = parts[t];
#pragma unroll
                for (int q = 1; q < 4; ++q)
                    z = __fadd_rn(z, parts[q * ROWS * P + t]);
                if (bias)
                    z = __fadd_rn(z, add);
                const float p  = expf(__fsub_rn(z, l));
                const bool has = target >= 0 && target < n;
                if (j == 0)
                    has_s[t / P] = has;
                if (has)
                    d = __fmul_rn(by, j == target ? __fsub_rn(p, 1.0f) : p);
            }
            ds[t] = d;
        }
        __syncthreads();
        if (t >= THREADS - 32 && lane < N) // a warp that has no more columns than another
            for (int r = 0; r < rows; ++r)
                sum_b = __fadd_rn(sum_b, ds[r * P + lane]);
        auto row_of = [&](int r, f32x2 (&d)[P / 2]) {
#pragma unroll
            for (int j = 0; j < P / 4; ++j) {
                const float4 q = *reinterpret_cast<const float4 *>(ds + r * P + 4 * j);
                d[2 * j] = pack2(q.x, q.y), d[2 * j + 1] = pack2(q.z, q.w);
            }
        };
        if (!back) {
#pragma unroll 2
            for (int r = 0; r < rows; ++r) {
                if (!has_s[r])
                    continue;
                f32x2 d[P / 2];
                row_of(r, d);
                const float *from = rows_at + r * k + mine; // beyond the last column: within shared memory, and of no use
#pragma unroll
                for (int i = 0; i < SLOTS; ++i) {
                    if (i >= turns)
                        break;
                    const float v = from[i * HALF];
#pragma unroll
                    for (int j = 0; j < N / 2; ++j)
                        reg[i][j] = fma2(pack2(v, v), d[j], reg[i][j]);
                }
            }
        } else if (dx) {
#pragma unroll 2
            for (int r = 0; r < rows; ++r) {
                f32x2 d[P / 2];
                row_of(r, d);
                float *to = dx + (tile * ROWS + r) * k + mine;
#pragma unroll
                for (int i = 0; i < SLOTS; ++i) {
                    if (i >= turns)
                        break;
                    f32x2 sum = 0;
#pragma unroll
                    for (int j = 0; j < N / 2; ++j)
                        sum = fma2(d[j], reg[i][j], sum);
                    float a, b;
                    unpack2(sum, a, b);
                    if (mine + i * HALF < k)
                        to[i * HALF] = __fadd_rn(a, b);
                }
            }
        }
        __syncthreads(); // all are through with the rows
        fetch(tile + (int64_t)RING * gridDim.x, at);
        at = at == RING - 1 ? 0 : at + 1;
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if (!partial)
        return;
    double *to = partial + (int64_t)blockIdx.x * ((int64_t)k * n + n);
    if (!back) {
#pragma unroll
        for (int i = 0; i < SLOTS; ++i)
#pragma unroll
            for (int j = 0; j < N / 2; ++j) {
                const int c = mine + i * HALF;
                float a, b;
                unpack2(reg[i][j], a, b);
                if (c < k && 2 * j < n)
                    to[(int64_t)c * n + 2 * j] = (double)a;
                if (c < k && 2 * j + 1 < n)
                    to[(int64_t)c * n + 2 * j + 1] = (double)b;
            }
    }
    if (t >= THREADS - 32 && lane < n)
        to[(int64_t)k * n + lane] = (double)sum_b;
}

bool ce_one_applicable(const float *x, int64_t k) { // n <= kFewClasses
    return k > 0 && k <= kOneColumns && (reinterpret_cast<uintptr_t>(x) & 15u) == 0;
}

template <int N, int RING, int THREADS>
ct_status launch_ce_one(
    const DeviceState *st, const float *x, const float *w, const float *bias, const int64_t *targets, const float *lse, const float *dloss, int64_t m,
    int64_t k, int64_t n, float *dx, float *dw, float *dbias) {
    constexpr int ROWS = THREADS / 32;
    const size_t smem  = (size_t)one_words(k, ROWS, (N + 3) / 4 * 4, RING) * 4;
    auto kernel        = ce_one_kernel<N, RING, THREADS>;
    static bool attr_set_dev[16] = {};
    if (!attr_set_dev[st->device & 15]) {
        CT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 224 * 1024));
        attr_set_dev[st->device & 15] = true;
    }
    const int64_t grid = blocks_for((m + ROWS - 1) / ROWS, (int64_t)st->sm_count * (512 / THREADS), kChainFew / ROWS), width = k * n + n;
    Scratch partial;
    if (dw || dbias)
        CT_TRY(partial.get((size_t)(grid * width) * 8));
    CT_CUDA(launch_dependent(kernel, dim3((unsigned)grid), dim3(THREADS), smem, stream(), x, w, bias, targets, lse, dloss, m, (int)k, (int)n, dx,
                             dw || dbias ? partial.as<double>() : nullptr));
    CT_LAUNCH_CHECK("ce_one");
    return dw || dbias ? fused::join_columns(partial.as<const double>(), grid, k * n, width, dw, dbias) : CT_OK;
}
// Two blocks of eight warps to an SM, whose phases overlap, where both fit: up to 8 classes, whose columns then fit the registers, in shared memory
// with two or three tiles of x, and enough rows to pay for as many blocks' beginnings (60000 x 785 x 8: 150 us with one, 135; 1000 x 785 x 10: 17
// with one, 25).  Else one of sixteen (60000 x 785 x 10: 160, as two 185).  N is classes rounded up; nine and ten have a form of their own,
// with a sixth fewer FMAs than that of twelve: 60000 x 785 x 10 166 so and 181, x 1024 x 10 189 and 203.
template <int N>
ct_status launch_ce_one_of(
    const DeviceState *st, const float *x, const float *w, const float *bias, const int64_t *targets, const float *lse, const float *dloss, int64_t m,
    int64_t k, int64_t n, float *dx, float *dw, float *dbias) {
    constexpr int64_t P = (N + 3) / 4 * 4, half = 112 * 1024 / 4;
    if constexpr (N <= 8) {
        const bool many = m >= (int64_t)st->sm_count * 64;
        if (many && one_words(k, 8, P, 3) <= half)
            return launch_ce_one<N, 3, 256>(st, x, w, bias, targets, lse, dloss, m, k, n, dx, dw, dbias);
        if (many && one_words(k, 8, P, 2) <= half)
            return launch_ce_one<N, 2, 256>(st, x, w, bias, targets, lse, dloss, m, k, n, dx, dw, dbias);
    }
    if constexpr (one_words(kOneColumns, 16, P, 3) > 2 * half) {
        if (one_words(k, 16, P, 3) > 2 * half)
            return launch_ce_one<N, 2, 512>(st, x, w, bias, targets, lse, dloss, m, k, n, dx, dw, dbias);
    }
    return launch_ce_one<N, 3, 512>(st, x, w, bias, targets, lse, dloss, m, k, n, dx, dw, dbias);
}

ct_status ce_few_grad(
    DeviceState *st, const float *x, const float *w, const float *bias, const int64_t *targets, const float *lse, const float *dloss, int64_t m, int64_t k,
    int64_t n, float *dx, float *dw, float *dbias) {
    if (ce_one_applicable(x, k)) {
        auto run = n <= 4 ? launch_ce_one_of<4> : n <= 8 ? launch_ce_one_of<8> : n <= 10 ? launch_ce_one_of<10> : n <= 12 ? launch_ce_one_of<12> : launch_ce_one_of<16>;
        return run(st, x, w, bias, targets, lse, dloss, m, k, n, dx, dw, dbias);
    }
    const int64_t blocks = (m + 255) / 256;
    fused::Parts parts;
    const size_t zp = parts.take((size_t)(m * n) * 4), pp = parts.take(dbias ? (size_t)(blocks * n) * 8 : 0);
    Scratch s;
    CT_TRY(s.get(parts.bytes));
    float *d = s.as<float>(zp);
    CT_TRY(few_logits(st, x, w, bias, m, k, n, d));
    CT_CUDA(launch_dependent(ce_few_slopes_kernel, dim3((unsigned)blocks), dim3(256), 0, stream(), d, targets, lse, dloss, m, (int)n,
                             dbias ? s.as<double>(pp) : nullptr));
    CT_LAUNCH_CHECK("ce_few_slopes");
    if (dbias)
        CT_TRY(fused::join_columns(s.as<const double>(pp), blocks, n, n, dbias, nullptr));
    if ((dw || dx) && k > 0) {
        const int64_t strips = (k + 255) / 256, parts = std::max((m + kChainFew - 1) / kChainFew, std::min<int64_t>((m + 63) / 64, (int64_t)st->sm_count * 4 / strips));
        Scratch sums;
        if (dw)
            CT_TRY(sums.get((size_t)(parts * k * n) * 8));
        auto back = n <= 4 ? ce_few_back_kernel<4> : n <= 8 ? ce_few_back_kernel<8> : n <= 12 ? ce_few_back_kernel<12> : ce_few_back_kernel<16>;
        CT_CUDA(launch_dependent(back, dim3((unsigned)(strips * parts)), dim3(256), 0, stream(), (const float *)d, x, w, targets, m, k, (int)n, strips,
                                 parts, dx, dw ? sums.as<double>() : nullptr));
        CT_LAUNCH_CHECK("ce_few_back");
        if (dw)
            CT_TRY(fused::join_columns(sums.as<const double>(), parts, k * n, k * n, dw, nullptr));
    }
    return CT_OK;
}

// Few rows: their logits are written.
struct LogitsStream {
    static constexpr bool kTwin = false;
    struct Params {
        const float *bias;
        float *out;
    };
    struct State {};
    __device__ static __forceinline__ void init(State &) {}
    template <int Q>
    __device__ static __forceinline__ void tile(const fused::Stream &p, const Params &e, State &, const float *z, int64_t c0, int cols, int t) {
        const int lane = t & 31, rows = p.m - 16 * Q < 16 ? p.m - 16 * Q : 16;
        for (int i = t >> 5; i < rows; i += fused::kStreamDrain) {
            const int r    = 16 * Q + i;
            const float rs = p.row_scale[r] * fused::kStreamUp;
#pragma unroll
            for (int c = lane; c < 128; c += 32)
                if (c < cols) {
                    const float v = __fmul_rn(z[i * fused::kStreamPitch + c], rs);
                    e.out[r * p.n + c0 + c] = e.bias ? __fadd_rn(v, __ldg(e.bias + c0 + c)) : v;
                }
        }
    }
    __device__ static __forceinline__ void finish(const fused::Stream &, const Params &, State &, float *, int) {}
};
ct_status few_rows_logits(DeviceState *st, const float *x, const float *w, const float *bias, int64_t m, int64_t k, int64_t n, float *z) {
    using namespace fused;
    if (takes_few_rows(m, n))
        return few_rows(st, x, w, bias, nullptr, nullptr, m, k, n, 0, z, nullptr, nullptr);
    const int64_t lk = padded(k);
    Parts parts;
    const size_t xp = parts.planes(m, lk), xi = parts.take((size_t)m * 4);
    Scratch s;
    CT_TRY(s.get(parts.bytes));
    const Planes px     = planes_at(s, xp, m, lk, lk);
    const Split operand = {x, nullptr, m, k, false, nullptr, px, s.as<float>(xi)};
    CT_TRY(split(st, &operand, 1));
    Stream p{};
    p.w = w, p.k = k, p.n = p.ld = n, p.row_scale = s.as<float>(xi);
    return launch_stream<LogitsStream>(st, px, p, LogitsStream::Params{bias, z}, "cross_entropy_grad", [](LogitsStream::Params f, int64_t) { return f; });
}

// Few rows: d of the logits.
struct FewSlopes {
    static constexpr int kMatrices = 1;
    const float *z, *lse, *dloss;
    const int64_t *targets;
    int64_t n;
    __device__ __forceinline__ bool has(int r) const { return targets[r] >= 0 && targets[r] < n; }
    __device__ __forceinline__ float at(int, int r, int64_t c) const {
        const float v = expf(__fsub_rn(z[r * n + c], lse[r]));
        return __fmul_rn(dloss ? dloss[r] : 1.0f, c == targets[r] ? __fsub_rn(v, 1.0f) : v);
    }
};
ct_status ce_few_rows_grad(
    DeviceState *st, const float *x, const float *w, const float *bias, const int64_t *targets, const float *lse, const float *dloss, int64_t m, int64_t k,
    int64_t n, float *dx, float *dw, float *dbias) {
    Scratch logits;
    CT_TRY(logits.get((size_t)(m * n) * 4));
    CT_TRY(few_rows_logits(st, x, w, bias, m, k, n, logits.as<float>()));
    fused::FewGrad p{};
    p.x = x, p.w[0] = w, p.dw[0] = dw, p.db[0] = dbias, p.dx = dx, p.k = k, p.n = n, p.m = (int)m;
    return fused::few_rows_grad(st, p, FewSlopes{logits.as<const float>(), lse, dloss, targets, n});
}

ct_status check_ce(const char *name, const void *x, const void *w, const void *targets, int64_t m, int64_t k, int64_t n) {
    if (m < 0 || k < 0 || n < 0)
        return fail(CT_ERR_INVALID, "%s: negative dimension", name);
    if (n == 0 && m > 0)
        return fail(CT_ERR_INVALID, "%s: no classes", name);
    if (m > fused::kMostSize || n > fused::kMostSize || k > fused::kMostSize)
        return fail(CT_ERR_TOO_LARGE, "%s: dimension too large", name);
    if (m > 0 && (!targets || (k > 0 && (!x || !w))))
        return fail(CT_ERR_INVALID, "%s: null pointer", name);
    return CT_OK;
}

// Rows whose logits are held at a time.
int64_t rows_at_once(int64_t m, int64_t n) { return std::max<int64_t>(1, std::min<int64_t>(m, (int64_t)(1u << 28) / n)); }

} // namespace
} // namespace ct

using namespace ct;

extern "C" {

ct_status ct_dense_cross_entropy(
    const float *x, const float *w, const float *bias, const int64_t *targets, int64_t m, int64_t k, int64_t n, float *loss, float *lse) {
    OpLock op_lock;
    DeviceState *st;
    CT_TRY(current(&st));
    CT_TRY(check_ce("dense_cross_entropy", x, w, targets, m, k, n));
    if (m == 0)
        return CT_OK;
    ProfScope prof("cross_entropy");
    const bool fused_form = n > kFewClasses && k > 0 && ct_get_precision() == CT_PREC_3XTF32;
    if (fused_form && !fused::takes_few_rows(m, n))
        return ce_fused(st, x, w, bias, targets, m, k, n, loss, lse);
    const int64_t piece = n <= kFewClasses ? m : rows_at_once(m, n);
    const int64_t slots = (n + kPartLogits - 1) / kPartLogits;
    Scratch logits, parts;
    CT_TRY(logits.get((size_t)(piece * n) * 4));
    if (slots > 2)
        CT_TRY(parts.get((size_t)(slots * piece) * 8 + (size_t)piece * 4));
    if (n <= kFewClasses) {
        CT_TRY(few_logits(st, x, w, bias, m, k, n, logits.as<float>()));
        CT_CUDA(launch_dependent(ce_few_kernel, dim3((unsigned)((m + 255) / 256)), dim3(256), 0, stream(), logits.as<const float>(), targets, m, (int)n,
                                 loss, lse));
        CT_LAUNCH_CHECK("ce_few");
        return CT_OK;
    }
    for (int64_t r = 0; r < m; r += piece) {
        const int64_t rows = std::min(piece, m - r);
        if (fused_form)
            CT_TRY(fused::few_rows(st, x + r * k, w, bias, nullptr, nullptr, rows, k, n, 0, logits.as<float>(), nullptr, nullptr));
        else
            CT_TRY(ct_dense(x + r * k, w, bias, rows, k, n, CT_ACT_NONE, logits.as<float>(), nullptr));
        if (slots > 2) {
            float2 *part     = parts.as<float2>();
            float *at_target = parts.as<float>((size_t)(slots * piece) * 8);
            CT_CUDA(launch_dependent(ce_parts_kernel, dim3((unsigned)slots, (unsigned)rows), dim3(256), 0, stream(), logits.as<const float>(), targets + r, rows,
                                     n, part, at_target));
            CT_LAUNCH_CHECK("ce_parts");
            CT_CUDA(launch_dependent(ce_join_kernel, dim3((unsigned)((rows + 7) / 8)), dim3(256), 0, stream(), (const float2 *)part, (int)slots,
                                     (const float *)at_target, targets + r, rows, n, loss ? loss + r : nullptr, lse ? lse + r : nullptr,
                                     (const uint32_t *)st->flags_dev));
            CT_LAUNCH_CHECK("ce_join");
            continue;
        }
        CT_CUDA(launch_dependent(ce_rows_kernel, dim3((unsigned)rows), dim3(256), 0, stream(), logits.as<const float>(), targets + r, n,
                                 loss ? loss + r : nullptr, lse ? lse + r : nullptr));
        CT_LAUNCH_CHECK("ce_rows");
    }
    return CT_OK;
}

ct_status ct_dense_cross_entropy_grad(
    const float *x, const float *w, const float *bias, const int64_t *targets, const float *lse, const float *dloss, int64_t m, int64_t k, int64_t n,
    float *dx, float *dw, float *dbias) {
    OpLock op_lock;
    DeviceState *st;
    CT_TRY(current(&st));
    CT_TRY(check_ce("dense_cross_entropy_grad", x, w, targets, m, k, n));
    if (m > 0 && !lse)
        return fail(CT_ERR_INVALID, "dense_cross_entropy_grad: null pointer");
    if (m == 0) { // sums of nothing
        if (dw && k * n > 0)
            CT_CUDA(cudaMemsetAsync(dw, 0, (size_t)(k * n) * 4, stream()));
        if (dbias && n > 0)
            CT_CUDA(cudaMemsetAsync(dbias, 0, (size_t)n * 4, stream()));
        return CT_OK;
    }
    ProfScope prof("cross_entropy_grad");
    if (m <= fused::kFewRows && m * n <= (int64_t)1 << 28 && k > 0 && ct_get_precision() == CT_PREC_3XTF32 && (dx || dw || dbias))
        return ce_few_rows_grad(st, x, w, bias, targets, lse, dloss, m, k, n, dx, dw, dbias);
    if (n > kFewClasses && k > 0 && ct_get_precision() == CT_PREC_3XTF32)
        return ce_grad_fused(st, x, w, bias, targets, lse, dloss, m, k, n, dx, dw, dbias);
    if (n <= kFewClasses)
        return ce_few_grad(st, x, w, bias, targets, lse, dloss, m, k, n, dx, dw, dbias);
    const int64_t piece = rows_at_once(m, n);
    Scratch logits, turned, sums, kept;
    CT_TRY(logits.get((size_t)(piece * n) * 4));
    float *d = logits.as<float>();
    if (dx && k > 0) {
        CT_TRY(turned.get((size_t)(k * n) * 4));
        CT_TRY(ct_transpose(CT_F32, w, k, n, turned.as<float>()));
    }
    if (dw && k > 0)
        CT_TRY(kept.get((size_t)(piece * k) * 4));
    if (piece < m)
        CT_TRY(sums.get((size_t)(k * n + n) * 4));
    for (int64_t r = 0; r < m; r += piece) {
        const int64_t rows = std::min(piece, m - r);
        CT_TRY(ct_dense(x + r * k, w, bias, rows, k, n, CT_ACT_NONE, d, nullptr));
        const int64_t count = rows * n;
        CT_CUDA(launch_dependent(ce_slopes_kernel, dim3((unsigned)std::min<int64_t>((count + 255) / 256, (int64_t)st->sm_count * 16)), dim3(256), 0,
                                 stream(), d, targets + r, lse + r, dloss ? dloss + r : nullptr, count, n));
        CT_LAUNCH_CHECK("ce_slopes");
        if (dx && k > 0)
            CT_TRY(ct_matmul(CT_F32, d, CT_F32, turned.as<float>(), rows, n, k, dx + r * k));
        if (dw && k > 0) {
            CT_CUDA(launch_dependent(ce_rows_with_target_kernel, dim3((unsigned)std::min<int64_t>((rows * k + 255) / 256, (int64_t)st->sm_count * 16)),
                                     dim3(256), 0, stream(), x + r * k, targets + r, rows * k, k, n, kept.as<float>()));
            CT_LAUNCH_CHECK("ce_rows_with_target");
            CT_TRY(ct_matmul_tn(kept.as<const float>(), d, k, rows, n, r ? sums.as<float>() : dw));
            if (r)
                CT_TRY(ct_binary(CT_ADD, CT_F32, dw, CT_F32, sums.as<float>(), (uint64_t)(k * n), dw));
        }
        if (dbias) {
            float *to = r ? sums.as<float>() + k * n : dbias;
            CT_TRY(ct_sum_axis(CT_F32, d, rows, n, 0, to));
            if (r)
                CT_TRY(ct_binary(CT_ADD, CT_F32, dbias, CT_F32, to, (uint64_t)n, dbias));
        }
    }
    return CT_OK;
}

} // extern "C"
