// Distillation from the classes that a teacher thinks likeliest, and its gradient.
//
//   p = softmax(teacher / T) over a row's entries, q = softmax(z / T) over its classes
//   loss = T^2 sum p (log p - log q),  dz[c] = dloss T (q[c] - the sum of p over the entries of class c)
//
// Both are bound by memory: the logits are read once (4 bytes each), and on the way back written once (8).  Forward, a thread keeps a
// logit near the largest of its own and the sum of exponentials about it, which meet at the end; a row of a small batch is shared by the blocks of a cluster.
// Backward, lse is given: a row is q times a factor, from which its block takes the entries' p where it has written them.
// Measured (L2 flushed): 4096 x 131072 with 64 entries 318 us (2.15 GB, 1.03 of a copy), 64 x 32003 5.7 us; gradient 4096 x 50257 259 us (1.65 GB, 0.97),
// 60000 x 10 6.9 us (9 MB: a launch and a round of loads).  Rows of 33 to 8000 classes are further from a copy: 60000 x 128 15 us in line (46 MB, 0.48), x 1500 76
// (375 MB, 0.75), backward 21 (77 MB, 0.56) and 117 (735 MB, 0.96): a row's loads, its lanes' join and its entries come one after the other, and nothing of the next meanwhile.
// Times at the rules below are of a lone call between two events, L2 flushed, with the events' own 4 us or so, unless in line is said: call behind call.
#include "common.cuh"
#include "tc_ptx.cuh"

#include <algorithm>
#include <initializer_list>

namespace ct {
namespace {

using namespace ptx;

constexpr int kMostEntries = 1024;
constexpr float kLog2e     = 1.44269502162933349609375f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A logit that is the largest of some or near it, and the sum of exp((z - top) / T) over them; a NaN or +infinity among them shows in the sum.
struct Sum {
    float top, sum;
};
__device__ __forceinline__ float about(float top) { return top == -INFINITY ? 0.0f : top; } // classes that are out leave a sum of 0
__device__ __forceinline__ Sum join(Sum a, Sum b, float c) {
    const float top = fmaxf(a.top, b.top), base = about(top);
    // one of the two exponentials is 1; of an empty side 0
    return {top, __fadd_rn(__fmul_rn(a.sum, ex2(__fmul_rn(__fsub_rn(a.top, base), c))), __fmul_rn(b.sum, ex2(__fmul_rn(__fsub_rn(b.top, base), c))))};
}
template <int N> __device__ __forceinline__ float sum_about(const float (&z)[N], float base, float c) {
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < N; ++i)
        sum[i & 3] = __fadd_rn(sum[i & 3], ex2(__fmul_rn(__fsub_rn(z[i], base), c)));
    return __fadd_rn(__fadd_rn(sum[0], sum[1]), __fadd_rn(sum[2], sum[3]));
}
// N more logits
template <int N> __device__ __forceinline__ void take(Sum &s, const float (&z)[N], float c) {
    float top = s.top;
#pragma unroll
    for (int i = 0; i < N; ++i)
        top = fmaxf(top, z[i]);
    const float base = about(top);
    s.sum            = __fmaf_rn(s.sum, ex2(__fmul_rn(__fsub_rn(s.top, base), c)), sum_about(z, base, c));
    s.top            = top;
}
template <int TPR> __device__ __forceinline__ Sum join_lanes(Sum s, float c) {
#pragma unroll
    for (int o = TPR / 2; o; o >>= 1)
        s = join(s, {__shfl_xor_sync(0xffffffffu, s.top, o), __shfl_xor_sync(0xffffffffu, s.sum, o)}, c);
    return s;
}
template <int TPR> __device__ __forceinline__ float max_lanes(float v) {
#pragma unroll
    for (int o = TPR / 2; o; o >>= 1)
        v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
template <int TPR> __device__ __forceinline__ float sum_lanes(float v) {
#pragma unroll
    for (int o = TPR / 2; o; o >>= 1)
        v = __fadd_rn(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// The entries' weights are p[j] = exp((teacher[j] - top) / T) / sum.
struct Weights {
    float top, sum;
    bool some; // whether there is any entry
};
__device__ __forceinline__ bool class_of(int64_t id, int64_t n) { return id >= 0 && id < n; }
// An entry of weight 0 is none: a row of nothing else is one without entries.
__device__ __forceinline__ bool entry_of(int64_t id, int64_t n, float teacher) { return class_of(id, n) && teacher != -INFINITY; }
__device__ __forceinline__ float lse_of(Sum s, float temperature) { return __fadd_rn(__fdiv_rn(about(s.top), temperature), logf(s.sum)); }
// The loss over T^2, sum p (log p - log q), cancels where p is near q, and T^2 is large just where the cancelling is worst: both distributions are flat then.
// So log p - log q of an entry is x - y + log(the classes' sum / the weights'), x = (teacher - its top) / T and y = (z - top) / T, in which
// logits' common offsets are gone (z / T - lse would round them), and rows whose sum is below kSmall at temperatures above kWarm are taken again in 64 bits.  What is
// left is off by T^2 times some 2^-20 (both sums' exponentials, 2^-22 each, and their arguments), 2^-16 at kWarm, and 2^-16 of a sum above kSmall.  (60000 rows of 10
// classes, all of them entries, T = 8: 17 us in line so, 9 in 32 bits; 300 of 1000 14 and 11.)
constexpr float kWarm = 4.0f, kSmall = 1.0f / 16.0f;
struct Ratio {
    float inv_sum, log; // 1 / the weights' sum; the logarithm of the classes' sum over it
};
__device__ __forceinline__ Ratio ratio_of(const Weights &w, const Sum &s) { return {__fdiv_rn(1.0f, w.sum), logf(__fdiv_rn(s.sum, w.sum))}; }
__device__ __forceinline__ float divergence(float u, float z, const Weights &w, const Sum &s, const Ratio &r, float inv_t) {
    const float x = __fsub_rn(u, w.top), p = __fmul_rn(expf(__fmul_rn(x, inv_t)), r.inv_sum);
    return p == 0.0f ? 0.0f : __fmul_rn(p, __fadd_rn(__fmul_rn(__fsub_rn(x, __fsub_rn(z, about(s.top))), inv_t), r.log)); // 0 log 0 is 0
}
__device__ __forceinline__ bool again_wide(float sum, float temperature) { return temperature > kWarm && sum < kSmall; }
__device__ __forceinline__ float loss_from(float sum, float temperature) { return __fmul_rn(__fmul_rn(temperature, temperature), sum); }

// In 64 bits: of the classes' exponentials, of the weights, and of these times x - y; one thread's part of those of `threads`.
struct Wide {
    double classes, weights, cross;
    __device__ __forceinline__ void add(const Wide &o) { classes += o.classes, weights += o.weights, cross += o.cross; }
    template <int TPR> __device__ __forceinline__ void add_lanes() {
#pragma unroll
        for (int o = TPR / 2; o; o >>= 1) {
            Wide b;
            b.classes = __shfl_xor_sync(0xffffffffu, classes, o), b.weights = __shfl_xor_sync(0xffffffffu, weights, o);
            b.cross = __shfl_xor_sync(0xffffffffu, cross, o);
            add(b);
        }
    }
    __device__ __forceinline__ float loss(float temperature) const {
        return (float)((double)temperature * (double)temperature * (cross / weights + log(classes / weights)));
    }
};
__device__ __forceinline__ Wide wide_sums(
    const float *src, int64_t n, float z_top, const int64_t *__restrict__ ids, const float *__restrict__ teacher, int top, float u_top, float temperature, int t,
    int threads) {
    const double inv_t = 1.0 / (double)temperature;
    Wide s = {0.0, 0.0, 0.0};
#pragma unroll 1
    for (int64_t i = t; i < n; i += threads)
        s.classes += exp(((double)src[i] - (double)z_top) * inv_t);
#pragma unroll 1
    for (int j = t; j < top; j += threads) {
        const int64_t id = ids[j];
        if (!class_of(id, n))
            continue;
        const double x = ((double)teacher[j] - (double)u_top) * inv_t, e = exp(x);
        if ((float)e > 0.0f) { // as in 32 bits, an entry of no weight adds nothing
            s.weights += e;
            s.cross += e * (x - ((double)src[id] - (double)z_top) * inv_t);
        }
    }
    return s;
}
// The lse of a row; of one whose classes are all out, there is no distribution.
__device__ __forceinline__ float lse_given(float lse) { return lse == -INFINITY ? NAN : lse; }
// exp(z / T - lse) of a logit: 1 / T in two parts.  -infinity becomes a number, which neither part makes a NaN.
__device__ __forceinline__ float probability(float z, float inv_t, float inv_t_rest, float lse) {
    asm("max.NaN.f32 %0, %0, 0fFF7FFFFF;" : "+f"(z));
    return ex2(__fmul_rn(__fmaf_rn(z, inv_t, __fmaf_rn(z, inv_t_rest, -lse)), kLog2e));
}

// A row's entries in the registers of its TPR threads, E each: entry e TPR + t; none: -1.  All loads are on their way before one is looked at.
template <int TPR, int E> struct Entries {
    int id[E];
    float u[E];
    __device__ __forceinline__ Entries(const int64_t *__restrict__ ids, const float *__restrict__ teacher, int top, int64_t n, bool here, int t) {
        int64_t wide[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int j = max(min(e * TPR + t, top - 1), 0);
            wide[e]     = here && top > 0 ? ids[j] : -1;
            u[e]        = here && top > 0 ? teacher[j] : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < E; ++e)
            id[e] = e * TPR + t < top && entry_of(wide[e], n, u[e]) ? (int)wide[e] : -1;
    }
    __device__ __forceinline__ Weights weights(float inv_t) const {
        float most = -INFINITY, sum = 0.0f;
        bool some = false;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (id[e] >= 0) {
                some = true;
                most = fmaxf(most, u[e]);
                sum  = u[e] != u[e] ? NAN : sum; // (fmaxf passes over it)
            }
        most             = max_lanes<TPR>(most);
        const float base = about(most);
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (id[e] >= 0)
                sum = __fadd_rn(sum, expf(__fmul_rn(__fsub_rn(u[e], base), inv_t)));
        const unsigned group = TPR == 32 ? 0xffffffffu : ((1u << (TPR & 31)) - 1) << ((threadIdx.x & 31) / TPR * TPR);
        return {base, sum_lanes<TPR>(sum), (__ballot_sync(0xffffffffu, some) & group) != 0};
    }
};

// src, ids and teacher are those of the row; lanes whose row is not `here` go along.
template <int TPR, int E>
__device__ __forceinline__ float loss_of(
    const Entries<TPR, E> &entries, const float (&z)[E], const Sum &s, const float *src, int64_t n, const int64_t *__restrict__ ids,
    const float *__restrict__ teacher, int top, float temperature, float inv_t, bool here, int t) {
    const Weights w = entries.weights(inv_t);
    const Ratio r   = ratio_of(w, s);
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e)
        if (entries.id[e] >= 0)
            sum = __fadd_rn(sum, divergence(entries.u[e], z[e], w, s, r, inv_t));
    sum              = sum_lanes<TPR>(sum);
    float loss       = loss_from(sum, temperature);
    const bool again = here && w.some && again_wide(sum, temperature);
    if (__any_sync(0xffffffffu, again)) {
        Wide wide = {0.0, 0.0, 0.0};
        if (again)
            wide = wide_sums(src, n, s.top, ids, teacher, top, w.top, temperature, t, TPR);
        wide.add_lanes<TPR>();
        loss = again ? wide.loss(temperature) : loss;
    }
    return w.some ? loss : 0.0f;
}

// ---- rows of few classes: TPR threads to a row, V of its logits in each ---------------------------

template <int TPR, int V, int E>
__global__ void __launch_bounds__(256) distill_short_kernel(
    const float *__restrict__ logits, const int64_t *__restrict__ ids, const float *__restrict__ teacher, int64_t m, int n, int top, float temperature,
    float inv_t, float *__restrict__ loss, float *__restrict__ lse, int early) {
    griddep_wait();
    if (early)
        griddep_launch_dependents();
    const int t       = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    const bool here   = row < m; // the others go along
    const float c     = __fmul_rn(inv_t, kLog2e);
    const float *src  = logits + (here ? row * n : 0);
    const Entries<TPR, E> entries(ids + (here ? row * top : 0), teacher + (here ? row * top : 0), loss ? top : 0, n, here, t);
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i)
        z[i] = here ? src[min(i * TPR + t, n - 1)] : 0.0f;
    float at[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
        at[e] = entries.id[e] >= 0 ? src[entries.id[e]] : 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i)
        z[i] = i * TPR + t < n ? z[i] : -INFINITY;
    Sum s = {-INFINITY, 0.0f};
    take(s, z, c);
    s = join_lanes<TPR>(s, c);
    if (loss) {
        const float value = loss_of(entries, at, s, src, n, ids + (here ? row * top : 0), teacher + (here ? row * top : 0), top, temperature, inv_t, here, t);
        if (here && t == 0)
            loss[row] = value;
    }
    if (lse && here && t == 0)
        lse[row] = lse_of(s, temperature);
}

// Takes the entries' weights off a row that the TPR threads have written, memory that they share: TPR entries after another, of which the first of a class
// takes off the weights of all.
template <int TPR, int E>
__device__ __forceinline__ void take_off(const Entries<TPR, E> &entries, const Weights &w, float inv_t, float by, int top, int t, float *row) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
        if (e * TPR >= top)
            break;
        const float p = expf(__fmul_rn(__fsub_rn(entries.u[e], w.top), inv_t));
        float total   = 0.0f;
        bool first    = entries.id[e] >= 0;
        for (int o = 0; o < min(TPR, top - e * TPR); ++o) {
            const int id    = __shfl_sync(0xffffffffu, entries.id[e], o, TPR);
            const float one = __shfl_sync(0xffffffffu, p, o, TPR);
            if (id == entries.id[e])
                total = __fadd_rn(total, one), first &= o >= t;
        }
        if (first)
            row[entries.id[e]] = __fmaf_rn(-total, by, row[entries.id[e]]);
        __syncwarp();
    }
}

// Rows lie in shared memory while their entries' weights are taken off.
template <int TPR, int V, int E>
__global__ void __launch_bounds__(256) distill_grad_short_kernel(
    const float *logits, const int64_t *__restrict__ ids, const float *__restrict__ teacher, const float *__restrict__ lse,
    const float *__restrict__ dloss, int64_t m, int n, int top, float temperature, float inv_t, float inv_t_rest, float *dlogits) {
    __shared__ float rows[256 / TPR][TPR * V];
    griddep_wait();
    const int t       = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    const bool here   = row < m;
    const float *src  = logits + (here ? row * n : 0);
    float *dst        = dlogits + (here ? row * n : 0);
    float *mine       = rows[threadIdx.x / TPR];
    const Entries<TPR, E> entries(ids + (here ? row * top : 0), teacher + (here ? row * top : 0), top, n, here, t);
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i)
        z[i] = here ? src[min(i * TPR + t, n - 1)] : 0.0f;
    const float l = here ? lse_given(lse[row]) : 0.0f, given = here && dloss ? dloss[row] : 1.0f, scale = __fmul_rn(given, temperature);
    const Weights w = entries.weights(inv_t);
#pragma unroll
    for (int i = 0; i < V; ++i)
        mine[i * TPR + t] = w.some ? __fmul_rn(probability(z[i], inv_t, inv_t_rest, l), scale) : 0.0f;
    __syncwarp();
    take_off(entries, w, inv_t, __fdiv_rn(scale, w.sum), top, t, mine);
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (here && i * TPR + t < n)
            dst[i * TPR + t] = mine[i * TPR + t];
}

// ---- longer rows: a block to a row, or to a part of one -------------------------------------------

// 16-byte pieces of a stretch of floats at any address, from a multiple of 128 bytes on: `head` values before the first, and `tail` behind the last.
struct Stretch {
    int head, pieces, tail;
};
__device__ __forceinline__ Stretch stretch_of(const float *p, int64_t count) {
    Stretch s;
    s.head   = (int)min((int64_t)((32 - ((reinterpret_cast<uintptr_t>(p) >> 2) & 31)) & 31), count);
    s.pieces = ((int)count - s.head) / 4;
    s.tail   = (int)count - s.head - 4 * s.pieces;
    return s;
}

constexpr int kThreads = 256, kAtOnce = 4; // pieces of a thread that are on their way together

// Loads without conditions (with them each would wait for the one before): the last piece again.
template <int THREADS> __device__ __forceinline__ void load_pieces(float4 (&z)[kAtOnce], const float4 *from, int i, int pieces) {
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u)
        z[u] = from[min(i + u * THREADS, pieces - 1)];
}
// The sum of a stretch by THREADS threads; z: its first pieces, on their way.  A thread adds up its turns, of 16 logits, in 64 bits, about a logit that moves only
// when one 256 times as likely comes: a move is off by 2^-22, and four of them leave nothing of what was before.  (In 32 bits and about the largest so far, lse of 2^27
// logits that rise little by little was off by 6e-5, and now by a rounding.)
template <int THREADS>
__device__ __forceinline__ Sum sum_stretch(const float *src, const Stretch &st, float4 (&f)[kAtOnce], float c, int t) {
    const float *body = src + st.head;
    Sum s             = {-INFINITY, 0.0f};
    for (int i = t; i < st.head + st.tail; i += THREADS) {
        const float z[1] = {i < st.head ? src[i] : body[4 * st.pieces + i - st.head]};
        take(s, z, c);
    }
    const float reach = __fdiv_rn(8.0f, c);
    double sum        = (double)s.sum;
    for (int i = t; i < st.pieces;) {
        float z[4 * kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            const bool in = i + u * THREADS < st.pieces;
            z[4 * u] = in ? f[u].x : -INFINITY, z[4 * u + 1] = in ? f[u].y : -INFINITY;
            z[4 * u + 2] = in ? f[u].z : -INFINITY, z[4 * u + 3] = in ? f[u].w : -INFINITY;
        }
        i += THREADS * kAtOnce;
        if (i < st.pieces)
            load_pieces<THREADS>(f, reinterpret_cast<const float4 *>(body), i, st.pieces);
        float top = z[0];
#pragma unroll
        for (int q = 1; q < 4 * kAtOnce; ++q)
            top = fmaxf(top, z[q]);
        top              = top > __fadd_rn(s.top, reach) ? top : s.top;
        const float base = about(top), part = sum_about(z, base, c);
        sum   = fma(sum, (double)ex2(__fmul_rn(__fsub_rn(s.top, base), c)), (double)part);
        s.top = top;
    }
    s.sum = (float)sum;
    return s;
}
// f(z) of each logit of a stretch, written to a row that lies as far from 16 bytes (VEC), or at any address.
template <int THREADS, bool VEC, typename F>
__device__ __forceinline__ void map_stretch(const float *src, float *dst, int64_t count, const Stretch &st, float4 (&z)[kAtOnce], int t, F &&f) {
    if (VEC) {
        for (int q = t; q < st.head + st.tail; q += THREADS) {
            const int i = q < st.head ? q : st.pieces * 4 + q;
            dst[i]          = f(src[i]);
        }
        const float4 *from = reinterpret_cast<const float4 *>(src + st.head);
        float4 *to         = reinterpret_cast<float4 *>(dst + st.head);
        for (int i = t; i < st.pieces;) {
            float4 d[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
                d[u] = make_float4(f(z[u].x), f(z[u].y), f(z[u].z), f(z[u].w));
            const int now = i;
            i += THREADS * kAtOnce;
            if (i < st.pieces)
                load_pieces<THREADS>(z, from, i, st.pieces);
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
                if (now + u * THREADS < st.pieces)
                    to[now + u * THREADS] = d[u];
        }
    } else {
        for (int64_t i = t; i < count; i += THREADS * kAtOnce) {
            float v[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
                v[u] = src[min(i + u * THREADS, count - 1)];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
                if (i + u * THREADS < count)
                    dst[i + u * THREADS] = f(v[u]);
        }
    }
}

// Many rows: a warp to each.
constexpr int kWarpEntries = 128;
__global__ void __launch_bounds__(kThreads) distill_warp_kernel(
    const float *__restrict__ logits, const int64_t *__restrict__ ids, const float *__restrict__ teacher, int64_t m, int64_t n, int top, float temperature,
    float inv_t, float *__restrict__ loss, float *__restrict__ lse, int early) {
    griddep_wait();
    if (early)
        griddep_launch_dependents();
    const int lane    = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    if (row >= m)
        return;
    const float c    = __fmul_rn(inv_t, kLog2e);
    const float *src = logits + row * n;
    const Stretch st = stretch_of(src, n);
    float4 f[kAtOnce];
    if (lane < st.pieces)
        load_pieces<32>(f, reinterpret_cast<const float4 *>(src + st.head), lane, st.pieces);
    constexpr int E = kWarpEntries / 32;
    const Entries<32, E> entries(ids + row * top, teacher + row * top, loss ? top : 0, n, true, lane);
    float at[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
        at[e] = entries.id[e] >= 0 ? src[entries.id[e]] : 0.0f;
    const Sum s = join_lanes<32>(sum_stretch<32>(src, st, f, c, lane), c);
    if (loss) {
        const float value = loss_of(entries, at, s, src, n, ids + row * top, teacher + row * top, top, temperature, inv_t, true, lane);
        if (lane == 0)
            loss[row] = value;
    }
    if (lse && lane == 0)
        lse[row] = lse_of(s, temperature);
}

template <bool VEC>
__global__ void __launch_bounds__(kThreads) distill_grad_warp_kernel(
    const float *logits, const int64_t *__restrict__ ids, const float *__restrict__ teacher, const float *__restrict__ lse,
    const float *__restrict__ dloss, int64_t m, int64_t n, int top, float temperature, float inv_t, float inv_t_rest, float *dlogits) {
    griddep_wait();
    const int lane    = threadIdx.x & 31;
    const int64_t row = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    if (row >= m)
        return;
    const float *src = logits + row * n;
    float *dst       = dlogits + row * n;
    const Stretch st = VEC ? stretch_of(src, n) : Stretch{0, 0, 0};
    float4 z[kAtOnce];
    if (lane < st.pieces)
        load_pieces<32>(z, reinterpret_cast<const float4 *>(src + st.head), lane, st.pieces);
    const Entries<32, kWarpEntries / 32> entries(ids + row * top, teacher + row * top, top, n, true, lane);
    const float l = lse_given(lse[row]), scale = __fmul_rn(dloss ? dloss[row] : 1.0f, temperature);
    const Weights w = entries.weights(inv_t);
    map_stretch<32, VEC>(src, dst, n, st, z, lane, [&](float v) { return w.some ? __fmul_rn(probability(v, inv_t, inv_t_rest, l), scale) : 0.0f; });
    __syncwarp();
    if (w.some)
        take_off(entries, w, inv_t, __fdiv_rn(scale, w.sum), top, lane, dst);
}

// The entries of a row in shared memory; the sum of weights is left to one warp.
struct SharedEntries {
    float u[kMostEntries];
    int id[kMostEntries]; // none: -1
};
__device__ __forceinline__ Weights weights_of(const SharedEntries &s, int top, float inv_t, int lane) {
    float most = -INFINITY, sum = 0.0f;
    bool some = false;
    for (int j = lane; j < top; j += 32)
        if (s.id[j] >= 0) {
            some = true;
            most = fmaxf(most, s.u[j]);
            sum  = s.u[j] != s.u[j] ? NAN : sum;
        }
    most             = max_lanes<32>(most);
    const float base = about(most);
    for (int j = lane; j < top; j += 32)
        if (s.id[j] >= 0)
            sum = __fadd_rn(sum, expf(__fmul_rn(__fsub_rn(s.u[j], base), inv_t)));
    return {base, sum_lanes<32>(sum), __any_sync(0xffffffffu, some) != 0};
}

__global__ void __launch_bounds__(kThreads) distill_kernel(
    const float *__restrict__ logits, const int64_t *__restrict__ ids, const float *__restrict__ teacher, int64_t n, int top, float temperature,
    float inv_t, int parts, int64_t part, float *__restrict__ loss, float *__restrict__ lse, int early) {
    __shared__ SharedEntries entries;
    __shared__ float entry_z[kMostEntries];
    __shared__ Sum warps[kThreads / 32], blocks[8];
    __shared__ Wide wide[kThreads / 32];
    __shared__ float z_top, u_top;
    __shared__ bool again;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const uint32_t rank = parts > 1 ? cluster_rank() : 0;
    if (parts > 1)
        cluster_sync(); // every block of the cluster runs before another writes into its memory
    griddep_wait();
    if (early)
        griddep_launch_dependents();
    const int64_t row = blockIdx.x / parts;
    const float c     = __fmul_rn(inv_t, kLog2e);
    const float *src  = logits + row * n;
    const int64_t c0 = min(rank * part, n), count = min(part, n - c0);
    const Stretch st  = stretch_of(src + c0, count);
    float4 f[kAtOnce];
    if (t < st.pieces)
        load_pieces<kThreads>(f, reinterpret_cast<const float4 *>(src + c0 + st.head), t, st.pieces); // on its way while the entries are fetched
    if (rank == 0 && loss)
        for (int j = t; j < top; j += kThreads) {
            const int64_t id = ids[row * top + j];
            const float u    = teacher[row * top + j];
            entries.u[j]     = u;
            entries.id[j]    = entry_of(id, n, u) ? (int)id : -1;
            entry_z[j]       = class_of(id, n) ? src[id] : 0.0f;
        }
    Sum s = sum_stretch<kThreads>(src + c0, st, f, c, t);
    s = join_lanes<32>(s, c);
    if (lane == 0)
        warps[warp] = s;
    __syncthreads();
    if (warp == 0) {
        s = lane < kThreads / 32 ? warps[lane] : Sum{-INFINITY, 0.0f};
        s = join_lanes<32>(s, c);
    }
    if (parts > 1) {
        if (t == 0)
            asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(mapa(static_cast<uint32_t>(__cvta_generic_to_shared(&blocks[rank])), 0)), "f"(s.top),
                         "f"(s.sum)
                         : "memory");
        cluster_sync();
        if (rank == 0 && warp == 0) {
            s = lane < parts ? blocks[lane] : Sum{-INFINITY, 0.0f};
            s = join_lanes<32>(s, c);
        }
    }
    if (rank != 0)
        return;
    if (warp == 0) {
        if (loss) {
            const Weights w = weights_of(entries, top, inv_t, lane);
            const Ratio r   = ratio_of(w, s);
            float sum = 0.0f;
            for (int j = lane; j < top; j += 32)
                if (entries.id[j] >= 0)
                    sum = __fadd_rn(sum, divergence(entries.u[j], entry_z[j], w, s, r, inv_t));
            sum = sum_lanes<32>(sum);
            if (lane == 0) {
                loss[row] = w.some ? loss_from(sum, temperature) : 0.0f;
                z_top = s.top, u_top = w.top, again = w.some && again_wide(sum, temperature);
            }
        }
        if (lse && lane == 0)
            lse[row] = lse_of(s, temperature);
    }
    if (!loss || !(temperature > kWarm))
        return;
    __syncthreads();
    if (!again)
        return;
    Wide sums = wide_sums(src, n, z_top, ids + row * top, teacher + row * top, top, u_top, temperature, t, kThreads);
    sums.add_lanes<32>();
    if (lane == 0)
        wide[warp] = sums;
    __syncthreads();
    if (t == 0) {
        for (int w = 1; w < kThreads / 32; ++w)
            sums.add(wide[w]);
        loss[row] = sums.loss(temperature);
    }
}

template <bool VEC>
__global__ void __launch_bounds__(kThreads) distill_grad_kernel(
    const float *logits, const int64_t *__restrict__ ids, const float *__restrict__ teacher, const float *__restrict__ lse,
    const float *__restrict__ dloss, int64_t n, int top, float temperature, float inv_t, float inv_t_rest, int parts, int64_t part, float *dlogits) {
    __shared__ SharedEntries entries;
    griddep_wait();
    const int t       = threadIdx.x;
    const int64_t row = blockIdx.x / parts, c0 = min((int64_t)(blockIdx.x % parts) * part, n), count = min(part, n - c0);
    const float *src  = logits + row * n + c0;
    float *dst        = dlogits + row * n + c0;
    const Stretch st  = VEC ? stretch_of(src, count) : Stretch{0, 0, 0};
    float4 z[kAtOnce];
    if (t < st.pieces)
        load_pieces<kThreads>(z, reinterpret_cast<const float4 *>(src + st.head), t, st.pieces);
    bool mine = false;
    for (int j = t; j < top; j += kThreads) {
        const int64_t id = ids[row * top + j];
        const float u    = teacher[row * top + j];
        entries.u[j]     = u;
        entries.id[j]    = entry_of(id, n, u) ? (int)id : -1;
        mine |= entry_of(id, n, u);
    }
    const float l = lse_given(lse[row]), scale = __fmul_rn(dloss ? dloss[row] : 1.0f, temperature);
    const bool some = __syncthreads_or(mine);
    map_stretch<kThreads, VEC>(src, dst, count, st, z, t, [&](float v) { return some ? __fmul_rn(probability(v, inv_t, inv_t_rest, l), scale) : 0.0f; });
    if (!some)
        return;
    const Weights w = weights_of(entries, top, inv_t, t & 31);
    const float by  = __fdiv_rn(scale, w.sum);
    __syncthreads(); // the row has been written: each class takes its entries' weights off, by the first of them
    for (int j = t; j < top; j += kThreads) {
        const int id = entries.id[j];
        if (id < c0 || id >= c0 + count)
            continue;
        bool first = true;
        float p    = 0.0f;
        for (int i = 0; i < top; ++i)
            if (entries.id[i] == id) {
                first &= i >= j;
                p = __fadd_rn(p, expf(__fmul_rn(__fsub_rn(entries.u[i], w.top), inv_t)));
            }
        if (first)
            dst[id - c0] = __fmaf_rn(-p, by, dst[id - c0]);
    }
}

// Whether a warp takes a row, or a block; measured in line (us, 20 entries; a warp and a block, forward and backward): 1000 x 600 6.1 and 7.9, 5.6 and 8.7; 2000 x 1000
// 5.6 and 11.8, 5.6 and 13.3; 300 x 4000 5.7 and 5.8, 6.0 and 5.1 (L2 flushed 13 and 10, 14 and 10); 1000 x 4000 5.6 and 7.9, 6.3 and 9.6 (14 and 13, 17 and 16);
// 1500 x 4000 7.5 and 10.2, 8.4 and 11.0; 2000 x 6000 11.2 and 13.8, 15.2 and 19.4; 4700 x 4000 11.6 and 21.3, 25.7 and 33.5; 60000 x 1500 76 and 265, 117 and 317;
// 20000 x 6000 82 and 125, 161 and 177.  Backward a block from there on, forward from twice that: 20000 x 8000 107 and 130, 213 and 200; 20000 x 12000 155 and 173,
// 320 and 289; 20000 x 16000 210 and 212, 435 and 385; with few rows a block too: 2400 x 8000 18.5 and 16.5, 29.6 and 28.9, but 3000 x 12000 29 and 35, 52 and 50.
bool distill_by_warps(const DeviceState *st, int64_t m, int64_t n, int64_t top, bool backward) {
    return top <= kWarpEntries && (n <= 1024 || (n <= 6000 && m >= st->sm_count * 10) || (!backward && n <= 12000 && m >= st->sm_count * 20));
}

ct_status check_distill(const char *name, int64_t m, int64_t n, int64_t top, double temperature) {
    if (m < 0 || n < 0 || top < 0)
        return fail(CT_ERR_INVALID, "%s: negative dimension", name);
    if (m > 1 << 29 || n > 1 << 29)
        return fail(CT_ERR_TOO_LARGE, "%s: dimension too large", name);
    if (top > kMostEntries)
        return fail(CT_ERR_TOO_LARGE, "%s: more than %d entries to a row", name, kMostEntries);
    if (m > 0 && n == 0)
        return fail(CT_ERR_INVALID, "%s: no classes", name);
    if (!(temperature >= 1e-6 && temperature <= 1e6))
        return fail(CT_ERR_INVALID, "%s: temperature must be from 1e-6 to 1e6", name);
    return CT_OK;
}

} // namespace
} // namespace ct

using namespace ct;

extern "C" {

ct_status ct_distill(
    const float *logits, const int64_t *ids, const float *teacher, int64_t m, int64_t n, int64_t top, double temperature, float *loss, float *lse) {
    OpLock op_lock;
    DeviceState *st;
    CT_TRY(current(&st));
    CT_TRY(check_distill("distill", m, n, top, temperature));
    if (m == 0 || (!loss && !lse))
        return CT_OK;
    if (!logits || (top > 0 && loss && (!ids || !teacher)))
        return fail(CT_ERR_INVALID, "distill: null pointer");
    ProfScope prof("distill");
    const float warm = (float)temperature, inv_t = (float)(1.0 / (double)warm);
    int early        = 1;
    for (const float *to : {loss, lse})
        early &= lines_apart(to, m * 4, logits, m * n * 4) && lines_apart(to, m * 4, ids, m * top * 8) && lines_apart(to, m * 4, teacher, m * top * 4);
    auto short_rows = [&](auto kernel, int tpr) -> ct_status {
        CT_CUDA(launch_dependent(kernel, dim3((unsigned)((m + 256 / tpr - 1) / (256 / tpr))), dim3(256), 0, stream(), logits, ids, teacher, m, n, (int)top, warm, inv_t, loss, lse, early));
        CT_LAUNCH_CHECK("distill_short");
        return CT_OK;
    };
    // (us in line, 60000 rows; 8 threads with 4 values each, 8 with 16, 16 with 32, a warp; forward, then backward: 10 classes, 5 entries 8.5, 13.9, 36, 40, 7.5, 14.2,
    // 41, 33; 128 classes, 20 entries -, 14.8, 37, 43, -, 21, 47, 45; 512 classes, 64 entries -, -, 44, 49, -, -, 70, 83)
    if (n <= 32 && top <= 16)
        return short_rows(distill_short_kernel<8, 4, 2>, 8);
    if (n <= 128 && top <= 32)
        return short_rows(distill_short_kernel<8, 16, 4>, 8);
    if (n <= 512 && top <= 64)
        return short_rows(distill_short_kernel<16, 32, 4>, 16);
    if (distill_by_warps(st, m, n, top, false))
        return short_rows(distill_warp_kernel, 32);
    int parts = 1;
    // 131072 classes, 1, 2, 4 and 8 blocks to a row: 31, 19, 14, 10 us (1 row), 33, 22, 17, 16 (64), 37, 28, 25, 28 (148), 47, 40, 44, 47 (300), 70, 71, 76, 76 (600)
    while (parts < 8 && m * parts * 2 <= st->sm_count * 5 && n > (int64_t)parts * kThreads * 16)
        parts *= 2;
    const int64_t part = ((n + parts - 1) / parts + 3) & ~(int64_t)3;
    CT_CUDA(launch_dependent_cluster(distill_kernel, parts, dim3((unsigned)(m * parts)), dim3(kThreads), 0, stream(), logits, ids, teacher, n, (int)top, warm,
                                     inv_t, parts, part, loss, lse, early));
    CT_LAUNCH_CHECK("distill");
    return CT_OK;
}

ct_status ct_distill_grad(
    const float *logits, const int64_t *ids, const float *teacher, const float *lse, const float *dloss, int64_t m, int64_t n, int64_t top,
    double temperature, float *dlogits) {
    OpLock op_lock;
    DeviceState *st;
    CT_TRY(current(&st));
    CT_TRY(check_distill("distill_grad", m, n, top, temperature));
    if (m == 0)
        return CT_OK;
    if (!logits || !lse || !dlogits || (top > 0 && (!ids || !teacher)))
        return fail(CT_ERR_INVALID, "distill_grad: null pointer");
    ProfScope prof("distill_grad");
    const float warm = (float)temperature, inv_t = (float)(1.0 / (double)warm), rest = (float)(1.0 / (double)warm - (double)inv_t);
    auto short_rows = [&](auto kernel, int tpr) -> ct_status {
        CT_CUDA(launch_dependent(kernel, dim3((unsigned)((m + 256 / tpr - 1) / (256 / tpr))), dim3(256), 0, stream(), logits, ids, teacher, lse, dloss, m, n, (int)top, warm, inv_t, rest, dlogits));
        CT_LAUNCH_CHECK("distill_grad_short");
        return CT_OK;
    };
    if (n <= 32 && top <= 16)
        return short_rows(distill_grad_short_kernel<8, 4, 2>, 8);
    if (n <= 128 && top <= 32)
        return short_rows(distill_grad_short_kernel<8, 16, 4>, 8);
    if (n <= 512 && top <= 64)
        return short_rows(distill_grad_short_kernel<16, 32, 4>, 16);
    const bool alike = ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(dlogits)) & 15u) == 0; // 16 bytes of one are 16 of the other
    if (distill_by_warps(st, m, n, top, true))
        return alike ? short_rows(distill_grad_warp_kernel<true>, 32) : short_rows(distill_grad_warp_kernel<false>, 32);
    // Parts of about 16384 classes, or of less where rows are few; measured with 1, 2, 3, 4 and 8: 4096 x 50257 279, 266, 258, 264, 301 us; 4096 x 131072 689, 675,
    // 677, 659, 641; 1500 x 32003 78, 72, 74, 74, 82; 8000 x 16000 168, 173, 215, 201, 344; 1 x 131072 33 with one, 8 with 16 and 32
    int parts = (int)std::max<int64_t>(1, (n + 8192) / 16384);
    while (m * parts < st->sm_count * 8 && n > (int64_t)parts * kThreads * 16)
        parts *= 2;
    const int64_t part = ((n + parts - 1) / parts + 3) & ~(int64_t)3;
    auto launch        = [&](auto kernel) -> ct_status {
        CT_CUDA(launch_dependent(kernel, dim3((unsigned)(m * parts)), dim3(kThreads), 0, stream(), logits, ids, teacher, lse, dloss, n, (int)top, warm, inv_t,
                                 rest, parts, part, dlogits));
        CT_LAUNCH_CHECK("distill_grad");
        return CT_OK;
    };
    return alike ? launch(distill_grad_kernel<true>) : launch(distill_grad_kernel<false>);
}

} // extern "C"
