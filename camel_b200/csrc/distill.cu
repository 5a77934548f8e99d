// Distillation from the classes that a teacher thinks likeliest, and its gradient.
//
//   p = softmax(teacher / T) over a row's entries, q = softmax(z / T) over its classes
//   loss = T^2 sum p (log p - log q),  dz[c] = dloss T (q[c] - the sum of p over the entries of class c)
//
// Both are bound by memory: the logits are read once (4 bytes each), and on the way back written once (8).  Forward, a thread keeps the
// maximum of its logits and the sum of exponentials about it, which meet at the end; a row of a small batch is shared by the blocks of a cluster.
// Backward, lse is given: a row is q times a factor, from which its block takes the entries' p where it has written them.
#include "common.cuh"
#include "tc_ptx.cuh"

#include <algorithm>
#include <cfloat>

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

// The largest of some logits and the sum of exp((z - top) / T); a NaN or +infinity among them shows in the sum.
struct Sum {
    float top, sum;
};
__device__ __forceinline__ float about(float top) { return top == -INFINITY ? 0.0f : top; } // classes that are out leave a sum of 0
__device__ __forceinline__ Sum join(Sum a, Sum b, float c) {
    const float top = fmaxf(a.top, b.top), base = about(top);
    // one of the two exponentials is 1; of an empty side 0
    return {top, __fadd_rn(__fmul_rn(a.sum, ex2(__fmul_rn(__fsub_rn(a.top, base), c))), __fmul_rn(b.sum, ex2(__fmul_rn(__fsub_rn(b.top, base), c))))};
}
// N more logits
template <int N> __device__ __forceinline__ void take(Sum &s, const float (&z)[N], float c) {
    float top = s.top;
#pragma unroll
    for (int i = 0; i < N; ++i)
        top = fmaxf(top, z[i]);
    const float base = about(top);
    float sum[4]     = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < N; ++i)
        sum[i & 3] = __fadd_rn(sum[i & 3], ex2(__fmul_rn(__fsub_rn(z[i], base), c)));
    s.sum = __fmaf_rn(s.sum, ex2(__fmul_rn(__fsub_rn(s.top, base), c)), __fadd_rn(__fadd_rn(sum[0], sum[1]), __fadd_rn(sum[2], sum[3])));
    s.top = top;
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

// The entries' weights are p[j] = exp(teacher[j] / T - top) / sum.  entry(j, &u): whether entry j has a class, and its teacher logit.
struct Weights {
    float top, sum;
    bool some; // whether there is any entry
};
template <int TPR, typename F> __device__ __forceinline__ Weights weights_of(int top, float inv_t, int t, F &&entry) {
    float most = -INFINITY;
    bool some  = false, bad = false;
    for (int j = t; j < top; j += TPR) {
        float u;
        if (entry(j, u)) {
            some = true;
            bad |= u != u;
            most = fmaxf(most, u);
        }
    }
    most           = max_lanes<TPR>(most);
    const float base = about(most);
    float sum      = bad ? NAN : 0.0f;
    for (int j = t; j < top; j += TPR) {
        float u;
        if (entry(j, u))
            sum = __fadd_rn(sum, expf(__fmul_rn(__fsub_rn(u, base), inv_t)));
    }
    const unsigned group = TPR == 32 ? 0xffffffffu : ((1u << (TPR & 31)) - 1) << ((threadIdx.x & 31) / TPR * TPR);
    return {base, sum_lanes<TPR>(sum), (__ballot_sync(0xffffffffu, some) & group) != 0};
}
// T^2 times the sum of p (log p - (z / T - lse)).  entry(j, &u, &z)
template <int TPR, typename F>
__device__ __forceinline__ float loss_of(const Weights &w, int top, float temperature, float inv_t, float lse, int t, F &&entry) {
    const float log_sum = logf(w.sum), inv_sum = __fdiv_rn(1.0f, w.sum);
    float loss = 0.0f;
    for (int j = t; j < top; j += TPR) {
        float u, z;
        if (entry(j, u, z)) {
            const float x = __fmul_rn(__fsub_rn(u, w.top), inv_t), p = __fmul_rn(expf(x), inv_sum);
            if (p != 0.0f) // 0 log 0 is 0
                loss = __fmaf_rn(p, __fsub_rn(__fsub_rn(x, log_sum), __fsub_rn(__fdiv_rn(z, temperature), lse)), loss);
        }
    }
    loss = __fmul_rn(__fmul_rn(temperature, temperature), sum_lanes<TPR>(loss));
    return w.some ? loss : 0.0f;
}
__device__ __forceinline__ float lse_of(Sum s, float temperature) { return __fadd_rn(__fdiv_rn(about(s.top), temperature), logf(s.sum)); }

__device__ __forceinline__ bool class_of(int64_t id, int64_t n) { return id >= 0 && id < n; }

// ---- rows of few classes: TPR threads to a row, V of its logits in each ---------------------------

template <int TPR, int V>
__global__ void __launch_bounds__(256) distill_short_kernel(
    const float *__restrict__ logits, const int64_t *__restrict__ ids, const float *__restrict__ teacher, int64_t m, int n, int top, float temperature,
    float inv_t, float *__restrict__ loss, float *__restrict__ lse) {
    griddep_wait();
    griddep_launch_dependents();
    const int t       = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    const bool here   = row < m; // the others go along
    const float c     = __fmul_rn(inv_t, kLog2e);
    const float *src  = logits + (here ? row * n : 0);
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i)
        z[i] = here && i * TPR + t < n ? src[i * TPR + t] : -INFINITY;
    Sum s = {-INFINITY, 0.0f};
    take(s, z, c);
    s             = join_lanes<TPR>(s, c);
    const float l = lse_of(s, temperature);
    if (loss) {
        const int count       = here ? top : 0;
        const int64_t *row_id = ids + (here ? row * top : 0);
        const float *row_u    = teacher + (here ? row * top : 0);
        const Weights w       = weights_of<TPR>(count, inv_t, t, [&](int j, float &u) { return u = row_u[j], class_of(row_id[j], n); });
        const float value     = loss_of<TPR>(w, count, temperature, inv_t, l, t, [&](int j, float &u, float &zj) {
            const int64_t id = row_id[j];
            const bool has   = class_of(id, n);
            u = row_u[j], zj = has ? src[id] : 0.0f;
            return has;
        });
        if (here && t == 0)
            loss[row] = value;
    }
    if (lse && here && t == 0)
        lse[row] = l;
}

// exp(z / T - lse) of a logit: 1 / T in two parts.  -infinity becomes a number, which neither part makes a NaN.
__device__ __forceinline__ float probability(float z, float inv_t, float inv_t_rest, float lse) {
    asm("max.NaN.f32 %0, %0, 0fFF7FFFFF;" : "+f"(z));
    return ex2(__fmul_rn(__fmaf_rn(z, inv_t, __fmaf_rn(z, inv_t_rest, -lse)), kLog2e));
}

// The entries of a row, in shared or global memory: from where the row has been written, each class takes its weights off once.
template <int TPR, typename F, typename G>
__device__ __forceinline__ void take_off(const Weights &w, int top, float inv_t, float scale, int t, float *row, int64_t c0, int64_t c1, F &&id_of, G &&u_of) {
    const float by = __fdiv_rn(scale, w.sum);
    for (int j = t; j < top; j += TPR) {
        const int64_t id = id_of(j);
        if (id < c0 || id >= c1)
            continue;
        bool first = true;
        float p    = 0.0f;
        for (int i = 0; i < top; ++i)
            if (id_of(i) == id) { // a class may stand in several entries
                first &= i >= j;
                p = __fadd_rn(p, expf(__fmul_rn(__fsub_rn(u_of(i), w.top), inv_t)));
            }
        if (first)
            row[id] = __fmaf_rn(-p, by, row[id]);
    }
}

template <int TPR, int V>
__global__ void __launch_bounds__(256) distill_grad_short_kernel(
    const float *logits, const int64_t *__restrict__ ids, const float *__restrict__ teacher, const float *__restrict__ lse,
    const float *__restrict__ dloss, int64_t m, int n, int top, float temperature, float inv_t, float inv_t_rest, float *dlogits) {
    griddep_wait();
    const int t       = threadIdx.x % TPR;
    const int64_t row = (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR;
    const bool here   = row < m;
    const float *src  = logits + (here ? row * n : 0);
    float *dst        = dlogits + (here ? row * n : 0);
    float z[V];
#pragma unroll
    for (int i = 0; i < V; ++i)
        z[i] = here && i * TPR + t < n ? src[i * TPR + t] : 0.0f;
    const int count       = here ? top : 0;
    const int64_t *row_id = ids + (here ? row * top : 0);
    const float *row_u    = teacher + (here ? row * top : 0);
    const Weights w       = weights_of<TPR>(count, inv_t, t, [&](int j, float &u) { return u = row_u[j], class_of(row_id[j], n); });
    const float l = here ? lse[row] : 0.0f, scale = here ? __fmul_rn(dloss ? dloss[row] : 1.0f, temperature) : 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (here && i * TPR + t < n)
            dst[i * TPR + t] = w.some ? __fmul_rn(probability(z[i], inv_t, inv_t_rest, l), scale) : 0.0f;
    __syncwarp();
    if (w.some)
        take_off<TPR>(w, count, inv_t, scale, t, dst, 0, n, [&](int j) { return row_id[j]; }, [&](int j) { return row_u[j]; });
}

// ---- longer rows: a block to a row, or to a part of one -------------------------------------------

// 16-byte pieces of a stretch of floats at any address: `head` values before the first, and `tail` behind the last.
struct Stretch {
    int64_t head, pieces, tail;
};
__device__ __forceinline__ Stretch stretch_of(const float *p, int64_t count) {
    Stretch s;
    s.head   = min((int64_t)((4 - ((reinterpret_cast<uintptr_t>(p) >> 2) & 3)) & 3), count);
    s.pieces = (count - s.head) / 4;
    s.tail   = count - s.head - 4 * s.pieces;
    return s;
}

constexpr int kThreads = 256;

__global__ void __launch_bounds__(kThreads) distill_kernel(
    const float *__restrict__ logits, const int64_t *__restrict__ ids, const float *__restrict__ teacher, int64_t n, int top, float temperature,
    float inv_t, int parts, int64_t part, float *__restrict__ loss, float *__restrict__ lse) {
    __shared__ float entry_u[kMostEntries], entry_z[kMostEntries];
    __shared__ bool entry_has[kMostEntries];
    __shared__ Sum warps[kThreads / 32], blocks[8];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const uint32_t rank = parts > 1 ? cluster_rank() : 0;
    if (parts > 1)
        cluster_sync(); // every block of the cluster runs before another writes into its memory
    griddep_wait();
    griddep_launch_dependents();
    const int64_t row = blockIdx.x / parts;
    const float c     = __fmul_rn(inv_t, kLog2e);
    const float *src  = logits + row * n;
    if (rank == 0 && loss)
        for (int j = t; j < top; j += kThreads) {
            const int64_t id = ids[row * top + j];
            entry_has[j]     = class_of(id, n);
            entry_u[j]       = teacher[row * top + j];
            entry_z[j]       = class_of(id, n) ? src[id] : 0.0f;
        }
    const int64_t c0 = min(rank * part, n), count = min(part, n - c0);
    const Stretch st = stretch_of(src + c0, count);
    const float *body = src + c0 + st.head;
    Sum s = {-INFINITY, 0.0f};
    if (t < st.head + st.tail) {
        const float z[1] = {t < st.head ? src[c0 + t] : body[4 * st.pieces + t - st.head]};
        take(s, z, c);
    }
    constexpr int kAtOnce = 4;
    for (int64_t i = t; i < st.pieces; i += kThreads * kAtOnce) {
        float z[4 * kAtOnce];
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
            float4 f = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
            if (i + u * kThreads < st.pieces)
                f = __ldcs(reinterpret_cast<const float4 *>(body) + i + u * kThreads);
            z[4 * u] = f.x, z[4 * u + 1] = f.y, z[4 * u + 2] = f.z, z[4 * u + 3] = f.w;
        }
        take(s, z, c);
    }
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
    if (rank == 0 && warp == 0) {
        const float l = lse_of(s, temperature);
        if (loss) {
            const Weights w   = weights_of<32>(top, inv_t, lane, [&](int j, float &u) { return u = entry_u[j], entry_has[j]; });
            const float value = loss_of<32>(w, top, temperature, inv_t, l, lane,
                                            [&](int j, float &u, float &z) { return u = entry_u[j], z = entry_z[j], entry_has[j]; });
            if (lane == 0)
                loss[row] = value;
        }
        if (lse && lane == 0)
            lse[row] = l;
    }
}

template <bool VEC>
__global__ void __launch_bounds__(kThreads) distill_grad_kernel(
    const float *logits, const int64_t *__restrict__ ids, const float *__restrict__ teacher, const float *__restrict__ lse,
    const float *__restrict__ dloss, int64_t n, int top, float temperature, float inv_t, float inv_t_rest, int parts, int64_t part, float *dlogits) {
    __shared__ int64_t entry_id[kMostEntries];
    __shared__ float entry_u[kMostEntries];
    griddep_wait();
    const int t       = threadIdx.x;
    const int64_t row = blockIdx.x / parts, c0 = min((int64_t)(blockIdx.x % parts) * part, n), count = min(part, n - c0);
    const float *src  = logits + row * n + c0;
    float *dst        = dlogits + row * n + c0;
    bool mine         = false;
    for (int j = t; j < top; j += kThreads) {
        const int64_t id = ids[row * top + j];
        entry_id[j]      = class_of(id, n) ? id : -1;
        entry_u[j]       = teacher[row * top + j];
        mine |= class_of(id, n);
    }
    const float l = lse[row], scale = __fmul_rn(dloss ? dloss[row] : 1.0f, temperature);
    const bool some = __syncthreads_or(mine);
    auto slope      = [&](float z) { return some ? __fmul_rn(probability(z, inv_t, inv_t_rest, l), scale) : 0.0f; };
    constexpr int kAtOnce = 4;
    if (VEC) {
        const Stretch st = stretch_of(src, count);
        if (t < st.head + st.tail) {
            const int64_t i = t < st.head ? t : st.pieces * 4 + t;
            dst[i]          = slope(src[i]);
        }
        const float4 *from = reinterpret_cast<const float4 *>(src + st.head);
        float4 *to         = reinterpret_cast<float4 *>(dst + st.head);
        for (int64_t i = t; i < st.pieces; i += kThreads * kAtOnce) {
            float4 z[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
                z[u] = i + u * kThreads < st.pieces ? __ldcs(from + i + u * kThreads) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
                if (i + u * kThreads < st.pieces)
                    __stcs(to + i + u * kThreads, make_float4(slope(z[u].x), slope(z[u].y), slope(z[u].z), slope(z[u].w)));
        }
    } else {
        for (int64_t i = t; i < count; i += kThreads * kAtOnce) {
            float z[kAtOnce];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
                z[u] = i + u * kThreads < count ? __ldcs(src + i + u * kThreads) : 0.0f;
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u)
                if (i + u * kThreads < count)
                    __stcs(dst + i + u * kThreads, slope(z[u]));
        }
    }
    __syncthreads();
    if (some) {
        const Weights w = weights_of<32>(top, inv_t, t & 31, [&](int j, float &u) { return u = entry_u[j], entry_id[j] >= 0; });
        take_off<kThreads>(w, top, inv_t, scale, t, dlogits + row * n, c0, c0 + count, [&](int j) { return entry_id[j]; }, [&](int j) { return entry_u[j]; });
    }
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
    if (n <= 512) {
        auto launch = [&](auto kernel, int tpr) -> ct_status {
            CT_CUDA(launch_dependent(kernel, dim3((unsigned)((m + 256 / tpr - 1) / (256 / tpr))), dim3(256), 0, stream(), logits, ids, teacher, m, (int)n, (int)top,
                                     warm, inv_t, loss, lse));
            CT_LAUNCH_CHECK("distill_short");
            return CT_OK;
        };
        return n <= 32 ? launch(distill_short_kernel<8, 4>, 8) : launch(distill_short_kernel<32, 16>, 32);
    }
    int parts = 1;
    while (parts < 8 && m * parts * 2 <= st->sm_count * 4 && n > (int64_t)parts * kThreads * 16)
        parts *= 2;
    const int64_t part = ((n + parts - 1) / parts + 3) & ~(int64_t)3;
    CT_CUDA(launch_dependent_cluster(distill_kernel, parts, dim3((unsigned)(m * parts)), dim3(kThreads), 0, stream(), logits, ids, teacher, n, (int)top, warm,
                                     inv_t, parts, part, loss, lse));
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
    if (n <= 512) {
        auto launch = [&](auto kernel, int tpr) -> ct_status {
            CT_CUDA(launch_dependent(kernel, dim3((unsigned)((m + 256 / tpr - 1) / (256 / tpr))), dim3(256), 0, stream(), logits, ids, teacher, lse, dloss, m,
                                     (int)n, (int)top, warm, inv_t, rest, dlogits));
            CT_LAUNCH_CHECK("distill_grad_short");
            return CT_OK;
        };
        return n <= 32 ? launch(distill_grad_short_kernel<8, 4>, 8) : launch(distill_grad_short_kernel<32, 16>, 32);
    }
    int parts = 1;
    while (m * parts < st->sm_count * 8 && n > (int64_t)parts * kThreads * 16)
        parts *= 2;
    const int64_t part = ((n + parts - 1) / parts + 3) & ~(int64_t)3;
    auto launch        = [&](auto kernel) -> ct_status {
        CT_CUDA(launch_dependent(kernel, dim3((unsigned)(m * parts)), dim3(kThreads), 0, stream(), logits, ids, teacher, lse, dloss, n, (int)top, warm, inv_t,
                                 rest, parts, part, dlogits));
        CT_LAUNCH_CHECK("distill_grad");
        return CT_OK;
    };
    const bool alike = ((reinterpret_cast<uintptr_t>(logits) ^ reinterpret_cast<uintptr_t>(dlogits)) & 15u) == 0;
    return alike ? launch(distill_grad_kernel<true>) : launch(distill_grad_kernel<false>);
}

} // extern "C"
