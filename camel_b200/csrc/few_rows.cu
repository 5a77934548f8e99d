// Products of few rows (a token, a handful of them): x . w, or both projections of a gated layer with the gate.
//
// Bound by reading the weights once.  A strip of 64 columns of each of two matrices (or 128 of one) belongs to a cluster of up to
// eight CTAs, each with a part of k; a lane has four columns, a warp every eighth row of the part, so that one wave of CTAs asks for the whole of a
// 1024 x 4096 matrix at once.  The warps' sums meet in shared memory, the cluster's in distributed shared memory: no second launch.
// Sums are float32, chains of k / 64 (k / 8 where one CTA has all of k) before the tree.
#include "fused_product.cuh"
#include "gate.cuh"

#include <type_traits>

namespace ct {
namespace fused {
namespace {

constexpr int kPart = 512; // values of k whose x a CTA holds in shared memory at a time

struct FewParams {
    const float *x, *w[2], *bias[2]; // the two matrices, or the two halves of a strip of one
    float *out, *gate_pre, *up_pre;
    int64_t k, n;
    int m, parts, vec;
};

// GATE < 0: no gate; column c of half 1 is column 64 + c of the strip.
template <int M, int GATE>
__global__ void __launch_bounds__(256, M == 1 ? 4 : M == 4 ? 3 : 2) few_rows_kernel(const __grid_constant__ FewParams p) {
    __shared__ float xs[M][kPart];
    __shared__ __align__(16) float sums[8][M][128]; // [0]: the CTA's, read by the cluster
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = lane >> 4;
    const int rank = (int)(blockIdx.x % p.parts);
    constexpr int WIDE = GATE < 0 ? 128 : 64;
    const int64_t c0 = (int64_t)(blockIdx.x / p.parts) * WIDE, col = c0 + (GATE < 0 ? half * 64 : 0) + (lane & 15) * 4;
    const int64_t each = (p.k + p.parts - 1) / p.parts, k0 = min(p.k, rank * each), k1 = min(p.k, k0 + each);
    griddep_wait();
    griddep_launch_dependents();
    float acc[M][4];
#pragma unroll
    for (int r = 0; r < M; ++r)
        acc[r][0] = acc[r][1] = acc[r][2] = acc[r][3] = 0.0f;
    const float *w = p.w[GATE < 0 ? 0 : half];
    for (int64_t from = k0; from < k1; from += kPart) {
        const int count  = (int)min((int64_t)kPart, k1 - from);
        const float *src = w + from * p.n + col;
        constexpr int U  = 8; // loads in flight
        for (int i0 = warp; i0 < (count + 63) / 64 * 64; i0 += 8 * U) {
            float4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + 8 * u;
                v[u]        = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                if (i < count) {
                    const float *at = src + (int64_t)i * p.n;
                    if (p.vec) {
                        if (col < p.n)
                            v[u] = __ldcs(reinterpret_cast<const float4 *>(at));
                    } else {
                        v[u].x = col < p.n ? __ldcs(at) : 0.0f, v[u].y = col + 1 < p.n ? __ldcs(at + 1) : 0.0f;
                        v[u].z = col + 2 < p.n ? __ldcs(at + 2) : 0.0f, v[u].w = col + 3 < p.n ? __ldcs(at + 3) : 0.0f;
                    }
                }
            }
            if (i0 == warp) { // x behind the first weights
                __syncthreads(); // the last part's has been read
                for (int i = threadIdx.x; i < M * count; i += 256) {
                    const int r = i / count, c = i % count;
                    xs[r][c] = r < p.m ? p.x[(int64_t)r * p.k + from + c] : 0.0f;
                }
                __syncthreads();
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int i = i0 + 8 * u;
                if (i < count)
#pragma unroll
                    for (int r = 0; r < M; ++r) {
                        const float a = xs[r][i];
                        acc[r][0] = __fmaf_rn(a, v[u].x, acc[r][0]), acc[r][1] = __fmaf_rn(a, v[u].y, acc[r][1]);
                        acc[r][2] = __fmaf_rn(a, v[u].z, acc[r][2]), acc[r][3] = __fmaf_rn(a, v[u].w, acc[r][3]);
                    }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < M; ++r)
        *reinterpret_cast<float4 *>(&sums[warp][r][lane * 4]) = make_float4(acc[r][0], acc[r][1], acc[r][2], acc[r][3]);
    __syncthreads();
    for (int i = threadIdx.x; i < M * 128; i += 256) {
        float s = sums[0][i / 128][i % 128];
#pragma unroll
        for (int q = 1; q < 8; ++q)
            s = __fadd_rn(s, sums[q][i / 128][i % 128]);
        sums[0][i / 128][i % 128] = s;
    }
    if (p.parts > 1)
        ptx::cluster_sync();
    else
        __syncthreads();
    auto total = [&](int r, int c) { // over the cluster, in order
        float s = 0.0f;
        for (int q = 0; q < p.parts; ++q) {
            float v;
            if (p.parts == 1) {
                v = sums[0][r][c];
            } else {
                const uint32_t at = ptx::mapa(ptx::smem_u32(&sums[0][r][c]), (uint32_t)q);
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
            }
            s = q ? __fadd_rn(s, v) : v;
        }
        return s;
    };
    for (int i = rank * 256 + threadIdx.x; i < p.m * WIDE; i += p.parts * 256) {
        const int r = i / WIDE, c = i % WIDE;
        const int64_t at = c0 + c;
        if (at >= p.n)
            continue;
        float g = total(r, c);
        if (p.bias[0])
            g = __fadd_rn(g, p.bias[0][at]);
        if (GATE >= 0) {
            float u = total(r, 64 + c);
            if (p.bias[1])
                u = __fadd_rn(u, p.bias[1][at]);
            if (p.gate_pre)
                p.gate_pre[r * p.n + at] = g;
            if (p.up_pre)
                p.up_pre[r * p.n + at] = u;
            g = __fmul_rn(gate_value<GATE < 0 ? 0 : GATE>(g), u);
        }
        p.out[r * p.n + at] = g;
    }
    if (p.parts > 1)
        ptx::cluster_sync(); // a CTA's sums stay until the others have read them
}

template <int M, int GATE> ct_status launch_few(DeviceState *st, FewParams &p) {
    constexpr int WIDE   = GATE < 0 ? 128 : 64;
    const int64_t strips = (p.n + WIDE - 1) / WIDE;
    p.parts              = 1;
    while (p.parts < 8 && strips * p.parts * 2 <= (int64_t)st->sm_count * (M == 1 ? 4 : M == 4 ? 3 : 2) && p.k >= p.parts * 2 * 64) // in one wave
        p.parts *= 2;
    CT_CUDA(launch_dependent_cluster(few_rows_kernel<M, GATE>, p.parts, dim3((unsigned)(strips * p.parts)), dim3(256), 0, stream(), p));
    CT_LAUNCH_CHECK("few_rows");
    return CT_OK;
}

template <int GATE> ct_status few_rows_of(DeviceState *st, FewParams &p) {
    if (p.m == 1)
        return launch_few<1, GATE>(st, p);
    if (p.m <= 4)
        return launch_few<4, GATE>(st, p);
    return launch_few<8, GATE>(st, p);
}

} // namespace

ct_status few_rows(
    DeviceState *st, const float *x, const float *w, const float *bias, const float *w_up, const float *b_up, int64_t m, int64_t k, int64_t n, int gate,
    float *out, float *gate_pre, float *up_pre) {
    FewParams p{};
    p.w[0] = w, p.w[1] = w_up ? w_up : w, p.bias[0] = bias, p.bias[1] = b_up;
    p.k = k, p.n = n;
    p.vec = (n & 3) == 0 && (reinterpret_cast<uintptr_t>(w) & 15u) == 0 && (reinterpret_cast<uintptr_t>(w_up) & 15u) == 0 ? 1 : 0;
    for (int64_t r = 0; r < m; r += 8) { // the weights come from L2 the second time
        p.m = (int)std::min<int64_t>(8, m - r);
        p.x = x + r * k, p.out = out + r * n;
        p.gate_pre = gate_pre ? gate_pre + r * n : nullptr, p.up_pre = up_pre ? up_pre + r * n : nullptr;
        if (!w_up)
            CT_TRY(few_rows_of<-1>(st, p));
        else
            CT_TRY(with_gate(gate, [&](auto G) { return few_rows_of<G.value>(st, p); }));
    }
    return CT_OK;
}

} // namespace fused
} // namespace ct
