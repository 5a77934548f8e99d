// Gradients of products of few rows: from the gradients d of the sums (two matrices: of both) in one kernel
//
//   dx = d . w^T (of two matrices the sum over both), dw = x^T . d, db = column sums of d
//
// Bound by reading the weights and writing their gradient, once each: a block has 1024 columns and a part of the rows of a matrix, a lane four
// columns (32 apart: any alignment is whole lines), whose d stay in registers while the rows go by, the next ones on their way.  A row's value of dw is a few products in
// the lane; its parts of dx are summed over the lane's columns, by halves over the warp, in shared memory over the block, and in 64 bits over
// the blocks beside it (join_columns).  d itself comes from what D computes it of, again in each part.
// As operand planes and tiles, which mostly hold nothing, 1 x 975 x 37218 with the logits took 317 us, so 102; 16 x 1024 x 32000 250, so 172.
#pragma once

#include "fastmath.cuh"
#include "fused_product.cuh"

namespace ct {
namespace fused {

struct FewGrad {
    const float *x, *w[2];
    float *dw[2], *db[2], *dx; // each may be null
    double *partial;           // [matrix x strip][m][k]: parts of dx, or null: dx itself
    int64_t k, n, each;        // each: rows of a part, a multiple of 8
    int m, strips, parts;
};
constexpr int kFewGradColumns = 1024; // of a block

#ifdef __CUDACC__

// v[0 .. COUNT) summed over the warp, halves of the values to halves of the lanes: lane l ends up with the COUNT / 16 values from
// (l >> 1) * COUNT / 16 on.
template <int COUNT> __device__ __forceinline__ void sum_by_halves(float (&v)[COUNT]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int step = 0; step < 4; ++step) {
        const int half = COUNT >> (step + 1), o = 16 >> step;
        const bool up  = lane & o;
#pragma unroll
        for (int i = 0; i < COUNT / 2; ++i)
            if (i < half) {
                const float keep = up ? v[i + half] : v[i], give = up ? v[i] : v[i + half];
                v[i]             = __fadd_rn(keep, __shfl_xor_sync(0xffffffffu, give, o));
            }
    }
#pragma unroll
    for (int i = 0; i < COUNT / 16; ++i)
        v[i] = __fadd_rn(v[i], __shfl_xor_sync(0xffffffffu, v[i], 1));
}

// D: kMatrices; has(r): whether row r takes part (else at is 0 and x is not looked at); at(which, r, c).  M: rows, rounded up.
template <class D, int M>
__global__ void __launch_bounds__(256, M == 4 ? 3 : 2) few_grad_kernel(const __grid_constant__ FewGrad p, const __grid_constant__ D d) {
    constexpr int KK = M == 16 ? 2 : 4, ROWS = 512 / M; // rows of w at a time; whose x and sums are in shared memory at a time
    extern __shared__ __align__(16) float few_smem[];
    __shared__ __align__(16) float xs[ROWS][M];
    __shared__ float sums[8][ROWS * M];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int strip = (int)(blockIdx.x % p.strips), part = (int)(blockIdx.x / p.strips % p.parts), which = (int)(blockIdx.x / p.strips / p.parts);
    const int64_t c0 = (int64_t)strip * kFewGradColumns, k0 = part * p.each, k1 = min(p.k, k0 + p.each);
    const int wide = (int)min((int64_t)kFewGradColumns, p.n - c0);
    griddep_wait();
    griddep_launch_dependents();
    const bool active = warp * 128 < wide, back = p.dx != nullptr;
    const float *w = p.w[which];
    float *dw      = p.dw[which];
    int64_t col[4];
    bool here[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int c = warp * 128 + q * 32 + lane;
        col[q] = c0 + c, here[q] = c < wide;
    }
    float v[KK][4], next[KK][4];
    auto load = [&](int64_t row, float (&to)[KK][4]) {
#pragma unroll
        for (int i = 0; i < KK; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                to[i][q] = back && here[q] && row + i < k1 ? __ldcs(w + (row + i) * p.n + col[q]) : 0.0f;
    };
    load(k0, next); // d is computed meanwhile
    for (int i = t; i < M * kFewGradColumns; i += 256) { // one copy of the code, however many values
        const int r = i / kFewGradColumns, c = i % kFewGradColumns;
        few_smem[i] = r < p.m && c < wide && d.has(r) ? d.at(which, r, c0 + c) : 0.0f;
    }
    __syncthreads();
    f32x2 dd[M / 2][4]; // of rows 2 j and 2 j + 1
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int c = warp * 128 + q * 32 + lane;
#pragma unroll
        for (int j = 0; j < M / 2; ++j)
            dd[j][q] = pack2(few_smem[2 * j * kFewGradColumns + c], few_smem[(2 * j + 1) * kFewGradColumns + c]);
        if (part == 0 && p.db[which] && here[q]) {
            float s = 0.0f;
#pragma unroll
            for (int j = 0; j < M / 2; ++j) {
                float a, b;
                unpack2(dd[j][q], a, b);
                s = __fadd_rn(__fadd_rn(s, a), b);
            }
            p.db[which][col[q]] = s;
        }
    }
    for (int64_t from = k0; from < k1; from += ROWS) {
        const int rows = (int)min((int64_t)ROWS, k1 - from);
        __syncthreads(); // the rows before these are through
        for (int i = t; i < ROWS * M; i += 256) {
            const int r = i / ROWS, kk = i % ROWS;
            xs[kk][r] = r < p.m && kk < rows && dw && d.has(r) ? p.x[r * p.k + from + kk] : 0.0f;
        }
        __syncthreads();
        if (active)
            for (int r0 = 0; r0 < rows; r0 += KK) {
#pragma unroll
                for (int i = 0; i < KK; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        v[i][q] = next[i][q];
                load(from + r0 + KK, next);
                if (dw)
#pragma unroll
                    for (int i = 0; i < KK; ++i) {
                        f32x2 s[4] = {0, 0, 0, 0};
#pragma unroll
                        for (int j = 0; j < M / 2; ++j) {
                            const f32x2 a = *reinterpret_cast<const f32x2 *>(&xs[r0 + i][2 * j]);
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                s[q] = fma2(a, dd[j][q], s[q]);
                        }
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            float a, b;
                            unpack2(s[q], a, b);
                            if (here[q] && r0 + i < rows)
                                __stcs(dw + (from + r0 + i) * p.n + col[q], __fadd_rn(a, b));
                        }
                    }
                if (back) {
                    float part_of[KK * M];
#pragma unroll
                    for (int i = 0; i < KK; ++i)
#pragma unroll
                        for (int j = 0; j < M / 2; ++j) {
                            f32x2 s = 0;
#pragma unroll
                            for (int q = 0; q < 4; ++q)
                                s = fma2(pack2(v[i][q], v[i][q]), dd[j][q], s);
                            unpack2(s, part_of[i * M + 2 * j], part_of[i * M + 2 * j + 1]);
                        }
                    sum_by_halves<KK * M>(part_of);
                    if (!(lane & 1))
#pragma unroll
                        for (int i = 0; i < KK * M / 16; ++i)
                            sums[warp][r0 * M + (lane >> 1) * (KK * M / 16) + i] = part_of[i];
                }
            }
        __syncthreads();
        if (back)
            for (int i = t; i < ROWS * M; i += 256) {
                const int kk = i % ROWS, r = i / ROWS;
                if (kk >= rows || r >= p.m)
                    continue;
                float s = sums[0][kk * M + r];
                for (int q = 1; q * 128 < wide; ++q)
                    s = __fadd_rn(s, sums[q][kk * M + r]);
                const int64_t at = r * p.k + from + kk;
                if (p.partial)
                    p.partial[((int64_t)which * p.strips + strip) * p.m * p.k + at] = (double)s;
                else
                    p.dx[at] = s;
            }
    }
}

template <class D, int M> ct_status launch_few_grad(DeviceState *st, FewGrad p, const D &d) {
    const int64_t strips = (p.n + kFewGradColumns - 1) / kFewGradColumns, lots = strips * D::kMatrices;
    // as many parts as fill the machine, of at least eight rows
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>((p.k + 7) / 8, (int64_t)st->sm_count * (M == 4 ? 3 : 2) / lots));
    p.each   = (p.k + parts * 8 - 1) / (parts * 8) * 8;
    p.parts  = (int)((p.k + p.each - 1) / p.each);
    p.strips = (int)strips;
    Scratch partial;
    if (p.dx && lots > 1) {
        CT_TRY(partial.get((size_t)(lots * p.m * p.k) * 8));
        p.partial = partial.as<double>();
    }
    const int smem = M * kFewGradColumns * 4;
    auto kernel    = few_grad_kernel<D, M>;
    static bool attr_set_dev[16] = {};
    if (!attr_set_dev[st->device & 15]) {
        CT_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        attr_set_dev[st->device & 15] = true;
    }
    CT_CUDA(launch_dependent(kernel, dim3((unsigned)(lots * p.parts)), dim3(256), (size_t)smem, stream(), p, d));
    CT_LAUNCH_CHECK("few_rows_grad");
    return p.partial ? join_columns(p.partial, lots, p.m * p.k, p.m * p.k, p.dx, nullptr) : CT_OK;
}

// At most kFewRows rows; k > 0, and something to compute.
template <class D> ct_status few_rows_grad(DeviceState *st, const FewGrad &p, const D &d) {
    if (p.m <= 4)
        return launch_few_grad<D, 4>(st, p, d);
    if (p.m <= 8)
        return launch_few_grad<D, 8>(st, p, d);
    return launch_few_grad<D, 16>(st, p, d);
}

#endif

} // namespace fused
} // namespace ct
