// Softmax cross entropy of a dense layer's logits, and its gradient, without keeping the logits.
//
//   lse = log(sum exp z), loss = lse - z[target];  d = dloss (exp(z - lse) - [target]),  dx = d . w^T, dw = x^T . d, dbias = column sums of d
#include "common.cuh"

#include <algorithm>

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

ct_status check_ce(const char *name, const void *x, const void *w, const void *targets, int64_t m, int64_t k, int64_t n) {
    if (m < 0 || k < 0 || n < 0)
        return fail(CT_ERR_INVALID, "%s: negative dimension", name);
    if (n == 0 && m > 0)
        return fail(CT_ERR_INVALID, "%s: no classes", name);
    if (m > 0x7fffffff || n > 0x7fffffff || k > 0x7fffffff)
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
    const int64_t piece = rows_at_once(m, n);
    Scratch logits;
    CT_TRY(logits.get((size_t)(piece * n) * 4));
    for (int64_t r = 0; r < m; r += piece) {
        const int64_t rows = std::min(piece, m - r);
        CT_TRY(ct_dense(x + r * k, w, bias, rows, k, n, CT_ACT_NONE, logits.as<float>(), nullptr));
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
    const int64_t piece = rows_at_once(m, n);
    Scratch logits, turned, sums;
    CT_TRY(logits.get((size_t)(piece * n) * 4));
    float *d = logits.as<float>();
    if (dx && k > 0) {
        CT_TRY(turned.get((size_t)(k * n) * 4));
        CT_TRY(ct_transpose(CT_F32, w, k, n, turned.as<float>()));
    }
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
            CT_TRY(ct_matmul_tn(x + r * k, d, k, rows, n, r ? sums.as<float>() : dw));
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
