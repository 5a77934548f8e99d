// Gated dense layer: out = gate(x . w_gate + b_gate) * (x . w_up + b_up), and its gradient.
#include "common.cuh"
#include "gate.cuh"

#include <algorithm>
#include <type_traits>

namespace ct {
namespace {

// out = gate(g) * u
template <int GATE>
__global__ void __launch_bounds__(256) gated_product_kernel(const float *g, const float *u, int64_t count, float *out) {
    griddep_wait();
    griddep_launch_dependents();
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256)
        out[i] = __fmul_rn(gate_value<GATE>(g[i]), u[i]);
}

// dg and du
template <int GATE>
__global__ void __launch_bounds__(256) gated_slopes_kernel(
    const float *__restrict__ g, const float *__restrict__ u, const float *__restrict__ dout, int64_t count, float *__restrict__ dg,
    float *__restrict__ du) {
    griddep_wait();
    griddep_launch_dependents();
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
        float value, slope;
        gate_slope<GATE>(g[i], value, slope);
        dg[i] = __fmul_rn(__fmul_rn(dout[i], u[i]), slope);
        du[i] = __fmul_rn(dout[i], value);
    }
}

unsigned grid_of(const DeviceState *st, int64_t count) {
    return (unsigned)std::min<int64_t>((count + 255) / 256, (int64_t)st->sm_count * 16);
}

ct_status check_gated(const char *name, int64_t m, int64_t k, int64_t n, int gate) {
    if (m < 0 || k < 0 || n < 0)
        return fail(CT_ERR_INVALID, "%s: negative dimension", name);
    if (!valid_gate(gate))
        return fail(CT_ERR_INVALID, "%s: unknown gate", name);
    return CT_OK;
}

} // namespace
} // namespace ct

using namespace ct;

extern "C" {

ct_status ct_dense_gated(
    const float *x, const float *w_gate, const float *b_gate, const float *w_up, const float *b_up, int64_t m, int64_t k, int64_t n, ct_gate gate,
    float *out, float *gate_pre, float *up_pre) {
    OpLock op_lock;
    DeviceState *st;
    CT_TRY(current(&st));
    CT_TRY(check_gated("dense_gated", m, k, n, gate));
    if (m == 0 || n == 0)
        return CT_OK;
    if (!out || (k > 0 && (!x || !w_gate || !w_up)))
        return fail(CT_ERR_INVALID, "dense_gated: null pointer");
    ProfScope prof("dense_gated");
    const int64_t count = m * n;
    Scratch scratch;
    float *g = gate_pre, *u = up_pre;
    if (!g || !u) {
        CT_TRY(scratch.get((size_t)count * 8));
        g = g ? g : scratch.as<float>();
        u = u ? u : scratch.as<float>((size_t)count * 4);
    }
    CT_TRY(ct_dense(x, w_gate, b_gate, m, k, n, CT_ACT_NONE, g, nullptr));
    CT_TRY(ct_dense(x, w_up, b_up, m, k, n, CT_ACT_NONE, u, nullptr));
    return with_gate(gate, [&](auto G) -> ct_status {
        CT_CUDA(launch_dependent(gated_product_kernel<G.value>, dim3(grid_of(st, count)), dim3(256), 0, stream(), (const float *)g, (const float *)u, count,
                                 out));
        CT_LAUNCH_CHECK("gated_product");
        return CT_OK;
    });
}

ct_status ct_dense_gated_grad(
    const float *x, const float *w_gate, const float *w_up, const float *gate_pre, const float *up_pre, const float *dout, int64_t m, int64_t k,
    int64_t n, ct_gate gate, float *dx, float *dw_gate, float *dw_up, float *db_gate, float *db_up) {
    OpLock op_lock;
    DeviceState *st;
    CT_TRY(current(&st));
    CT_TRY(check_gated("dense_gated_grad", m, k, n, gate));
    if (m > 0 && n > 0 && (!gate_pre || !up_pre || !dout))
        return fail(CT_ERR_INVALID, "dense_gated_grad: null pointer");
    if (m > 0 && n > 0 && k > 0 && ((dx && (!w_gate || !w_up)) || ((dw_gate || dw_up) && !x)))
        return fail(CT_ERR_INVALID, "dense_gated_grad: null pointer");
    ProfScope prof("dense_gated_grad");
    if (m == 0 || n == 0) { // sums of nothing
        auto clear = [&](float *p, int64_t count) {
            return p && count > 0 ? cudaMemsetAsync(p, 0, (size_t)count * 4, stream()) : cudaSuccess;
        };
        CT_CUDA(clear(dx, m * k));
        CT_CUDA(clear(dw_gate, k * n));
        CT_CUDA(clear(dw_up, k * n));
        CT_CUDA(clear(db_gate, n));
        CT_CUDA(clear(db_up, n));
        return CT_OK;
    }
    const int64_t count = m * n;
    Scratch slopes;
    CT_TRY(slopes.get((size_t)count * 8));
    float *dg = slopes.as<float>(), *du = dg + count;
    CT_TRY(with_gate(gate, [&](auto G) -> ct_status {
        CT_CUDA(launch_dependent(gated_slopes_kernel<G.value>, dim3(grid_of(st, count)), dim3(256), 0, stream(), gate_pre, up_pre, dout, count, dg, du));
        CT_LAUNCH_CHECK("gated_slopes");
        return CT_OK;
    }));
    if (k > 0 && dw_gate)
        CT_TRY(ct_matmul_tn(x, dg, k, m, n, dw_gate));
    if (k > 0 && dw_up)
        CT_TRY(ct_matmul_tn(x, du, k, m, n, dw_up));
    if (db_gate)
        CT_TRY(ct_sum_axis(CT_F32, dg, m, n, 0, db_gate));
    if (db_up)
        CT_TRY(ct_sum_axis(CT_F32, du, m, n, 0, db_up));
    if (k > 0 && dx) {
        Scratch turned;
        CT_TRY(turned.get((size_t)(k * n + m * k) * 4));
        float *wt = turned.as<float>(), *part = wt + k * n;
        CT_TRY(ct_transpose(CT_F32, w_gate, k, n, wt));
        CT_TRY(ct_matmul(CT_F32, dg, CT_F32, wt, m, n, k, part));
        CT_TRY(ct_transpose(CT_F32, w_up, k, n, wt));
        CT_TRY(ct_matmul(CT_F32, du, CT_F32, wt, m, n, k, dx));
        CT_TRY(ct_binary(CT_ADD, CT_F32, part, CT_F32, dx, (uint64_t)(m * k), dx));
    }
    return CT_OK;
}

} // extern "C"
