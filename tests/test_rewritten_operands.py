"""Buffers that are read, rewritten and read again, by kernels that follow one another without a pause: the second reading sees the second
values.  Kernels are launched early (programmatic dependent launch), so three of them may be on the machine at once."""
import numpy as np
import pytest

import camel_b200._lib as L
from camel_b200 import tensor as T

gpu = pytest.mark.gpu
TIMES = 40


@gpu
@pytest.mark.parametrize("m,k,n", [(1462, 652, 10), (1605, 1017, 11), (1462, 652, 8), (1000, 400, 4), (600, 300, 16), (1462, 652, 17), (8, 652, 300),
                                   (300, 300, 300), (2000, 512, 64), (5000, 785, 10)])
def test_product_of_a_transposed_operand_twice(m, k, n):
    """As a gradient does: both weights' transposed copies in one buffer, one after the other."""
    rng = np.random.default_rng(m + n)
    a, first, second = (T.from_numpy(rng.normal(0, 1, s).astype(np.float32)) for s in ((m, k), (n, k), (n, k)))
    turned, one, two = T.zeros([k, n]), T.zeros([m, n]), T.zeros([m, n])

    def run(wait):
        for w, out in ((first, one), (second, two)):
            L.check(L.lib.ct_transpose(L.F32, w.ptr, n, k, turned.ptr))
            if wait:
                T.sync()
            L.check(L.lib.ct_matmul(L.F32, a.ptr, L.F32, turned.ptr, m, k, n, out.ptr))
            if wait:
                T.sync()
        return one.numpy().tobytes(), two.numpy().tobytes()

    want = run(True)
    assert [run(False) == want for _ in range(TIMES)] == [True] * TIMES


def operators(rng, m, k, n):
    """name -> (calls of an operator on the shared buffers, its outputs)"""
    f = lambda *s: T.from_numpy(rng.normal(0, 0.2, s).astype(np.float32))  # noqa: E731
    z = lambda *s: T.zeros(list(s))  # noqa: E731
    x, w, wu, b, dy = f(m, k), f(k, n), f(k, n), f(n), f(m, n)
    t = T.from_numpy(rng.integers(-1, n, m))
    lse = T.from_numpy(np.full(m, 30.0, np.float32))
    out, g, u, dx, dw, dwu, db, dbu, row = z(m, n), z(m, n), z(m, n), z(m, k), z(k, n), z(k, n), z(n), z(n), z(m)
    gamma, dg, dbeta, y, yy = f(k), z(k), z(k), z(m, k), z(m, k)
    p = L.lib
    return {
        "dense": ([x, w, b], lambda: p.ct_dense(x.ptr, w.ptr, b.ptr, m, k, n, L.ACT_RELU, out.ptr, None), [out]),
        "matmul": ([x, w], lambda: p.ct_matmul(L.F32, x.ptr, L.F32, w.ptr, m, k, n, out.ptr), [out]),
        "matmul_tn": ([x, dy], lambda: p.ct_matmul_tn(x.ptr, dy.ptr, k, m, n, dw.ptr), [dw]),
        "sum_axis": ([x], lambda: p.ct_sum_axis(L.F32, x.ptr, m, k, 0, dg.ptr), [dg]),
        "softmax": ([x], lambda: p.ct_softmax_rows(x.ptr, m, k, y.ptr), [y]),
        "layer_norm": ([x, gamma], lambda: p.ct_layer_norm(x.ptr, gamma.ptr, None, m, k, 1e-5, y.ptr), [y]),
        "layer_norm_grad": ([x, gamma], lambda: p.ct_layer_norm_grad(x.ptr, gamma.ptr, yy.ptr, m, k, 1e-5, dx.ptr, dg.ptr, dbeta.ptr), [dx, dg, dbeta]),
        "dense_gated": ([x, w, wu, b], lambda: p.ct_dense_gated(x.ptr, w.ptr, b.ptr, wu.ptr, b.ptr, m, k, n, L.GATE_SILU, out.ptr, g.ptr, u.ptr), [out, g, u]),
        "dense_gated_grad": ([x, w, wu, dy], lambda: p.ct_dense_gated_grad(x.ptr, w.ptr, wu.ptr, dy.ptr, dy.ptr, dy.ptr, m, k, n, L.GATE_SILU, dx.ptr, dw.ptr,
                                                                           dwu.ptr, db.ptr, dbu.ptr), [dx, dw, dwu, db, dbu]),
        "cross_entropy": ([x, w, b], lambda: p.ct_dense_cross_entropy(x.ptr, w.ptr, b.ptr, t.ptr, m, k, n, row.ptr, lse.ptr), [row, lse]),
        "cross_entropy_grad": ([x, w, b], lambda: p.ct_dense_cross_entropy_grad(x.ptr, w.ptr, b.ptr, t.ptr, lse.ptr, None, m, k, n, dx.ptr, dw.ptr, db.ptr),
                               [dx, dw, db]),
    }


NAMES = ["dense", "matmul", "matmul_tn", "sum_axis", "softmax", "layer_norm", "layer_norm_grad", "dense_gated", "dense_gated_grad", "cross_entropy",
         "cross_entropy_grad"]


@gpu
@pytest.mark.parametrize("precision", ["3xtf32", "bf16"])
@pytest.mark.parametrize("m,k,n", [(1462, 652, 10), (4, 300, 70), (40, 200, 130), (300, 200, 260), (1500, 64, 12)])
@pytest.mark.parametrize("name", NAMES)
def test_operator_on_rewritten_inputs(name, m, k, n, precision):
    """The operator, its inputs doubled in place, the operator again: the same bytes as with pauses between."""
    L.check(L.lib.ct_set_precision(L.PREC_BF16 if precision == "bf16" else L.PREC_3XTF32))
    try:
        inputs, call, outputs = operators(np.random.default_rng(m + k + n), m, k, n)[name]
        kept = [a.numpy() for a in inputs]

        def run(wait):
            for a, v in zip(inputs, kept):
                L.check(L.lib.ct_h2d(a.ptr, v.ctypes.data, v.nbytes))
            L.check(call())
            for a in inputs:
                if wait:
                    T.sync()
                L.check(L.lib.ct_binary(L.ADD, L.F32, a.ptr, L.F32, a.ptr, a.numel, a.ptr))
            if wait:
                T.sync()
            L.check(call())
            T.check_async()
            return [o.numpy().tobytes() for o in outputs]

        want = run(True)
        assert [run(False) == want for _ in range(10)] == [True] * 10
    finally:
        L.check(L.lib.ct_set_precision(L.PREC_3XTF32))
