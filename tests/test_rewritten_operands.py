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


# ---- sequences of operators over a few buffers ---------------------------------------------------------

QUARTER = 1 << 18  # values; a buffer has four, an operator's operands are different quarters of different buffers


def size(rng, most):
    return max(1, int(round(np.exp(rng.uniform(0, np.log(most))))))


def dimensions(rng):
    while True:
        m, k, n = size(rng, 3000), size(rng, 900), rng.integers(1, 18) if rng.uniform() < 0.3 else size(rng, 900)
        if max(m * k, k * n, m * n) <= QUARTER:
            return int(m), int(k), int(n)


def any_call(rng, buffers, targets):
    """One operator with operands and outputs in the buffers, no output over an operand except where operators allow it."""
    i, j, l, o = rng.permutation(len(buffers))[:4]
    m, k, n = dimensions(rng)
    at = lambda b, quarter=0: buffers[b].ptr + quarter * QUARTER * 4  # noqa: E731
    x, w, v, out = at(i), at(j, 1), at(l, 2), [at(o, q) for q in range(4)]
    act, p, f = int(rng.integers(0, 3)), L.lib, L.F32
    return [
        lambda: p.ct_transpose(f, x, k, n, out[0]),
        lambda: p.ct_matmul(f, x, f, w, m, k, n, out[0]),
        lambda: p.ct_matmul_tn(x, w, k, m, n, out[0]),
        lambda: p.ct_dense(x, w, v, m, k, n, act, out[0], None),
        lambda: p.ct_sum_axis(f, x, m, k, act & 1, out[0]),
        lambda: p.ct_binary(L.ADD, f, x, f, w, m * k, out[0]),
        lambda: p.ct_binary(L.ADD, f, x, f, w, m * k, x),
        lambda: p.ct_relu(x, m * k, out[0]),
        lambda: p.ct_softmax_rows(x, m, k, out[0]),
        lambda: p.ct_scaled_sub(x, w, 0.1, m * k, out[0]),
        lambda: p.ct_fill(f, 0.25, m, out[0]),
        lambda: p.ct_layer_norm(x, w, None, m, k, 1e-5, out[0]),
        lambda: p.ct_layer_norm(x, None, None, m, k, 1e-5, x),
        lambda: p.ct_layer_norm_grad(x, w, v, m, k, 1e-5, out[0], out[1], out[2]),
        lambda: p.ct_dense_gated(x, w, None, v, None, m, k, n, L.GATE_SILU, out[0], out[1], out[2]),
        lambda: p.ct_dense_gated_grad(x, w, v, at(i, 3), at(j, 3), at(l, 3), m, k, n, L.GATE_SILU, *out, out[3] + 4 * n),
        lambda: p.ct_dense_cross_entropy(x, w, None, targets.ptr, m, k, n, out[0], out[1]),
        lambda: p.ct_dense_cross_entropy_grad(x, w, None, targets.ptr, v, None, m, k, n, out[0], out[1], out[2]),
    ][int(rng.integers(0, 18))]


@gpu
@pytest.mark.parametrize("precision", ["3xtf32", "bf16"])
@pytest.mark.parametrize("seed", range(4))
def test_sequences_without_pauses(seed, precision):
    """Sequences of up to 14 operators leave the same bytes in all buffers as with a pause behind each, and recorded and replayed, too."""
    rng = np.random.default_rng(seed)
    first = [T.from_numpy(rng.normal(0, 0.3, 4 * QUARTER).astype(np.float32)) for _ in range(5)]
    buffers, kept = [T.zeros([4 * QUARTER]) for _ in first], [T.zeros([4 * QUARTER]) for _ in first]
    targets = T.from_numpy(rng.integers(-1, 300, 4096))

    def copy(to, source):
        for a, b in zip(to, source):
            L.check(L.lib.ct_d2d(a.ptr, b.ptr, a.nbytes))
        T.sync()

    def same():
        equal = [T.Tensor(L.BOOL, (2 * QUARTER,)) for _ in buffers]
        for e, a, b in zip(equal, buffers, kept):  # two values as an int64: NaN equals itself
            L.check(L.lib.ct_compare(L.EQ, L.I64, a.ptr, L.I64, b.ptr, 2 * QUARTER, e.ptr))
        return all(e.numpy().all() for e in equal)

    L.check(L.lib.ct_set_precision(L.PREC_BF16 if precision == "bf16" else L.PREC_3XTF32))
    try:
        for number in range(200):
            calls = [any_call(rng, buffers, targets) for _ in range(int(rng.integers(3, 15)))]
            copy(buffers, first)
            for call in calls:
                L.check(call())
                T.sync()
            copy(kept, buffers)
            for again in range(3):
                copy(buffers, first)
                for call in calls:
                    L.check(call())
                T.check_async()
                assert same(), (number, again)
            with T.Graph() as graph:
                for call in calls:
                    L.check(call())
            copy(buffers, first)
            graph.launch()
            T.check_async()
            assert same(), (number, "recorded")
            del graph  # not while the next one records
    finally:
        L.check(L.lib.ct_set_precision(L.PREC_3XTF32))
