"""Layer norm, the gated dense layer and the cross entropy of a dense layer: what holds whatever the number of rows, and the kernels
that only sizes beyond those of test_layers reach.  Definitions in 64 bits and bounds as there; tighter ones are derived here.
"""
import numpy as np
import pytest

import camel_b200._lib as L
from camel_b200 import tensor as T
from test_layers import U, ce_inputs, dev, gated_inputs, norm_inputs

gpu = pytest.mark.gpu


# ---- values that are no numbers -------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("precision", ["3xtf32", "bf16"])
@pytest.mark.parametrize("m,k,n", [(5, 40, 70), (16, 40, 70), (40, 40, 70), (200, 40, 70), (200, 40, 300), (1500, 33, 70)])
def test_gated_rows_of_zero_gradient_count(m, k, n, precision):
    """0 x NaN is a term of dw like any other, with any number of rows: x that is no number shows in its row of dw, and only there."""
    x, wg, wu, _, _ = gated_inputs(m, k, n, 51)
    g, u, dout = (np.random.default_rng(i).normal(0, 1, (m, n)).astype(np.float32) for i in range(3))
    dout[3] = 0.0
    x[3, 7], x[3, 9] = np.nan, np.inf
    L.check(L.lib.ct_set_precision(L.PREC_BF16 if precision == "bf16" else L.PREC_3XTF32))
    try:
        dx, dwg, dwu = (a.numpy() for a in T.dense_gated_grad(*[dev(a) for a in (x, wg, wu, g, u, dout)]))
    finally:
        L.check(L.lib.ct_set_precision(L.PREC_3XTF32))
    assert not dx[3].any() and np.isfinite(dx).all()
    rest = [c for c in range(k) if c not in (7, 9)]
    for dw in (dwg, dwu):
        assert np.isnan(dw[[7, 9]]).all() and np.isfinite(dw[rest]).all()


@gpu
@pytest.mark.parametrize("m,k,n", [(5, 40, 70), (40, 40, 70), (200, 40, 70), (200, 40, 24), (200, 40, 10), (200, 1100, 10)])
def test_cross_entropy_rows_of_zero_weight_count(m, k, n):
    """A row with a target and dloss = 0, where x holds a NaN: so are its logits, and 0 x NaN is a term of all sums over rows.  Without a
    target it is none."""
    x, w, b, t = ce_inputs(m, k, n, 52)
    t = np.abs(t) % n
    lse = T.dense_cross_entropy(dev(x), dev(w), dev(t), dev(b))[1]
    x[3, 7] = np.nan
    dloss = np.ones(m, np.float32)
    dloss[3] = 0.0
    dx, dw, db = (a.numpy() for a in T.dense_cross_entropy_grad(dev(x), dev(w), dev(t), lse, dev(b), dev(dloss)))
    rest = [r for r in range(m) if r != 3]
    assert np.isnan(dx[3]).all() and np.isfinite(dx[rest]).all() and np.isnan(dw).all() and np.isnan(db).all()
    t[3] = -1
    dx, dw, db = (a.numpy() for a in T.dense_cross_entropy_grad(dev(x), dev(w), dev(t), lse, dev(b), dev(dloss)))
    assert not dx[3].any() and not np.signbit(dx[3]).any() and np.isfinite(dx).all() and np.isfinite(dw).all() and np.isfinite(db).all()


@gpu
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("m,k,n", [(5, 40, 70), (40, 40, 70), (200, 40, 70), (200, 40, 10), (1500, 33, 300)])
def test_cross_entropy_weights_that_are_no_numbers(m, k, n, bad):
    """dloss that is NaN or infinite shows in its row of dx, also where the weights are zero, and in all of dw and db; other rows keep theirs."""
    x, w, b, t = ce_inputs(m, k, n, 53)
    t = np.abs(t) % n
    w[5] = 0.0
    lse = T.dense_cross_entropy(dev(x), dev(w), dev(t), dev(b))[1]
    dloss = np.ones(m, np.float32)
    clean = [a.numpy() for a in T.dense_cross_entropy_grad(dev(x), dev(w), dev(t), lse, dev(b), dev(dloss))]
    dloss[3] = bad
    dx, dw, db = (a.numpy() for a in T.dense_cross_entropy_grad(dev(x), dev(w), dev(t), lse, dev(b), dev(dloss)))
    rest = [r for r in range(m) if r != 3]
    assert (np.isnan(dx[3]).all() if np.isnan(bad) else not np.isfinite(dx[3]).any()) and not np.isfinite(dw).any() and not np.isfinite(db).any()
    assert np.abs(dx[rest] - clean[0][rest]).max() <= 1e-6 * np.abs(clean[0]).max()


# ---- layer norm -----------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("rows,cols", [(70, 785), (300, 4096), (3, 8193), (300, 8193), (40, 12345)])
@pytest.mark.parametrize("over", ["x", "dout"])
def test_layer_norm_grad_over_an_input(rows, cols, over):
    """dx in the place of x or of dout, with the columns' sums of both: the same bytes as beside them."""
    x, gamma, _, dy = norm_inputs(rows, cols, 54)
    want = [a.numpy() for a in T.layer_norm_grad(dev(x), dev(dy), dev(gamma))]
    tx, td, g = dev(x), dev(dy), dev(gamma)
    to = tx if over == "x" else td
    dg, db = T.zeros([cols]), T.zeros([cols])
    L.check(L.lib.ct_layer_norm_grad(tx.ptr, g.ptr, td.ptr, rows, cols, 1e-5, to.ptr, dg.ptr, db.ptr))
    for a, b in zip((to, dg, db), want):
        assert a.numpy().tobytes() == b.tobytes()


@gpu
@pytest.mark.parametrize("rows,cols,chain", [(1 << 26, 4, 256), (600000, 96, 256), (40000, 8193, 64), (300000, 8200, 64)])
def test_layer_norm_grad_sums_of_many_rows(rows, cols, chain):
    """Float32 sums of at most `chain` rows (up to 32 of them again), then 64 bits: beside ones, values that are half of a rounding each
    are lost to a sum that goes on."""
    import torch

    if rows * cols > 1 << 30:
        rows = (1 << 30) // cols
    x = torch.randn(rows, cols, device="cuda")
    dy = torch.full((rows, cols), 2.0 ** -25, device="cuda")
    if cols <= 8192:
        dy[:40000] = 1.0  # the first rows of all blocks
    else:
        dy[::max(8, -(-rows * -(-cols // 256) // 1184))] = 1.0  # of all parts
    dg, db = torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    torch.cuda.synchronize()
    L.check(L.lib.ct_layer_norm_grad(x.data_ptr(), None, dy.data_ptr(), rows, cols, 1e-5, None, dg.data_ptr(), db.data_ptr()))
    T.check_async()
    want = torch.stack([part.double().sum(0) for part in dy.split(1 << 20)]).sum(0)
    assert ((db.double() - want).abs() <= (chain + 32) * U * want).all()


@gpu
@pytest.mark.parametrize("cols", [1 << 17, (1 << 25) + 3])
def test_layer_norm_of_very_long_rows(cols):
    """Sums of at most 64 values, then 64 bits, then a tree of ten: squares of one size do not stop to count."""
    import torch

    x = torch.full((2, cols), 0.3, device="cuda")
    x[:, ::2] = -0.3
    x[1, 5] = 1000.0
    dy = torch.randn(2, cols, device="cuda")
    out, dx = torch.empty_like(x), torch.empty_like(x)
    torch.cuda.synchronize()
    L.check(L.lib.ct_layer_norm(x.data_ptr(), None, None, 2, cols, 1e-5, out.data_ptr()))
    L.check(L.lib.ct_layer_norm_grad(x.data_ptr(), None, dy.data_ptr(), 2, cols, 1e-5, dx.data_ptr(), None, None))
    T.check_async()
    d, g = x.double(), dy.double()
    d -= d.mean(1, keepdim=True)
    r = 1 / (d.square().mean(1, keepdim=True) + float(np.float32(1e-5))).sqrt()
    h = d * r
    depth = 64 + 12
    off_h = U * ((depth / 2 + 10) * h.abs() + (depth + 2) * d.abs().mean(1, keepdim=True) * r)
    assert ((out.double() - h).abs() <= off_h).all()
    mean_g, mean_gh = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    want = r * (g - mean_g - h * mean_gh)
    mixed = (g.abs() * (h.abs() + 1)).mean(1, keepdim=True)
    off = r * U * ((depth + 16) * (g.abs() + g.abs().mean(1, keepdim=True)) + 3 * (depth + 16) * (h.abs() + 1) * mixed)
    assert ((dx.double() - want).abs() <= off).all()
