"""Layer norm, the gated dense layer and the cross entropy of a dense layer: what holds whatever the number of rows, and the kernels
that only sizes beyond those of test_layers reach.  Definitions in 64 bits and bounds as there; tighter ones are derived here.
"""
import math

import numpy as np
import pytest

import camel_b200._lib as L
from camel_b200 import tensor as T
from test_layers import (GATES, U, ce64, ce_inputs, check_gated, check_gated_grad, dev, gate64, gated_grad64, gated_inputs, norm_bounds, norm_grad64,
                         norm_grad_bounds, norm_inputs, within)

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


@gpu
@pytest.mark.parametrize("rows", [600, 640])
@pytest.mark.parametrize("cols", [300, 400, 512, 700, 850, 1024, 1500, 2048, 2050, 3001, 4092, 5000, 8192])
def test_layer_norm_of_many_rows(rows, cols):
    """From four rows to an SM on a row has fewer threads."""
    x, gamma, beta, _ = norm_inputs(rows, cols, 55)
    y, _, _, _, off = norm_bounds(x, gamma, beta, 1e-5)
    within(T.layer_norm(dev(x), dev(gamma), dev(beta)).numpy(), y, off, "y")


@gpu
@pytest.mark.parametrize("rows,cols", [(300, 8193), (1000, 12345), (130, 40003), (1300, 500), (1300, 760), (1300, 890), (1300, 1000), (700, 7000)])
def test_layer_norm_grad_in_parts(rows, cols):
    """Rows above 8192 columns whose sums come from several parts; the forms of 1184 rows and more."""
    x, gamma, _, dy = norm_inputs(rows, cols, 56)
    want, off = norm_grad64(x, dy, gamma, 1e-5), norm_grad_bounds(x, dy, gamma, 1e-5, blocks=rows / 64)
    for name, a, b, c in zip(("dx", "dgamma", "dbeta"), T.layer_norm_grad(dev(x), dev(dy), dev(gamma)), want, off):
        within(a.numpy(), b, c, name)


# ---- gated dense layer: the kernels of larger sizes --------------------------------------------------


@gpu
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("m,k,n", [(1300, 130, 1100), (2100, 70, 523), (1281, 64, 1024), (5000, 33, 258)])
def test_dense_gated_on_pairs(m, k, n, gate):
    """Tiles of CTA pairs, each CTA of which has the columns of one matrix; ragged edges, with and without the sums kept."""
    x, wg, wu, bg, bu = gated_inputs(m, k, n, 57)
    check_gated(x, wg, wu, bg, bu, gate, keep=True)
    check_gated(x, wg, wu, None, bu, gate, keep=False)


@gpu
@pytest.mark.parametrize("n", [130, 260, 1030, 1500, 2050, 4100, 5504, 8192, 8300, 12290])
@pytest.mark.parametrize("m", [40, 700])
def test_dense_gated_grad_of_wide_layers(m, n):
    """Every form of the planes of d, rows that no block holds among them; without biases the other gradients have the same bytes."""
    k = 24
    x, wg, wu, _, _ = gated_inputs(m, k, n, 58)
    g, u, dout = (np.random.default_rng(i).normal(0, 1, (m, n)).astype(np.float32) for i in range(3))
    got = check_gated_grad(x, wg, wu, g, u, dout, "silu")
    alone = T.dense_gated_grad(*[dev(a) for a in (x, wg, wu, g, u, dout)], gate="silu")
    assert [a.numpy().tobytes() for a in alone] == [a.numpy().tobytes() for a in got[:3]]


@gpu
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("m", [8, 40, 200])
def test_slopes_at_the_ends(m, gate):
    """Where the exponential is 0 or its argument overflows, value and slope are their limits."""
    ends = np.array([-3e38, -1e30, -200.0, 200.0, 1e30, 3e38], np.float32)
    limit = {"sigmoid": (0, 1, 0, 0), "relu": (0, None, 0, 1), "silu": (0, None, 0, 1), "gelu": (0, None, 0, 1)}[gate]  # value and slope, below and above
    g = np.tile(ends, (m, 4))
    n = g.shape[1]
    one, x, w = np.ones((m, n), np.float32), np.zeros((m, 8), np.float32), np.zeros((8, n), np.float32)
    _, _, _, dbg, dbu = (a.numpy() for a in T.dense_gated_grad(*[dev(a) for a in (x, w, w, g, one, one)], gate=gate, bias=True))
    below, above = ends < 0, ends > 0
    for i in range(4):
        part = slice(6 * i, 6 * i + 6)
        assert (dbu[part][below] == m * limit[0]).all()
        assert (dbg[part][below] == m * limit[2]).all() and (dbg[part][above] == m * limit[3]).all()
        if limit[1] is not None:
            assert (dbu[part][above] == m * limit[1]).all()


# ---- cross entropy ----------------------------------------------------------------------------------


@gpu
@pytest.mark.parametrize("m", [2, 20, 200])
def test_cross_entropy_of_very_many_classes(m):
    """Sums of exponentials, of one size but for the target's: chains of at most 256 float32 terms."""
    import torch

    n = (1 << 24) + 40
    x, w = torch.ones(m, 1, device="cuda"), torch.full((1, n), -1.2, device="cuda")
    w[0, 7] = 0.0
    t = torch.full((m,), 7, device="cuda")
    loss, lse = torch.empty(m, device="cuda"), torch.empty(m, device="cuda")
    torch.cuda.synchronize()
    p = lambda a: a.data_ptr()  # noqa: E731
    L.check(L.lib.ct_dense_cross_entropy(p(x), p(w), None, p(t), m, 1, n, p(loss), p(lse)))
    T.check_async()
    want = np.log1p((n - 1) * np.exp(-np.float64(np.float32(1.2))))
    # a chain and the tree, exp and its argument, the logit of 1.2, the logarithm and the last addition
    off = U * (256 + 32 + 12) + 2 * U * 1.2 + 3 * U * want
    assert np.abs(lse.double().cpu().numpy() - want).max() <= off


# ---- sums over many rows --------------------------------------------------------------------------


def first_of_chains(m, pick):
    """Values that are half of a rounding beside one, and a one where a chain of sums begins: what follows it is lost to a chain that goes on."""
    import torch

    r = torch.arange(m, device="cuda")
    return torch.where(pick(r), 1.0, 2.0 ** -25)


@gpu
@pytest.mark.parametrize("m,n,pick", [(1 << 22, 250, lambda r: r < 4736), (1 << 20, 1000, lambda r: r < 592), (1 << 20, 2050, lambda r: r < 296),
                                      (1 << 17, 8200, lambda r: r % 10083 < 8)])
def test_gated_bias_gradients_of_many_rows(m, n, pick):
    """Float32 chains of at most 256 rows, which meet in 64 bits."""
    import torch

    k = 8
    x, w = torch.zeros(m, k, device="cuda"), torch.zeros(k, n, device="cuda")
    one = torch.ones(m, n, device="cuda")
    rows = first_of_chains(m, pick)
    dout = rows[:, None].expand(m, n).contiguous()
    db = torch.empty(2, n, device="cuda")
    torch.cuda.synchronize()
    p = lambda a: a.data_ptr()  # noqa: E731
    L.check(L.lib.ct_dense_gated_grad(p(x), p(w), p(w), p(one), p(one), p(dout), m, k, n, L.GATE_RELU, None, None, None, p(db[0]), p(db[1])))
    T.check_async()
    want = rows.double().sum().item()
    assert ((db.double() - want).abs() <= (256 + 32) * U * want).all()


@gpu
@pytest.mark.parametrize("m,k,n,chain,pick", [(1 << 23, 8, 32, 256, lambda r: r % 9447 < 8), (1 << 21, 16, 8, 1024, lambda r: (r % 8 == 0) & (r < 2368)),
                                              (1 << 21, 16, 12, 1024, lambda r: (r % 16 == 0) & (r < 2368)),
                                              (1 << 20, 1100, 8, 1024, lambda r: (r % 64 == 0) & (r < 118 * 64))])
def test_cross_entropy_gradients_of_many_rows(m, k, n, chain, pick):
    """db, and dw over few classes: float32 chains of at most `chain` rows."""
    import torch

    x, w, b = torch.ones(m, k, device="cuda"), torch.zeros(k, n, device="cuda"), torch.zeros(n, device="cuda")
    t = torch.zeros(m, device="cuda", dtype=torch.int64)
    lse = torch.full((m,), float(np.log(n)), device="cuda")
    dloss = first_of_chains(m, pick)
    dw, db = torch.empty_like(w), torch.empty_like(b)
    torch.cuda.synchronize()
    p = lambda a: a.data_ptr()  # noqa: E731
    L.check(L.lib.ct_dense_cross_entropy_grad(p(x), p(w), p(b), p(t), p(lse), p(dloss), m, k, n, None, p(dw), p(db)))
    T.check_async()
    want = dloss.double().sum().item() / n
    off = (chain + 32) * U + 2.0 ** -20  # and a probability: its exponent's rounding and its pair
    assert ((db[1:].double() - want).abs() <= off * want).all()
    if n <= 16:
        assert ((dw[:, 1:].double() - want).abs() <= off * want).all()


@gpu
def test_dimensions_that_are_too_large_are_refused_also_where_there_is_nothing_to_do():
    big, z = (1 << 29) + 1, None
    for rc in (L.lib.ct_dense_gated(z, z, z, z, z, 0, big, 4, 0, z, z, z), L.lib.ct_dense_gated_grad(z, z, z, z, z, z, 0, 1 << 33, 1 << 31, 0, z, z, z, z, z),
               L.lib.ct_dense_gated_grad(z, z, z, z, z, z, 4, big, 0, 0, z, z, z, z, z), L.lib.ct_layer_norm(z, z, z, 0, big, 1e-5, z),
               L.lib.ct_layer_norm(z, z, z, big, 0, 1e-5, z), L.lib.ct_layer_norm_grad(z, z, z, 0, big, 1e-5, z, z, z),
               L.lib.ct_dense_cross_entropy(z, z, z, z, 0, big, 4, z, z), L.lib.ct_dense_cross_entropy_grad(z, z, z, z, z, z, 0, 4, big, z, z, z)):
        assert rc == L.ERR_TOO_LARGE, L.lib.ct_last_error()


# ---- outputs that are not asked for, logits that are no numbers --------------------------------------


@gpu
@pytest.mark.parametrize("rows,cols", [(5, 40), (300, 200), (1300, 785), (300, 1024), (70, 3001), (40, 8193)])
def test_layer_norm_gradients_alone(rows, cols):
    x, gamma, _, dy = norm_inputs(rows, cols, 81)
    tx, td, g = dev(x), dev(dy), dev(gamma)
    want = [a.numpy().tobytes() for a in T.layer_norm_grad(tx, td, g)]
    for mask in range(1, 8):
        outs = [T.zeros([rows, cols]), T.zeros([cols]), T.zeros([cols])]
        p = [o.ptr if mask >> i & 1 else None for i, o in enumerate(outs)]
        L.check(L.lib.ct_layer_norm_grad(tx.ptr, g.ptr, td.ptr, rows, cols, 1e-5, *p))
        for i, o in enumerate(outs):
            assert o.numpy().tobytes() == want[i] if mask >> i & 1 else not o.numpy().any()


@gpu
@pytest.mark.parametrize("m,k,n", [(1, 40, 70), (16, 40, 70), (20, 40, 70), (40, 40, 2100), (200, 40, 70), (1300, 40, 1100)])
def test_dense_gated_keeps_what_is_asked_for(m, k, n):
    t = [dev(a) for a in gated_inputs(m, k, n, 82)]
    want = [a.numpy().tobytes() for a in T.dense_gated(*t, keep=True)]
    for mask in range(4):
        out, kept = T.zeros([m, n]), [T.zeros([m, n]), T.zeros([m, n])]
        p = [o.ptr if mask >> i & 1 else None for i, o in enumerate(kept)]
        L.check(L.lib.ct_dense_gated(t[0].ptr, t[1].ptr, t[3].ptr, t[2].ptr, t[4].ptr, m, k, n, L.GATE_SILU, out.ptr, *p))
        T.check_async()
        assert out.numpy().tobytes() == want[0]
        for i, o in enumerate(kept):
            assert o.numpy().tobytes() == want[1 + i] if mask >> i & 1 else not o.numpy().any()


CE_FORMS = [(1, 40, 70), (4, 40, 9000), (16, 40, 8), (20, 40, 70), (40, 40, 300), (64, 40, 4200), (200, 40, 300), (200, 40, 10), (1300, 40, 2100)]


@gpu
@pytest.mark.parametrize("m,k,n", CE_FORMS)
def test_cross_entropy_outputs_alone(m, k, n):
    x, w, b, t = (dev(a) for a in ce_inputs(m, k, n, 83))
    loss, lse = (a.numpy().tobytes() for a in T.dense_cross_entropy(x, w, t, b))
    one, other = T.zeros([m]), T.zeros([m])
    L.check(L.lib.ct_dense_cross_entropy(x.ptr, w.ptr, b.ptr, t.ptr, m, k, n, one.ptr, None))
    L.check(L.lib.ct_dense_cross_entropy(x.ptr, w.ptr, b.ptr, t.ptr, m, k, n, None, other.ptr))
    L.check(L.lib.ct_dense_cross_entropy(x.ptr, w.ptr, b.ptr, t.ptr, m, k, n, None, None))
    T.check_async()
    assert one.numpy().tobytes() == loss and other.numpy().tobytes() == lse


@gpu
@pytest.mark.parametrize("precision", ["3xtf32", "bf16"])
@pytest.mark.parametrize("m,k,n", CE_FORMS)
def test_logits_that_are_no_numbers(m, k, n, precision):
    """Biases of -infinity take classes out, all of them: lse -infinity; one of +infinity or NaN makes it NaN.  With any number of rows."""
    x, w, b, t = ce_inputs(m, k, n, 84)
    t[:] = n - 1
    L.check(L.lib.ct_set_precision(L.PREC_BF16 if precision == "bf16" else L.PREC_3XTF32))
    try:
        lse = lambda c: T.dense_cross_entropy(dev(x), dev(w), dev(t), dev(c))[1].numpy()  # noqa: E731
        assert np.isneginf(lse(np.full(n, -np.inf, np.float32))).all()
        only = np.full(n, -np.inf, np.float32)
        only[n // 2] = 1.0
        want = x.astype(np.float64) @ w[:, n // 2].astype(np.float64) + 1.0
        assert np.abs(lse(only) - want).max() <= 0.2  # bfloat16: 2^-7 of sum |x||w|
        for bad in (np.inf, np.nan):
            c = b.copy()
            c[n // 3] = bad
            assert np.isnan(lse(c)).all()
    finally:
        L.check(L.lib.ct_set_precision(L.PREC_3XTF32))
