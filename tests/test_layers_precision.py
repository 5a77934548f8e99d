"""Products of the gated layer and of the cross entropy at the bounds that the header gives, and under the reduced precision.

A pair of float16 holds a value to 2^-23 of itself, and to 2^-50 of its line's largest where that is more (below 2^-27 of it); the product
of two low terms is left out: 2^-22 of the product of the values, 2^-50 of that of the largest.  So the terms of a product are off by
2^-21 sum |a||b| and, of values that a line's largest outweighs, by 2^-48 k max|a| max|b| (SMALL).  The tensor core truncates a sum once per 16
values of k (2^-23 of it); the leading sum is drained every 128 values (256 at first) and goes on in float32, up to 32 slices are
added to one another; the cross products, 2^-10 of the leading ones, are not drained (two additions per 16 values).
"""
import numpy as np
import pytest

import camel_b200._lib as L
from camel_b200 import tensor as T
from test_layers import GATES, U, ce64, ce_inputs, dev, gate64, gated_grad64, gated_inputs, within

gpu = pytest.mark.gpu


def SUM(k):
    return 2.0 ** -21 + 17 * 2.0 ** -23 + (k / 128 + 34) * U + k / 8 * 2.0 ** -33


def SMALL(k, a, b):
    """a: the largest of each row of the result's left lines, b: of each column's."""
    return 2.0 ** -48 * k * a[:, None] * b[None, :]


def f64(*arrays):
    return [a.astype(np.float64) for a in arrays]


def most(a, axis):
    return np.abs(a).max(axis, initial=0).astype(np.float64)


@gpu
@pytest.mark.parametrize("m,k,n", [(20, 20000, 70), (100, 9000, 130), (200, 20000, 70), (1300, 5000, 1100)])
def test_long_sums_of_one_sign(m, k, n):
    """Nothing cancels, and every truncation of a sum is towards zero: without the draining 9e-6 at k = 5000."""
    rng = np.random.default_rng(k)
    x, w, v = (rng.uniform(0.5, 1, s).astype(np.float32) for s in ((m, k), (k, n), (k, n)))
    _, g, u = (a.numpy() for a in T.dense_gated(dev(x), dev(w), dev(v), keep=True))
    T.check_async()
    for got, b in ((g, w), (u, v)):
        want = np.matmul(*f64(x, b))
        within(got, want, SUM(k) * want + U * want, "kept sum")


@gpu
@pytest.mark.parametrize("m,k,n", [(20000, 40, 70), (40, 70, 20000), (300, 70, 9000)])
def test_long_sums_of_one_sign_on_the_way_back(m, k, n):
    rng = np.random.default_rng(m + n)
    x, wg, wu = (rng.uniform(0.5, 1, s).astype(np.float32) for s in ((m, k), (k, n), (k, n)))
    g, u, dout = (rng.uniform(0.5, 1, (m, n)).astype(np.float32) for _ in range(3))
    dx, dwg, dwu = (a.numpy() for a in T.dense_gated_grad(*[dev(a) for a in (x, wg, wu, g, u, dout)], gate="relu"))
    T.check_async()
    (wdx, wdwg, wdwu, _, _), _, _ = gated_grad64(x, wg, wu, g, u, dout, "relu")  # dg = dout u, du = dout g: a rounding each
    within(dx, wdx, (SUM(2 * n) + 3 * U) * wdx, "dx")
    within(dwg, wdwg, (SUM(m) + 3 * U) * wdwg, "dw_gate")
    within(dwu, wdwu, (SUM(m) + 3 * U) * wdwu, "dw_up")


def wide(rng, shape, decades):
    return (rng.normal(0, 1, shape) * 10.0 ** rng.uniform(-decades, decades, shape)).astype(np.float32)


@gpu
@pytest.mark.parametrize("decades", [2, 6, 12])
@pytest.mark.parametrize("m,k,n", [(20, 100, 70), (100, 300, 130), (200, 100, 70), (1300, 64, 1100)])
def test_lines_of_many_magnitudes(m, k, n, decades):
    """Values of one line up to 24 decades apart, in both operands."""
    rng = np.random.default_rng(decades + m)
    x, wg, wu = wide(rng, (m, k), decades), wide(rng, (k, n), decades), wide(rng, (k, n), decades)
    _, g, u = (a.numpy() for a in T.dense_gated(dev(x), dev(wg), dev(wu), keep=True))
    T.check_async()
    for got, w in ((g, wg), (u, wu)):
        a, b = f64(x, w)
        within(got, a @ b, (SUM(k) + U) * (np.abs(a) @ np.abs(b)) + SMALL(k, most(x, 1), most(w, 0)), "kept sum")


@gpu
@pytest.mark.parametrize("decades", [2, 6])
@pytest.mark.parametrize("m,k,n", [(20, 100, 70), (100, 30, 1030), (200, 100, 70), (1300, 64, 300)])
def test_gradients_of_many_magnitudes(m, k, n, decades):
    """Rows of d = [dg | du] have a scale each, which x takes over."""
    rng = np.random.default_rng(decades + m + 1)
    x, wg, wu, dout = wide(rng, (m, k), decades), wide(rng, (k, n), decades), wide(rng, (k, n), decades), wide(rng, (m, n), decades)
    g, u = (rng.normal(0, 1, (m, n)).astype(np.float32) for _ in range(2))
    got = [a.numpy() for a in T.dense_gated_grad(*[dev(a) for a in (x, wg, wu, g, u, dout)], gate="sigmoid", bias=True)]
    T.check_async()
    (dx, dwg, dwu, dbg, dbu), dg, du = gated_grad64(x, wg, wu, g, u, dout, "sigmoid")
    ax, ag, au, d64, u64 = [np.abs(a) for a in f64(x, wg, wu, dout, u)]
    s = gate64("sigmoid", g.astype(np.float64))
    off_g, off_u = 12 * U * d64 * u64 * s[1], 8 * U * d64 * s[0]  # the slope is a product of both sides, to 4 U each
    top = np.maximum(most(dg, 1), most(du, 1))
    xt = ax * top[:, None]  # x as it meets d under its rows' scales
    small = 2.0 ** -49 * (xt.sum(0) + m * xt.max(0))[:, None]
    bounds = ((SUM(2 * n) + U) * (np.abs(dg) @ ag.T + np.abs(du) @ au.T) + off_g @ ag.T + off_u @ au.T + SMALL(2 * n, top, np.maximum(most(wg, 1), most(wu, 1))),
              (SUM(m) + 2 * U) * (ax.T @ np.abs(dg)) + ax.T @ off_g + small, (SUM(m) + 2 * U) * (ax.T @ np.abs(du)) + ax.T @ off_u + small,
              (m + 16) * U * np.abs(dg).sum(0) + off_g.sum(0), (m + 16) * U * np.abs(du).sum(0) + off_u.sum(0))
    for name, a, b, c in zip(("dx", "dw_gate", "dw_up", "db_gate", "db_up"), got, (dx, dwg, dwu, dbg, dbu), bounds):
        within(a, b, c + 1e-300, name)


def ce_grad_at_bounds(x, w, b, t, lse, small=2.0 ** -50):
    """small: what d / dloss is held to where 2^-23 of itself is less."""
    m, k, n = x.shape[0], x.shape[1], w.shape[1]
    z, _, _, has, at, _ = ce64(x, w, b, t)
    ax, aw = [np.abs(a) for a in f64(x, w)]
    # the logits of the weights' planes by rows: x with their scales folded in, a line per row of x
    top = ax * most(w, 1)[None, :]
    off_z = (SUM(k) + U) * (ax @ aw) + 2 * U * (np.abs(z) + np.abs(b)) + 2.0 ** -48 * k * top.max(1)[:, None]
    got = [a.numpy() for a in T.dense_cross_entropy_grad(dev(x), dev(w), dev(t), dev(lse), dev(b))]
    T.check_async()
    l64 = lse.astype(np.float64)[:, None]
    p = np.exp(z - l64) * has[:, None]
    d = p.copy()
    d[np.arange(m)[has], at[has]] -= 1.0
    # a probability: its logit, the difference, the exponent's product and constant (a rounding each of |z - lse|), 2^-22 of exp and 2 U
    off_d = p * (np.expm1(off_z + 4 * U * np.abs(z - l64)) + 6 * U) + small * has[:, None]
    off_d[np.arange(m)[has], at[has]] += U
    off_d += 2 * U * np.abs(d)
    ad, top = np.abs(d), most(w, 1)
    want = [d @ w.astype(np.float64).T, x.astype(np.float64).T @ d, d.sum(0)]
    # x' has a scale per column, d one for all
    bounds = [(SUM(n) + 4 * U) * (ad @ aw.T) + off_d @ aw.T + 2.0 ** -49 * ad.sum(1)[:, None] * top[None, :],
              (SUM(m) + 4 * U) * (ax.T @ ad) + ax.T @ off_d + 2.0 ** -49 * most(x, 0)[:, None] * ad.sum(0)[None, :], (m + 16) * U * ad.sum(0) + off_d.sum(0)]
    for name, a, c, e in zip(("dx", "dw", "db"), got, want, bounds):
        within(a, c, e, name)
    return got, want


@gpu
@pytest.mark.parametrize("m,k,n", [(12, 48, 300), (40, 48, 300), (200, 48, 300), (200, 48, 24), (200, 48, 12), (1300, 40, 1500)])
@pytest.mark.parametrize("gap", [10.0, 20.0, 28.0])
def test_cross_entropy_gradient_of_confident_rows(m, k, n, gap):
    """The targets' logits stand out by 10 to 28: the probabilities of all other classes are 2^-14 to 2^-40, in every row."""
    x, w, b, t = ce_inputs(m, k, n, 61, scale=0.2)
    t = np.where(t >= 0, t % 3, t)
    t[1], t[2] = 0, 2
    w[:, :3] = 0.0
    b[:] *= 0.1
    b[:3] = 0.0
    for c in range(3):  # column c of x marks the rows of class c
        x[:, c] = np.where(t == c, 1.0, 0.0)
        w[c] = 0.0
        w[c, c] = gap
    lse = ce64(x, w, b, t)[1].astype(np.float32)
    got, want = ce_grad_at_bounds(x, w, b, t, lse)
    if gap == 10.0:  # there everything keeps its digits, also of the small classes
        assert np.abs(got[2][3:] - want[2][3:]).max() <= 2e-5 * np.abs(want[2][3:]).max()


@gpu
@pytest.mark.parametrize("m,n", [(12, 64), (40, 64), (200, 64), (40, 12)])
def test_probabilities_up_to_four(m, n):
    """lse smaller than the logits': exp(z - lse) up to 3.99 is what d is computed from."""
    x, w = np.random.default_rng(1).normal(0, 1, (m, 32)).astype(np.float32), np.zeros((32, n), np.float32)
    w[4] = 1e-3
    t = np.arange(m) % n
    ce_grad_at_bounds(x, w, np.zeros(n, np.float32), t, np.full(m, -np.log(3.97), np.float32))


# ---- the reduced precision ----------------------------------------------------------------------------


@pytest.fixture
def bf16():
    L.check(L.lib.ct_set_precision(L.PREC_BF16))
    yield
    L.check(L.lib.ct_set_precision(L.PREC_3XTF32))


HALF = 2.0 ** -8 * 2 + 2.0 ** -16 + 2.0 ** -14  # both operands rounded to bfloat16; sums of up to 2^13 values, truncated once per 16


@gpu
@pytest.mark.parametrize("gate", GATES)
@pytest.mark.parametrize("m,k,n", [(5, 33, 70), (40, 100, 64), (300, 64, 200), (1500, 40, 130)])
def test_bf16_gated_gradient(bf16, gate, m, k, n):
    x, wg, wu, _, _ = gated_inputs(m, k, n, 62)
    g, u, dout = (np.random.default_rng(i).normal(0, 1, (m, n)).astype(np.float32) for i in range(3))
    got = [a.numpy() for a in T.dense_gated_grad(*[dev(a) for a in (x, wg, wu, g, u, dout)], gate=gate, bias=True)]
    T.check_async()
    want, dg, du = gated_grad64(x, wg, wu, g, u, dout, gate)
    ax, ag, au = [np.abs(a) for a in f64(x, wg, wu)]
    dg, du = np.abs(dg), np.abs(du)
    d64 = np.abs(dout.astype(np.float64))
    tiny = 16 * U * (d64 * np.abs(u) * 1.2)  # a slope's roundings, where it is small as a difference
    bounds = (HALF * (dg @ ag.T + du @ au.T) + tiny @ ag.T, HALF * (ax.T @ dg) + ax.T @ tiny, HALF * (ax.T @ du), (m + 16) * U * dg.sum(0) + tiny.sum(0),
              (m + 24) * U * du.sum(0))
    for name, a, b, c in zip(("dx", "dw_gate", "dw_up", "db_gate", "db_up"), got, want, bounds):
        within(a, b, c + 1e-30, name)


@gpu
@pytest.mark.parametrize("m,k,n", [(5, 33, 70), (40, 100, 300), (300, 64, 200), (1300, 40, 17), (300, 64, 10)])
def test_bf16_cross_entropy_gradient(bf16, m, k, n):
    x, w, b, t = ce_inputs(m, k, n, 63)
    dloss = np.random.default_rng(3).uniform(0.5, 1, m).astype(np.float32)
    z, lse, _, has, at, _ = ce64(x, w, b, t)
    got = [a.numpy() for a in T.dense_cross_entropy_grad(dev(x), dev(w), dev(t), dev(lse.astype(np.float32)), dev(b), dev(dloss))]
    T.check_async()
    ax, aw = [np.abs(a) for a in f64(x, w)]
    weight = np.where(has, dloss.astype(np.float64), 0.0)[:, None]
    p = np.exp(z - lse[:, None])
    d = p.copy()
    d[np.arange(m), at] -= 1.0
    d, off = d * weight, weight * (p * (np.expm1(HALF * (ax @ aw)) + 1e-5) + 4 * U)
    ad = np.abs(d) + off
    want = (d @ w.astype(np.float64).T, x.astype(np.float64).T @ d, d.sum(0))
    bounds = (HALF * (ad @ aw.T) + off @ aw.T, HALF * (ax.T @ ad) + ax.T @ off, (m + 16) * U * ad.sum(0) + off.sum(0))
    for name, a, c, e in zip(("dx", "dw", "db"), got, want, bounds):
        within(a, c, e, name)


@gpu
def test_bf16_cross_entropy_in_pieces_of_rows(bf16):
    """More logits than are held at a time (2^28): dw and db are added up over the pieces."""
    import torch

    m, k, n = 2100, 16, 131072
    gen = torch.Generator(device="cuda").manual_seed(64)
    x, w, b = (torch.randn(*s, device="cuda", generator=gen) * f for s, f in (((m, k), 1.0), ((k, n), 0.5), ((n,), 0.3)))
    x, w = x.bfloat16().float(), w.bfloat16().float()  # nothing to round in the logits
    t = torch.randint(n, (m,), device="cuda", generator=gen)
    t[::7] = -1
    loss, lse, dx, dw, db = torch.empty(m, device="cuda"), torch.empty(m, device="cuda"), torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    torch.cuda.synchronize()
    p = lambda a: a.data_ptr()  # noqa: E731
    L.check(L.lib.ct_dense_cross_entropy(p(x), p(w), p(b), p(t), m, k, n, p(loss), p(lse)))
    L.check(L.lib.ct_dense_cross_entropy_grad(p(x), p(w), p(b), p(t), p(lse), None, m, k, n, p(dx), p(dw), p(db)))
    T.check_async()
    xd, wd, bd = x.double(), w.double(), b.double()
    rdw, rdb, adw, adb = torch.zeros_like(wd), torch.zeros_like(bd), torch.zeros_like(wd), torch.zeros_like(bd)
    for i in range(0, m, 300):
        z = xd[i:i + 300] @ wd + bd
        l64 = torch.logsumexp(z, 1)
        assert (lse[i:i + 300].double() - l64).abs().max() <= 1e-5
        has = t[i:i + 300] >= 0
        d = (z - l64[:, None]).exp() * has[:, None]
        rows = torch.nonzero(has)[:, 0]
        d[rows, t[i:i + 300][rows]] -= 1.0
        rdx = d @ wd.T
        # d: its logit's sum of 17 values and rounding, |z| up to 20, the logsumexp's 1e-5; dx: 2^13 truncations of a sum over the classes
        assert ((dx[i:i + 300].double() - rdx).abs() <= (HALF + 2.0 ** -10 + 2e-5) * (d.abs() @ wd.abs().T)).all()
        rdw += xd[i:i + 300].T @ d
        rdb += d.sum(0)
        adw += xd[i:i + 300].abs().T @ d.abs()
        adb += d.abs().sum(0)
    assert ((dw.double() - rdw).abs() <= (HALF + 2e-5) * adw).all() and ((db.double() - rdb).abs() <= ((m + 16) * U + 2e-5) * adb).all()
