"""Layer norm, the gated dense layer, the cross entropy of a dense layer, and their gradients.

Each is compared with its definition in 64 bits.  Bounds are derived, per output value:
 * float32 products (split float16 pairs): a pair holds a value to 2^-23 of itself, the product of two low terms is left out
   (2^-22), and the tensor core truncates once per 16 values of k (2^-23 of the sum so far), so
   |error| <= (2^-20 + (k / 16 + 2) 2^-23) sum |a||b|  =: PRODUCT(k) sum |a||b|.
 * sums of float32: depth x 2^-24 of the sum of magnitudes, depth the longest chain of additions.
 * a rounding: 2^-24 of the value.  exp, erf and the like: 2 ulp = 2^-22 of the value, and of an argument's error its slope.
"""
import ctypes as C
import math

import numpy as np
import pytest

import camel_b200._lib as L
from camel_b200 import tensor as T
from camel_b200._lib import CamelTensorError

gpu = pytest.mark.gpu
U = 2.0 ** -24


def PRODUCT(k):
    return 2.0 ** -20 + (k / 16 + 2) * 2.0 ** -23


def dev(a):
    return T.from_numpy(np.ascontiguousarray(a))


def within(got, want, bound, what):
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, what
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} beyond their bound, worst {np.nanmax(np.abs(got - want) / bound):.3g} of it"


# ---- layer norm -----------------------------------------------------------------------------------


def norm64(x, gamma, beta, eps):
    x = x.astype(np.float64)
    d = x - x.mean(1, keepdims=True)
    r = 1.0 / np.sqrt((d * d).mean(1, keepdims=True) + float(np.float32(eps)))
    h = d * r
    y = h
    if gamma is not None:
        y = y * gamma
    if beta is not None:
        y = y + beta
    return y, h, r


def depth_of(cols):
    """Additions in a row: at most 32 values to a thread (cols / 1024 in rows of more than 32768), five in the warp, five across."""
    return max(32, cols / 1024) + 10


def norm_bounds(x, gamma, beta, eps):
    """h: d is rounded (U |d|); the rest of the mean is off by depth U mean|d|, the variance by (depth + 4) U of itself, r by half that + 4."""
    y, h, r = norm64(x, gamma, beta, eps)
    depth = depth_of(x.shape[1])
    off_h = U * ((depth / 2 + 10) * np.abs(h) + depth + 2)
    off_y = off_h * (1.0 if gamma is None else np.abs(gamma.astype(np.float64))) + 3 * U * (np.abs(y) + (0.0 if beta is None else np.abs(beta)))
    return y, h, r, off_h, off_y


def norm_grad64(x, dy, gamma, eps):
    _, h, r = norm64(x, None, None, eps)
    dy = dy.astype(np.float64)
    g = dy if gamma is None else dy * gamma
    dx = r * (g - g.mean(1, keepdims=True) - h * (g * h).mean(1, keepdims=True))
    return dx, (dy * h).sum(0), dy.sum(0)


def norm_grad_bounds(x, dy, gamma, eps, blocks=148):
    _, h, r, off_h, _ = norm_bounds(x, None, None, eps)
    dy = np.abs(dy.astype(np.float64))
    g = dy if gamma is None else dy * np.abs(gamma)
    depth, a = depth_of(x.shape[1]), np.abs(h)
    mixed = (g * (a + 1)).mean(1, keepdims=True)
    # g, its mean, h times the mean of g h, each with its own error and that of r: (depth + 16) U, and twice that where h and the mean both err
    dx = r * U * ((depth + 16) * (g + g.mean(1, keepdims=True)) + 3 * (depth + 16) * (a + 1) * mixed)
    rows = x.shape[0] / blocks + 16  # a thread's chain; the parts are added in 64 bits
    return dx, (dy * off_h).sum(0) + rows * U * (dy * a).sum(0) + 1e-300, rows * U * dy.sum(0) + 1e-300


NORM_SHAPES = [(1, 1), (3, 1), (1, 2), (5, 3), (1, 1024), (7, 31), (33, 257), (700, 96), (700, 100), (2, 785), (650, 785), (5, 1023), (900, 1024),
               (3, 1025), (64, 2048), (9, 4095), (640, 4096), (2, 4100), (4, 8191), (3, 8192), (2, 8193), (3, 12345), (2, 16384), (2, 20001),
               (2, 32768), (2, 40003)]


def norm_inputs(rows, cols, seed=0, mean=1.0):
    rng = np.random.default_rng(seed + rows * 7919 + cols)
    x = (rng.normal(0, 1, (rows, cols)) * rng.uniform(0.1, 3, (rows, 1)) + mean * rng.normal(0, 1, (rows, 1))).astype(np.float32)
    return x, rng.normal(1, 0.3, cols).astype(np.float32), rng.normal(0, 0.5, cols).astype(np.float32), rng.normal(0, 1, (rows, cols)).astype(np.float32)


@gpu
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_layer_norm(rows, cols):
    x, gamma, beta, dy = norm_inputs(rows, cols)
    for g, b in ((gamma, beta), (None, beta), (gamma, None), (None, None)):
        y, _, _, _, off = norm_bounds(x, g, b, 1e-5)
        got = T.layer_norm(dev(x), None if g is None else dev(g), None if b is None else dev(b)).numpy()
        within(got, y, off, "y")


@gpu
@pytest.mark.parametrize("rows,cols", NORM_SHAPES)
def test_layer_norm_grad(rows, cols):
    x, gamma, _, dy = norm_inputs(rows, cols, 1)
    for g in (gamma, None):
        want, off = norm_grad64(x, dy, g, 1e-5), norm_grad_bounds(x, dy, g, 1e-5)
        got = T.layer_norm_grad(dev(x), dev(dy), None if g is None else dev(g))
        for name, a, b, c in zip(("dx", "dgamma", "dbeta"), got, want, off):
            within(a.numpy(), b, c, name)


@gpu
def test_layer_norm_grad_many_rows():
    """More rows than blocks: each block walks several, and sums them."""
    for rows, cols in ((5000, 40), (9000, 300), (4000, 785), (2000, 2048), (1500, 4096)):
        x, gamma, _, dy = norm_inputs(rows, cols, 2)
        want, off = norm_grad64(x, dy, gamma, 1e-5), norm_grad_bounds(x, dy, gamma, 1e-5)
        for name, a, b, c in zip(("dx", "dgamma", "dbeta"), T.layer_norm_grad(dev(x), dev(dy), dev(gamma)), want, off):
            within(a.numpy(), b, c, name)


@gpu
@pytest.mark.parametrize("cols", [64, 785, 2048, 20001])
def test_layer_norm_of_rows_far_from_zero(cols):
    """A mean of 1e4 beside a spread of 1: the first mean is rounded to 2^-10, the second takes that back."""
    x, gamma, beta, dy = norm_inputs(6, cols, 3)
    x = (x + np.float32(1e4)).astype(np.float32)
    y, _, _, _, off = norm_bounds(x, gamma, beta, 1e-5)
    # d = x - m is exact here or rounded by U |d|, and |d| is larger than |x - mean| by the first mean's error, depth U 1e4
    within(T.layer_norm(dev(x), dev(gamma), dev(beta)).numpy(), y, 2 * off, "y")
    want, goff = norm_grad64(x, dy, gamma, 1e-5), norm_grad_bounds(x, dy, gamma, 1e-5)
    for name, a, b, c in zip(("dx", "dgamma", "dbeta"), T.layer_norm_grad(dev(x), dev(dy), dev(gamma)), want, goff):
        within(a.numpy(), b, 2 * c, name)


@gpu
def test_layer_norm_constant_rows_infinities_and_nan():
    x = np.ones((6, 300), np.float32)
    x[1] = 0.0
    x[2, 7] = np.inf
    x[3, 9] = np.nan
    x[4] = np.arange(300)
    gamma, beta = np.full(300, 2.0, np.float32), np.full(300, 0.5, np.float32)
    y = T.layer_norm(dev(x), dev(gamma), dev(beta)).numpy()
    assert (y[[0, 1, 5]] == 0.5).all() and np.isnan(y[[2, 3]]).all() and np.isfinite(y[4]).all()
    dx, dgamma, dbeta = T.layer_norm_grad(dev(x), dev(np.ones_like(x)), dev(gamma))
    assert np.isnan(dx.numpy()[[2, 3]]).all() and np.isfinite(dx.numpy()[[0, 1, 4, 5]]).all()
    assert np.isnan(dgamma.numpy()).all() and (dbeta.numpy() == 6).all()


@gpu
def test_layer_norm_empty_unaligned_and_in_place():
    assert T.layer_norm(dev(np.zeros((0, 8), np.float32))).shape == (0, 8)
    dx, dgamma, dbeta = T.layer_norm_grad(dev(np.zeros((0, 8), np.float32)), dev(np.zeros((0, 8), np.float32)))
    assert dx.shape == (0, 8) and not dgamma.numpy().any() and not dbeta.numpy().any()
    x, gamma, beta, dy = norm_inputs(40, 1024, 4)
    y, _, _, _, off = norm_bounds(x, gamma, beta, 1e-5)
    # a matrix whose rows are 16-byte multiples on an address that is not
    flat = dev(np.concatenate([[0.0], x.reshape(-1)]).astype(np.float32))
    view = T.wrap_device(flat.ptr + 4, L.F32, x.shape, keep=flat)
    within(T.layer_norm(view, dev(gamma), dev(beta)).numpy(), y, off, "y")
    first = T.layer_norm(dev(x), dev(gamma), dev(beta)).numpy()
    t, g, b = dev(x), dev(gamma), dev(beta)
    L.check(L.lib.ct_layer_norm(t.ptr, g.ptr, b.ptr, 40, 1024, 1e-5, t.ptr))
    assert t.numpy().tobytes() == first.tobytes()
    # only some of the gradients, and dx over dout
    want = [a.numpy().tobytes() for a in T.layer_norm_grad(dev(x), dev(dy), g)]
    tx, td, tb = dev(x), dev(dy), T.zeros([1024])
    L.check(L.lib.ct_layer_norm_grad(tx.ptr, g.ptr, td.ptr, 40, 1024, 1e-5, td.ptr, None, tb.ptr))
    assert [td.numpy().tobytes(), tb.numpy().tobytes()] == [want[0], want[2]]


# ---- gated dense layer ----------------------------------------------------------------------------

GATES = ("sigmoid", "relu", "silu", "gelu")
_erf = np.vectorize(math.erf, otypes=[np.float64])


def gate64(gate, g):
    """Value and slope."""
    if gate == "relu":
        return np.maximum(g, 0.0), (g > 0).astype(np.float64)
    if gate == "gelu":
        cdf = 0.5 * (1.0 + _erf(g / math.sqrt(2.0)))
        return g * cdf, cdf + g * np.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)
    s = 1.0 / (1.0 + np.exp(-g))
    return (s, s * (1 - s)) if gate == "sigmoid" else (g * s, s * (1 + g * (1 - s)))


def gated_inputs(m, k, n, seed=0):
    rng = np.random.default_rng(seed + m * 31 + k * 17 + n)
    s = 1.0 / math.sqrt(max(k, 1))
    f = lambda std, *shape: rng.normal(0, std, shape).astype(np.float32)  # noqa: E731
    return f(1, m, k), f(s, k, n), f(s, k, n), f(0.3, n), f(0.3, n)


def check_gated(x, wg, wu, bg, bu, gate, keep=True):
    t = [None if a is None else dev(a) for a in (x, wg, wu, bg, bu)]
    got = T.dense_gated(*t, gate=gate, keep=keep)
    T.check_async()
    out, *kept = got if keep else (got,)
    d = lambda a: 0.0 if a is None else a.astype(np.float64)  # noqa: E731
    pre = {}
    for name, w, b in (("gate", wg, bg), ("up", wu, bu)):
        z = d(x) @ d(w) + d(b)
        pre[name] = z, PRODUCT(x.shape[1]) * (np.abs(d(x)) @ np.abs(d(w))) + 2 * U * (np.abs(z) + np.abs(d(b)))
    (g, off_g), (u, off_u) = pre["gate"], pre["up"]
    if kept:
        within(kept[0].numpy(), g, off_g + 1e-300, "gate_pre")
        within(kept[1].numpy(), u, off_u + 1e-300, "up_pre")
    a, _ = gate64(gate, g)
    # no slope is above 1.13 (relu jumps by none: it is continuous)
    off_a = 1.13 * off_g + 8 * U * np.abs(a) + 1e-30
    within(out.numpy(), a * u, off_a * np.abs(u) + np.abs(a) * off_u + off_a * off_u + 2 * U * np.abs(a * u) + 1e-30, "out")
    return out


GATED_SHAPES = [(1, 1, 1), (1, 7, 5), (1, 1024, 513), (2, 64, 100), (3, 33, 4096), (5, 300, 301), (8, 256, 640), (9, 785, 64), (16, 128, 1000),
                (17, 100, 33), (33, 65, 129), (64, 512, 512), (100, 1, 40), (127, 31, 127), (128, 64, 128), (129, 200, 130), (300, 771, 250),
                (513, 96, 700), (1537, 130, 515)]


@gpu
@pytest.mark.parametrize("m,k,n", GATED_SHAPES)
def test_dense_gated(m, k, n):
    x, wg, wu, bg, bu = gated_inputs(m, k, n)
    for i, gate in enumerate(GATES):
        check_gated(x, wg, wu, *((bg, bu), (None, bu), (bg, None), (None, None))[(i + m) % 4], gate, keep=(i + n) % 2 == 0)


@gpu
def test_dense_gated_long_k():
    """k beyond what one accumulator sums."""
    for m, k, n in ((40, 5000, 70), (200, 2300, 260), (1, 9000, 20)):
        check_gated(*gated_inputs(m, k, n, 5), "silu")


def gated_grad64(x, wg, wu, g, u, dout, gate):
    x, wg, wu, g, u, dout = (a.astype(np.float64) for a in (x, wg, wu, g, u, dout))
    a, s = gate64(gate, g)
    du, dg = dout * a, dout * u * s
    return (dg @ wg.T + du @ wu.T, x.T @ dg, x.T @ du, dg.sum(0), du.sum(0)), dg, du


def check_gated_grad(x, wg, wu, g, u, dout, gate):
    (dx, dwg, dwu, dbg, dbu), dg, du = gated_grad64(x, wg, wu, g, u, dout, gate)
    got = T.dense_gated_grad(*[dev(a) for a in (x, wg, wu, g, u, dout)], gate=gate, bias=True)
    T.check_async()
    m, k, n = x.shape[0], x.shape[1], wg.shape[1]
    ax, ag, au = np.abs(x.astype(np.float64)), np.abs(wg.astype(np.float64)), np.abs(wu.astype(np.float64))
    # dg and du: a slope is a sum of up to two terms of magnitude 1.2, eight roundings; the row of the planes that holds them holds
    # them to 2^-23, and to 2^-49 of the row's largest
    d64, u64 = np.abs(dout.astype(np.float64)), np.abs(u.astype(np.float64))
    row = np.maximum(np.abs(dg).max(1, keepdims=True, initial=0), np.abs(du).max(1, keepdims=True, initial=0)) * 2.0 ** -36
    off_g, off_u = 8 * U * d64 * u64 * 1.2 + 8 * U * np.abs(dg) + row, 8 * U * np.abs(du) + row
    adg, adu = np.abs(dg), np.abs(du)
    tiny = 1e-30
    bounds = (PRODUCT(2 * n) * (adg @ ag.T + adu @ au.T) + off_g @ ag.T + off_u @ au.T + tiny,
              PRODUCT(m) * (ax.T @ adg) + ax.T @ off_g + tiny, PRODUCT(m) * (ax.T @ adu) + ax.T @ off_u + tiny,
              (m + 16) * U * adg.sum(0) + off_g.sum(0) + tiny, (m + 16) * U * adu.sum(0) + off_u.sum(0) + tiny)
    for name, a, b, c in zip(("dx", "dw_gate", "dw_up", "db_gate", "db_up"), got, (dx, dwg, dwu, dbg, dbu), bounds):
        within(a.numpy(), b, c, name)
    return got


@gpu
@pytest.mark.parametrize("m,k,n", [s for s in GATED_SHAPES if s != (3, 33, 4096)] + [(3, 33, 1030), (2000, 40, 36), (1000, 300, 24)])
def test_dense_gated_grad(m, k, n):
    x, wg, wu, _, _ = gated_inputs(m, k, n, 7)
    rng = np.random.default_rng(m + k + n)
    for gate in GATES if m * n < 50000 else ("silu",):
        g, u, dout = (rng.normal(0, s, (m, n)).astype(np.float32) for s in (1.5, 1.0, 1e-3))
        check_gated_grad(x, wg, wu, g, u, dout, gate)


@gpu
def test_dense_gated_grad_rows_of_all_magnitudes():
    """Rows of the gradient from 1e-25 to 1, one of zeros: each is as exact as it would be alone."""
    m, k, n = 200, 130, 150
    x, wg, wu, _, _ = gated_inputs(m, k, n, 8)
    rng = np.random.default_rng(1)
    g, u, dout = (rng.normal(0, 1, (m, n)).astype(np.float32) for _ in range(3))
    dout *= (10.0 ** rng.uniform(-25, 0, (m, 1))).astype(np.float32)
    dout[17] = 0.0
    check_gated_grad(x, wg, wu, g, u, dout, "silu")


@gpu
def test_dense_gated_extreme_gates():
    """Where exp overflows: sigmoid and its slope are 0 or 1, nothing is NaN."""
    m, n = 40, 60
    g = np.tile(np.array([-3e38, -200, -104, -89, -30, -0.0, 0.0, 30, 89, 104, 200, 3e38], np.float32), (m, 5))
    u, dout = np.full((m, n), 2.0, np.float32), np.full((m, n), 0.5, np.float32)
    x, w = np.eye(m, n, dtype=np.float32), np.eye(n, dtype=np.float32)[:, :n]
    for gate in GATES:
        got = T.dense_gated_grad(dev(x), dev(w), dev(w), dev(g), dev(u), dev(dout), gate=gate, bias=True)
        limit = {"sigmoid": 1, "relu": 0, "silu": 0, "gelu": 0}[gate]
        dwg = got[1].numpy()
        assert np.isfinite(dwg).all(), gate
        s = gate64(gate, np.clip(g.astype(np.float64), -700, 700))[1]
        within(got[3].numpy(), (dout * u * s).sum(0), 1e-5 * (1 + np.abs((dout * u * s).sum(0))), gate)
        assert limit in (0, 1)


@gpu
def test_dense_gated_infinity_and_nan_stay_in_their_rows():
    m, k, n = 70, 90, 110
    x, wg, wu, bg, bu = gated_inputs(m, k, n, 9)
    clean = T.dense_gated(*[dev(a) for a in (x, wg, wu, bg, bu)]).numpy()
    x2 = x.copy()
    x2[3, 5], x2[20, 0], x2[40, 89] = np.nan, np.inf, 3e38
    got = T.dense_gated(*[dev(a) for a in (x2, wg, wu, bg, bu)]).numpy()
    rest = [r for r in range(m) if r not in (3, 20, 40)]
    # a product may take other terms for all rows because of one (ct_precision), so each of the two is within its own bound
    d = lambda a: a.astype(np.float64)  # noqa: E731
    off = PRODUCT(k) * (np.abs(d(x)) @ np.maximum(np.abs(d(wg)), np.abs(d(wu)))) + 4 * U * 10
    g, u = np.abs(d(x) @ d(wg) + d(bg)), np.abs(d(x) @ d(wu) + d(bu))
    within(got[rest], d(clean)[rest], (2 * (1.13 * off * u + g * off + off * off) + 1e-5 * U)[rest] + 20 * U * np.abs(d(clean)[rest]), "other rows")
    assert np.isnan(got[3]).all() and not np.isfinite(got[20]).any()


# ---- cross entropy of a dense layer ---------------------------------------------------------------


def ce_inputs(m, k, n, seed=0, scale=2.0):
    rng = np.random.default_rng(seed + m * 31 + k * 17 + n)
    x = rng.normal(0, 1, (m, k)).astype(np.float32)
    w = rng.normal(0, scale / math.sqrt(max(k, 1)), (k, n)).astype(np.float32)
    b = rng.normal(0, 0.5, n).astype(np.float32)
    t = rng.integers(0, n, m)
    t[rng.uniform(size=m) < 0.15] = -1
    if m > 2:
        t[1], t[2] = 0, n - 1
    return x, w, b, t


def ce64(x, w, b, t):
    z = x.astype(np.float64) @ w.astype(np.float64) + (0.0 if b is None else b.astype(np.float64))
    top = z.max(1, keepdims=True)
    lse = (top + np.log(np.exp(z - top).sum(1, keepdims=True)))[:, 0]
    has = (t >= 0) & (t < w.shape[1])
    at = np.where(has, t, 0)
    off_z = PRODUCT(x.shape[1]) * (np.abs(x.astype(np.float64)) @ np.abs(w.astype(np.float64))) + 2 * U * (np.abs(z) + (0.0 if b is None else np.abs(b)))
    return z, lse, np.where(has, lse - z[np.arange(len(t)), at], 0.0), has, at, off_z


def ce_off_lse(z, lse, off_z):
    """The logits' own errors, a sum of up to 256 terms in a row before the tree, exp of differences (their rounding), the logarithm."""
    return off_z.max(1) + U * (300 + 8 * np.abs(z - lse[:, None]).max(1) + 8 + 2 * np.abs(lse)) + 2 * U * np.abs(z).max(1)


def check_ce(x, w, b, t):
    z, lse, loss, has, at, off_z = ce64(x, w, b, t)
    got = T.dense_cross_entropy(dev(x), dev(w), dev(t), None if b is None else dev(b))
    T.check_async()
    off = ce_off_lse(z, lse, off_z)
    within(got[1].numpy(), lse, off, "lse")
    within(got[0].numpy(), loss, off + off_z[np.arange(len(t)), at] + 2 * U * (np.abs(lse) + np.abs(loss)), "loss")
    assert not got[0].numpy()[~has].any()
    return got


CE_SHAPES = [(1, 1, 1), (1, 5, 2), (1, 64, 1000), (4, 100, 10), (300, 785, 10), (7, 33, 33), (64, 256, 3001), (3, 20, 40003), (127, 31, 127),
             (128, 64, 256), (129, 65, 257), (500, 40, 1030), (1000, 128, 36), (260, 513, 2100)]


@gpu
@pytest.mark.parametrize("m,k,n", CE_SHAPES)
def test_dense_cross_entropy(m, k, n):
    x, w, b, t = ce_inputs(m, k, n)
    check_ce(x, w, b, t)
    check_ce(x, w, None, t)


def check_ce_grad(x, w, b, t, dloss):
    z, lse, _, has, at, off_z = ce64(x, w, b, t)
    m, k, n = x.shape[0], x.shape[1], w.shape[1]
    lse32 = lse.astype(np.float32)
    got = T.dense_cross_entropy_grad(dev(x), dev(w), dev(t), dev(lse32), None if b is None else dev(b), None if dloss is None else dev(dloss))
    T.check_async()
    weight = np.where(has, 1.0 if dloss is None else dloss.astype(np.float64), 0.0)[:, None]
    p = np.exp(z - lse32.astype(np.float64)[:, None])
    d = p.copy()
    d[np.arange(m), at] -= 1.0
    d *= weight
    # p: the logit's error and the rounding of z - lse, of exp's argument and of exp; d is held to 2^-22, and to 2^-36 of 1
    off_p = p * (off_z + U * (2 * np.abs(z - lse[:, None]) + 8) + 2 * U * np.abs(z)) + 2.0 ** -36
    off_d = np.abs(weight) * (off_p + 4 * U * np.abs(p)) + 4 * U * np.abs(d)
    off_d[np.arange(m), at] += 2 * U * np.abs(weight[:, 0])
    ax, aw, ad = np.abs(x.astype(np.float64)), np.abs(w.astype(np.float64)), np.abs(d)
    want = [d @ w.astype(np.float64).T, x.astype(np.float64).T @ d, d.sum(0)]
    bounds = [PRODUCT(n) * (ad @ aw.T) + off_d @ aw.T + 1e-30, PRODUCT(m) * (ax.T @ ad) + ax.T @ off_d + 1e-30, (m + 16) * U * ad.sum(0) + off_d.sum(0) + 1e-30]
    assert len(got) == (3 if b is not None else 2)
    for name, a, c, e in zip(("dx", "dw", "db"), got, want, bounds):
        within(a.numpy(), c, e, name)
    return got


@gpu
@pytest.mark.parametrize("m,k,n", CE_SHAPES)
def test_dense_cross_entropy_grad(m, k, n):
    x, w, b, t = ce_inputs(m, k, n, 3)
    dloss = np.random.default_rng(m).uniform(-1, 1, m).astype(np.float32) / m
    check_ce_grad(x, w, b, t, dloss)
    check_ce_grad(x, w, None, t, None)


@gpu
def test_dense_cross_entropy_targets():
    """No row with a target; targets far outside; the same class in every row; a class that is certain."""
    x, w, b, t = ce_inputs(140, 48, 300, 5)
    for t in (np.full(140, -1), np.where(np.arange(140) % 2, 300, -(2 ** 62)), np.full(140, 299), np.full(140, 2 ** 40)):
        check_ce(x, w, b, t)
        got = check_ce_grad(x, w, b, t, np.ones(140, np.float32))
        if not ((t >= 0) & (t < 300)).any():
            assert not any(a.numpy().any() for a in got)
    b2 = b.copy()
    b2[7] = 60.0  # exp(-60) of everything else
    t = np.full(140, 7)
    check_ce(x, w, b2, t)
    check_ce_grad(x, w, b2, t, None)


@gpu
def test_dense_cross_entropy_masked_classes():
    """Classes that a bias of -inf or of the type's lowest value takes out, for n that is and is not whole tiles."""
    for n in (256, 700):
        x, w, b, t = ce_inputs(60, 32, n, 6)
        t[:] = np.random.default_rng(0).integers(0, 20, 60)
        for low in (-np.inf, np.finfo(np.float32).min):
            b2 = b.copy()
            b2[20:] = low
            z, lse, loss, *_ = ce64(x, w[:, :20], b[:20], t)
            got = T.dense_cross_entropy(dev(x), dev(w), dev(t), dev(b2))
            assert np.allclose(got[1].numpy(), lse, rtol=0, atol=2e-5) and np.allclose(got[0].numpy(), loss, rtol=0, atol=4e-5)
            dx, dw, db = T.dense_cross_entropy_grad(dev(x), dev(w), dev(t), got[1], dev(b2))
            assert np.isfinite(dx.numpy()).all() and not dw.numpy()[:, 20:].any() and not db.numpy()[20:].any()


@gpu
def test_dense_cross_entropy_nan_and_infinity_stay_in_their_rows():
    x, w, b, t = ce_inputs(150, 64, 500, 7)
    t = np.abs(t) % 500
    clean = [a.numpy() for a in T.dense_cross_entropy(dev(x), dev(w), dev(t), dev(b))]
    x2 = x.copy()
    x2[5, 3], x2[77, 0] = np.nan, np.inf
    got = [a.numpy() for a in T.dense_cross_entropy(dev(x2), dev(w), dev(t), dev(b))]
    rest = [r for r in range(150) if r not in (5, 77)]
    z, l64, _, _, _, off_z = ce64(x, w, b, t)
    for a, c in zip(got, clean):  # as above: within twice the bound of one
        within(a[rest], c.astype(np.float64)[rest], (4 * ce_off_lse(z, l64, off_z))[rest], "other rows")
        assert np.isnan(a[5])
    assert not np.isfinite(got[1][77])


# ---- together -------------------------------------------------------------------------------------


def block64(p, x, t):
    import torch

    xh = torch.nn.functional.layer_norm(x, (x.shape[1],), p["gamma"], p["beta"], float(np.float32(1e-5)))
    h = torch.nn.functional.silu(xh @ p["wg"] + p["bg"]) * (xh @ p["wu"] + p["bu"])
    return torch.nn.functional.cross_entropy((h @ p["wd"]) @ p["wv"] + p["bv"], t, ignore_index=-1, reduction="sum")


@gpu
def test_a_training_step():
    """layer norm -> gated layer -> dense -> cross entropy over a vocabulary, and back, against differentiation in 64 bits."""
    import torch

    rng = np.random.default_rng(11)
    m, k, n, v = 90, 96, 200, 1500
    f = lambda std, *s: rng.normal(0, std, s).astype(np.float32)  # noqa: E731
    p = dict(gamma=1 + f(0.1, k), beta=f(0.1, k), wg=f(0.1, k, n), bg=f(0.1, n), wu=f(0.1, k, n), bu=f(0.1, n), wd=f(0.07, n, k), wv=f(0.2, k, v), bv=f(0.2, v))
    x, t = f(1.0, m, k), rng.integers(-1, v, m)
    q = {key: torch.tensor(a, dtype=torch.float64, requires_grad=True) for key, a in p.items()}
    xt = torch.tensor(x, dtype=torch.float64, requires_grad=True)
    want = block64(q, xt, torch.tensor(t))
    want.backward()

    d = {key: dev(a) for key, a in p.items()}

    def step(dx_in, targets):
        y = T.layer_norm(dx_in, d["gamma"], d["beta"])
        h, g, u = T.dense_gated(y, d["wg"], d["wu"], d["bg"], d["bu"], keep=True)
        z = T.dense(h, d["wd"])
        loss, lse = T.dense_cross_entropy(z, d["wv"], targets, d["bv"])
        dz, dwv, dbv = T.dense_cross_entropy_grad(z, d["wv"], targets, lse, d["bv"])
        dh, dwd = T.matmul(dz, T.transpose(d["wd"])), T.matmul_tn(h, dz)
        dy, dwg, dwu, dbg, dbu = T.dense_gated_grad(y, d["wg"], d["wu"], g, u, dh, bias=True)
        dx, dgamma, dbeta = T.layer_norm_grad(dx_in, dy, d["gamma"])
        return dict(loss=loss, x=dx, gamma=dgamma, beta=dbeta, wg=dwg, wu=dwu, bg=dbg, bu=dbu, wd=dwd, wv=dwv, bv=dbv)

    tx, tt = dev(x), dev(t)
    got = step(tx, tt)
    T.check_async()
    assert abs(float(got["loss"].numpy().astype(np.float64).sum()) - want.item()) <= 1e-5 * abs(want.item())
    for key, a in got.items():
        if key == "loss":
            continue
        w = (xt if key == "x" else q[key]).grad.numpy()
        # six steps, each of a few float32 products of up to 1500 values: 1e-5 of the largest together
        assert np.abs(a.numpy() - w).max() <= 2e-5 * np.abs(w).max(), key

    # recorded and replayed it gives the same bytes
    first = {key: a.numpy().tobytes() for key, a in got.items()}
    with T.Graph() as graph:
        graph.keep = step(tx, tt)
    for _ in range(2):
        graph.launch()
        T.check_async()
        assert {key: a.numpy().tobytes() for key, a in graph.keep.items()} == first


@gpu
def test_repeated_calls_and_other_streams_give_the_same_bytes():
    import torch

    x, wg, wu, bg, bu = gated_inputs(300, 200, 260, 12)
    cx, cw, cb, ct = ce_inputs(300, 200, 900, 12)
    g, u, dout = (np.random.default_rng(i).normal(0, 1, (300, 260)).astype(np.float32) for i in range(3))
    nx, gamma, beta, dy = norm_inputs(300, 260, 12)
    d = [dev(a) for a in (x, wg, wu, bg, bu, cx, cw, cb, ct, g, u, dout, nx, gamma, beta, dy)]

    def all_of():
        out = [T.layer_norm(d[12], d[13], d[14]), *T.layer_norm_grad(d[12], d[15], d[13]), T.dense_gated(*d[:5])]
        out += T.dense_gated_grad(*d[:3], *d[9:12], bias=True)
        loss, lse = T.dense_cross_entropy(d[5], d[6], d[8], d[7])
        return out + [loss, lse, *T.dense_cross_entropy_grad(d[5], d[6], d[8], lse, d[7])]

    want = [a.numpy().tobytes() for a in all_of()]
    assert [a.numpy().tobytes() for a in all_of()] == want
    T.sync()
    stream = torch.cuda.Stream()
    L.check(L.lib.ct_set_stream(stream.cuda_stream))
    try:
        got = all_of()
        assert [a.numpy().tobytes() for a in got] == want
        del got
        T.sync()
    finally:
        L.check(L.lib.ct_set_stream(None))


@gpu
def test_bf16_precision():
    """Under the reduced precision the products round their operands to bfloat16: 2^-8 each, of sum |a||b|."""
    x, wg, wu, bg, bu = gated_inputs(200, 256, 192, 13)
    cx, cw, cb, ct = ce_inputs(200, 256, 500, 13)
    L.check(L.lib.ct_set_precision(L.PREC_BF16))
    try:
        out = T.dense_gated(*[dev(a) for a in (x, wg, wu, bg, bu)]).numpy()
        loss, lse = T.dense_cross_entropy(dev(cx), dev(cw), dev(ct), dev(cb))
        dx, dw, db = T.dense_cross_entropy_grad(dev(cx), dev(cw), dev(ct), lse, dev(cb))
        T.check_async()
    finally:
        L.check(L.lib.ct_set_precision(L.PREC_3XTF32))
    d = lambda a: a.astype(np.float64)  # noqa: E731
    gp, up = d(x) @ d(wg) + d(bg), d(x) @ d(wu) + d(bu)
    off = 2.0 ** -7 * (np.abs(d(x)) @ np.maximum(np.abs(d(wg)), np.abs(d(wu)))) + 1e-5
    a = gate64("silu", gp)[0]
    within(out, a * up, 1.13 * off * (np.abs(up) + off) + np.abs(a) * off, "out")
    z, want, *_ = ce64(cx, cw, cb, ct)
    within(lse.numpy(), want, (2.0 ** -7 * (np.abs(d(cx)) @ np.abs(d(cw)))).max(1) + 1e-4, "lse")
    assert np.isfinite(dx.numpy()).all() and np.isfinite(dw.numpy()).all()


# ---- refusals -------------------------------------------------------------------------------------


@gpu
def test_refusals():
    f = lambda *s: dev(np.ones(s, np.float32))  # noqa: E731
    i = lambda *s: dev(np.zeros(s, np.int64))  # noqa: E731
    refused = [
        lambda: T.layer_norm(f(4)), lambda: T.layer_norm(i(4, 4)), lambda: T.layer_norm(f(4, 4), f(3)), lambda: T.layer_norm(f(4, 4), None, i(4)),
        lambda: T.layer_norm(f(4, 4), eps=-1.0), lambda: T.layer_norm(f(4, 4), eps=float("nan")),
        lambda: T.layer_norm_grad(f(4, 4), f(4, 5)), lambda: T.layer_norm_grad(f(4, 4), f(4, 4), f(5)),
        lambda: T.dense_gated(f(4, 4), f(5, 4), f(5, 4)), lambda: T.dense_gated(f(4, 4), f(4, 4), f(4, 5)),
        lambda: T.dense_gated(f(4, 4), f(4, 4), f(4, 4), f(5)), lambda: T.dense_gated(f(4, 4), f(4, 4), f(4, 4), gate="tanh"),
        lambda: T.dense_gated(i(4, 4), f(4, 4), f(4, 4)),
        lambda: T.dense_gated_grad(f(4, 3), f(3, 5), f(3, 5), f(4, 5), f(4, 5), f(4, 4)),
        lambda: T.dense_cross_entropy(f(4, 3), f(3, 5), f(4)), lambda: T.dense_cross_entropy(f(4, 3), f(3, 5), i(5)),
        lambda: T.dense_cross_entropy(f(4, 3), f(4, 5), i(4)), lambda: T.dense_cross_entropy(f(4, 3), f(3, 5), i(4), f(4)),
        lambda: T.dense_cross_entropy(f(4, 3), f(3, 0), i(4)),
        lambda: T.dense_cross_entropy_grad(f(4, 3), f(3, 5), i(4), f(3)), lambda: T.dense_cross_entropy_grad(f(4, 3), f(3, 5), i(4), f(4), None, f(5)),
    ]
    for n, call in enumerate(refused):
        with pytest.raises(CamelTensorError) as e:
            call()
        assert e.value.status == L.ERR_INVALID, n
    a, p = f(4, 4), f(4, 4)
    for rc in (L.lib.ct_layer_norm(None, None, None, 4, 4, 1e-5, a.ptr), L.lib.ct_layer_norm(a.ptr, None, None, -1, 4, 1e-5, a.ptr),
               L.lib.ct_layer_norm_grad(a.ptr, None, None, 4, 4, 1e-5, p.ptr, None, None),
               L.lib.ct_dense_gated(a.ptr, a.ptr, None, a.ptr, None, 4, 4, 4, 9, p.ptr, None, None),
               L.lib.ct_dense_gated(a.ptr, a.ptr, None, a.ptr, None, 4, 4, 4, 0, None, None, None),
               L.lib.ct_dense_gated(a.ptr, None, None, a.ptr, None, 4, 4, 4, 0, p.ptr, None, None),
               L.lib.ct_dense_gated_grad(a.ptr, a.ptr, a.ptr, a.ptr, None, a.ptr, 4, 4, 4, 0, p.ptr, None, None, None, None),
               L.lib.ct_dense_gated_grad(None, a.ptr, a.ptr, a.ptr, a.ptr, a.ptr, 4, 4, 4, 0, None, p.ptr, None, None, None),
               L.lib.ct_dense_cross_entropy(a.ptr, a.ptr, None, None, 4, 4, 4, p.ptr, None),
               L.lib.ct_dense_cross_entropy_grad(a.ptr, a.ptr, None, a.ptr, None, None, 4, 4, 4, p.ptr, None, None)):
        assert rc == L.ERR_INVALID, L.lib.ct_last_error()


@gpu
def test_empty_batches():
    f = lambda *s: dev(np.ones(s, np.float32))  # noqa: E731
    i = lambda *s: dev(np.zeros(s, np.int64))  # noqa: E731
    assert T.dense_gated(f(0, 4), f(4, 6), f(4, 6)).shape == (0, 6)
    got = T.dense_gated_grad(f(0, 4), f(4, 6), f(4, 6), f(0, 6), f(0, 6), f(0, 6), bias=True)
    assert [a.shape for a in got] == [(0, 4), (4, 6), (4, 6), (6,), (6,)] and not any(a.numpy().any() for a in got)
    loss, lse = T.dense_cross_entropy(f(0, 4), f(4, 6), i(0))
    assert loss.shape == lse.shape == (0,)
    dx, dw, db = T.dense_cross_entropy_grad(f(0, 4), f(4, 6), i(0), f(0), f(6))
    assert dx.shape == (0, 4) and not dw.numpy().any() and not db.numpy().any()
    # no inner dimension: the biases alone
    bg, bu = np.array([1.0, -2.0, 0.5], np.float32), np.array([3.0, 4.0, 5.0], np.float32)
    out = T.dense_gated(f(5, 0), f(0, 3), f(0, 3), dev(bg), dev(bu), gate="relu").numpy()
    assert (out == np.array([3.0, 0.0, 2.5], np.float32)).all()
    loss, lse = T.dense_cross_entropy(f(5, 0), f(0, 3), i(5), dev(bg))
    assert np.allclose(lse.numpy(), np.log(np.exp(bg.astype(np.float64)).sum()), atol=1e-6)


def test_without_a_device_the_new_entry_points_refuse():
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    z = C.c_void_p(0)
    for rc in (L.lib.ct_layer_norm(z, z, z, 1, 1, 1e-5, z), L.lib.ct_layer_norm_grad(z, z, z, 1, 1, 1e-5, z, z, z),
               L.lib.ct_dense_gated(z, z, z, z, z, 1, 1, 1, 0, z, z, z), L.lib.ct_dense_gated_grad(z, z, z, z, z, z, 1, 1, 1, 0, z, z, z, z, z),
               L.lib.ct_dense_cross_entropy(z, z, z, z, 1, 1, 1, z, z), L.lib.ct_dense_cross_entropy_grad(z, z, z, z, z, z, 1, 1, 1, z, z, z)):
        assert rc == L.ERR_NO_DEVICE
