"""Layer norm, the gated dense layer and the cross entropy of a dense layer: calls that programs make less often - buffers at any
address, memory that holds anything, a vocabulary in pieces, rows without a target, two recordings at once.  Values are compared with
those of the plain call (bytes, where the same kernels run) or with the definition in 64 bits, under the bounds of test_layers.
"""
import math

import numpy as np
import pytest

import camel_b200._lib as L
from camel_b200 import tensor as T
from test_layers import (PRODUCT, U, ce64, ce_inputs, ce_off_lse, check_ce, check_ce_grad, check_gated, check_gated_grad, dev, gated_inputs, norm_bounds,
                         norm_grad64, norm_grad_bounds, norm_inputs, within)

gpu = pytest.mark.gpu


class Buffer:
    """A float (or int) array on the device `shift` values past an aligned address, with sentinels before and behind."""

    def __init__(self, shape, values=None, shift=1, dtype=np.float32):
        self.shape, self.shift, self.dtype = shape, shift, dtype
        self.count = int(np.prod(shape))
        self.sentinel = np.array([-77], dtype)[0]
        flat = np.full(self.count + shift + 64, self.sentinel, dtype)
        if values is not None:
            flat[shift:shift + self.count] = values.reshape(-1)
        self.whole = dev(flat)
        self.ptr = self.whole.ptr + shift * flat.itemsize

    def numpy(self):
        flat = self.whole.numpy()
        assert (flat[:self.shift] == self.sentinel).all() and (flat[self.shift + self.count:] == self.sentinel).all(), "written outside"
        return flat[self.shift:self.shift + self.count].reshape(self.shape)


def ptr(b):
    return None if b is None else b.ptr


@gpu
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
@pytest.mark.parametrize("rows,cols", [(5, 7), (600, 48), (70, 785), (1200, 800), (9, 2050), (4, 4096), (3, 5001)])
def test_layer_norm_at_any_address(rows, cols, shift):
    x, gamma, beta, dy = norm_inputs(rows, cols, 21)
    bx, bd = Buffer(x.shape, x, shift), Buffer(x.shape, dy, (shift * 3) % 4)
    bg, bb = Buffer((cols,), gamma, shift), Buffer((cols,), beta, (shift + 1) % 4)
    out, dx, dg, db = Buffer(x.shape, None, (shift + 2) % 4), Buffer(x.shape, None, shift), Buffer((cols,), None, 1), Buffer((cols,), None, shift)
    L.check(L.lib.ct_layer_norm(bx.ptr, bg.ptr, bb.ptr, rows, cols, 1e-5, out.ptr))
    y, _, _, _, off = norm_bounds(x, gamma, beta, 1e-5)
    within(out.numpy(), y, off, "y")
    L.check(L.lib.ct_layer_norm_grad(bx.ptr, bg.ptr, bd.ptr, rows, cols, 1e-5, dx.ptr, dg.ptr, db.ptr))
    for name, a, b, c in zip(("dx", "dgamma", "dbeta"), (dx, dg, db), norm_grad64(x, dy, gamma, 1e-5), norm_grad_bounds(x, dy, gamma, 1e-5)):
        within(a.numpy(), b, c, name)
    bx.numpy(), bd.numpy()


@gpu
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
@pytest.mark.parametrize("m,k,n", [(1, 70, 36), (5, 33, 130), (20, 200, 72), (50, 65, 300), (100, 130, 65), (150, 96, 264), (300, 75, 130)])
def test_dense_gated_at_any_address(m, k, n, shift):
    x, wg, wu, bg, bu = gated_inputs(m, k, n, 22)
    t = [Buffer(a.shape, a, (shift + i) % 4) for i, a in enumerate((x, wg, wu, bg, bu))]
    out, g, u = Buffer((m, n), None, shift), Buffer((m, n), None, (shift + 1) % 4), Buffer((m, n), None, 0)
    L.check(L.lib.ct_dense_gated(t[0].ptr, t[1].ptr, t[3].ptr, t[2].ptr, t[4].ptr, m, k, n, L.GATE_SILU, out.ptr, g.ptr, u.ptr))
    T.check_async()
    want = T.dense_gated(*[dev(a) for a in (x, wg, wu, bg, bu)], keep=True)
    for a, b in zip((out, g, u), want):  # the same products of the same terms, wherever they lie
        assert a.numpy().tobytes() == b.numpy().tobytes()
    rng = np.random.default_rng(m)
    dout = rng.normal(0, 1, (m, n)).astype(np.float32)
    d, dx = Buffer((m, n), dout, (shift + 3) % 4), Buffer((m, k), None, shift)
    dwg, dwu, dbg, dbu = Buffer((k, n), None, shift), Buffer((k, n), None, (shift + 2) % 4), Buffer((n,), None, 1), Buffer((n,), None, 3)
    L.check(L.lib.ct_dense_gated_grad(t[0].ptr, t[1].ptr, t[2].ptr, g.ptr, u.ptr, d.ptr, m, k, n, L.GATE_SILU, dx.ptr, dwg.ptr, dwu.ptr, dbg.ptr, dbu.ptr))
    T.check_async()
    want = T.dense_gated_grad(dev(x), dev(wg), dev(wu), want[1], want[2], dev(dout), bias=True)
    for a, b in zip((dx, dwg, dwu, dbg, dbu), want):
        assert a.numpy().tobytes() == b.numpy().tobytes()
    # one gradient alone
    for alone in range(5):
        outs = [Buffer(s, None, 0) if i == alone else None for i, s in enumerate(((m, k), (k, n), (k, n), (n,), (n,)))]
        L.check(L.lib.ct_dense_gated_grad(t[0].ptr, t[1].ptr, t[2].ptr, g.ptr, u.ptr, d.ptr, m, k, n, L.GATE_SILU, *[ptr(o) for o in outs]))
        got = outs[alone].numpy().astype(np.float64)
        ref = want[alone].numpy().astype(np.float64)
        assert np.abs(got - ref).max() <= 1e-5 * np.abs(ref).max()
    for b in t:
        b.numpy()


@gpu
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
@pytest.mark.parametrize("m,k,n", [(1, 40, 100), (9, 64, 36), (30, 130, 264), (100, 65, 300), (200, 96, 520), (300, 75, 131), (40, 90, 10), (70, 64, 24)])
def test_dense_cross_entropy_at_any_address(m, k, n, shift):
    x, w, b, t = ce_inputs(m, k, n, 23)
    bx, bw, bb, bt = Buffer(x.shape, x, shift), Buffer(w.shape, w, (shift + 1) % 4), Buffer(b.shape, b, (shift + 2) % 4), Buffer(t.shape, t, 1, np.int64)
    loss, lse = Buffer((m,), None, shift), Buffer((m,), None, 3)
    L.check(L.lib.ct_dense_cross_entropy(bx.ptr, bw.ptr, bb.ptr, bt.ptr, m, k, n, loss.ptr, lse.ptr))
    T.check_async()
    z, l64, loss64, has, at, off_z = ce64(x, w, b, t)
    off = ce_off_lse(z, l64, off_z)
    within(lse.numpy(), l64, off, "lse")
    within(loss.numpy(), loss64, off + off_z[np.arange(m), at] + 2 * U * (np.abs(l64) + np.abs(loss64)), "loss")
    dloss = np.random.default_rng(m).uniform(0.5, 1, m).astype(np.float32)
    bl, dx, dw, db = Buffer((m,), dloss, 2), Buffer((m, k), None, shift), Buffer((k, n), None, (shift + 1) % 4), Buffer((n,), None, 1)
    l32 = Buffer((m,), l64.astype(np.float32), 1)
    L.check(L.lib.ct_dense_cross_entropy_grad(bx.ptr, bw.ptr, bb.ptr, bt.ptr, l32.ptr, bl.ptr, m, k, n, dx.ptr, dw.ptr, db.ptr))
    T.check_async()
    want = check_ce_grad(x, w, b, t, dloss)
    for a, c in zip((dx, dw, db), want):
        r = c.numpy().astype(np.float64)
        assert np.abs(a.numpy() - r).max() <= 1e-5 * np.abs(r).max() + 1e-30
    for alone in range(3):
        outs = [Buffer(s, None, 0) if i == alone else None for i, s in enumerate(((m, k), (k, n), (n,)))]
        L.check(L.lib.ct_dense_cross_entropy_grad(bx.ptr, bw.ptr, bb.ptr, bt.ptr, l32.ptr, bl.ptr, m, k, n, *[ptr(o) for o in outs]))
        r = want[alone].numpy().astype(np.float64)
        assert np.abs(outs[alone].numpy() - r).max() <= 1e-5 * np.abs(r).max() + 1e-30
    for q in (bx, bw, bb, bt, bl):
        q.numpy()


@gpu
@pytest.mark.parametrize("m,k,n", [(2100, 40, 36), (5000, 70, 90), (2500, 200, 33)])
def test_dense_gated_grad_of_many_rows(m, k, n):
    x, wg, wu, _, _ = gated_inputs(m, k, n, 24)
    g, u, dout = (np.random.default_rng(i).normal(0, 1, (m, n)).astype(np.float32) for i in range(3))
    check_gated_grad(x, wg, wu, g, u, dout, "gelu")


@gpu
@pytest.mark.parametrize("m", [1, 2, 3, 5, 8, 9, 16])
@pytest.mark.parametrize("k,n", [(1, 7), (97, 1300), (300, 3100), (41, 1024)])
def test_few_rows(m, k, n):
    """Blocks of 1024 columns and parts of the weights' rows; and 9 to 16 rows of wide layers, whose logits are streamed."""
    x, wg, wu, bg, bu = gated_inputs(m, k, n, 29)
    check_gated(x, wg, wu, bg, bu, "gelu")
    g, u, dout = (np.random.default_rng(i).normal(0, 1, (m, n)).astype(np.float32) for i in range(3))
    check_gated_grad(x, wg, wu, g, u, dout, "gelu")
    for classes in (n + 20, 2 * n + 100):
        x, w, b, t = ce_inputs(m, k, classes, 29)
        check_ce(x, w, b, t)
        check_ce_grad(x, w, b, t, np.random.default_rng(3).uniform(0.5, 1, m).astype(np.float32))


@gpu
@pytest.mark.parametrize("gate", ["sigmoid", "silu", "gelu"])
def test_gates_keep_their_small_values(gate):
    """Relative to the value, also where it is 1e-30: 2^-22 of the approximate exponential and ten roundings more, 14 in all."""
    g = np.concatenate([np.linspace(-12, 12, 4001), -np.geomspace(1e-6, 12, 4000)]).astype(np.float32)
    one = np.ones((1, 16), np.float32)
    out, pre, _ = T.dense_gated(dev(g[:, None]), dev(one), dev(0 * one), None, dev(np.ones(16, np.float32)), gate=gate, keep=True)
    assert (np.abs(pre.numpy() - g[:, None]) <= 2.0 ** -22 * np.abs(g[:, None])).all()
    x = pre.numpy()[:, 0].astype(np.float64)  # what the gate was given
    if gate == "gelu":
        want = x * 0.5 * np.array([math.erfc(-v / math.sqrt(2)) for v in x])
    else:
        s = np.where(x >= 0, 1 / (1 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))))
        want = s if gate == "sigmoid" else x * s
    within(out.numpy(), np.repeat(want[:, None], 16, 1), np.repeat(14 * U * np.abs(want)[:, None], 16, 1), gate)


@gpu
def test_dense_gated_wide_rows():
    """Rows of d that no block holds (n beyond 8192)."""
    m, k, n = 12, 24, 8300
    x, wg, wu, bg, bu = gated_inputs(m, k, n, 25)
    check_gated(x, wg, wu, bg, bu, "sigmoid")
    g, u, dout = (np.random.default_rng(i).normal(0, 1, (m, n)).astype(np.float32) for i in range(3))
    check_gated_grad(x, wg, wu, g, u, dout, "silu")


def big_ce(m, k, n):
    """Against 64 bits on the device, by the largest value: sums of up to n (or m) products."""
    import torch

    gen = torch.Generator(device="cuda").manual_seed(m + n)
    x = torch.randn(m, k, device="cuda", generator=gen)
    w = torch.randn(k, n, device="cuda", generator=gen) / math.sqrt(k)
    b = torch.randn(n, device="cuda", generator=gen) * 0.3
    t = torch.randint(n, (m,), device="cuda", generator=gen)
    t[::7] = -1
    loss, lse = torch.empty(m, device="cuda"), torch.empty(m, device="cuda")
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    dl = torch.rand(m, device="cuda", generator=gen) + 0.5
    torch.cuda.synchronize()
    p = lambda a: a.data_ptr()  # noqa: E731
    L.check(L.lib.ct_dense_cross_entropy(p(x), p(w), p(b), p(t), m, k, n, p(loss), p(lse)))
    L.check(L.lib.ct_dense_cross_entropy_grad(p(x), p(w), p(b), p(t), p(lse), p(dl), m, k, n, p(dx), p(dw), p(db)))
    T.check_async()
    wd, bd = w.double(), b.double()
    rdx, rdw, rdb = torch.empty(m, k, device="cuda", dtype=torch.float64), torch.zeros_like(wd), torch.zeros_like(bd)
    for i in range(0, m, 256):
        z = x[i:i + 256].double() @ wd + bd
        l64 = torch.logsumexp(z, 1)
        assert (lse[i:i + 256].double() - l64).abs().max() <= 1e-5
        d = (z - lse[i:i + 256].double()[:, None]).exp()
        has = t[i:i + 256] >= 0
        rows = torch.nonzero(has)[:, 0]
        at = t[i:i + 256][rows]
        assert (loss[i:i + 256][rows].double() - (l64[rows] - z[rows, at])).abs().max() <= 2e-5 and not loss[i:i + 256][~has].any()
        d[rows, at] -= 1.0
        d *= torch.where(has, dl[i:i + 256].double(), 0.0)[:, None]
        rdx[i:i + 256] = d @ wd.T
        rdw += x[i:i + 256].double().T @ d
        rdb += d.sum(0)
    for name, a, r in (("dx", dx, rdx), ("dw", dw, rdw), ("db", db, rdb)):
        err = ((a.double() - r).norm() / r.norm()).item()
        assert err <= 5e-6, (name, err)
        assert ((a.double() - r).abs().max() / r.abs().max()).item() <= 2e-5, name


@gpu
@pytest.mark.parametrize("m,k,n", [(4100, 40, 33001), (128, 17, 1048600), (2000, 64, 70000), (150, 40, 12001), (150, 41, 20004)])
def test_cross_entropy_vocabulary_in_pieces(m, k, n):
    big_ce(m, k, n)


@gpu
@pytest.mark.parametrize("m,k,n", [(30, 1024, 16), (9600, 1024, 4), (9500, 700, 3), (9500, 1000, 8), (40, 1024, 8), (200, 33, 15), (2500, 511, 12), (300, 1, 2)])
def test_few_classes(m, k, n):
    """Blocks of eight and of sixteen warps, two and three tiles on their way."""
    x, w, b, t = ce_inputs(m, k, n, 34)
    check_ce(x, w, b, t)
    check_ce_grad(x, w, b, t, np.random.default_rng(4).uniform(0.5, 1, m).astype(np.float32))


@gpu
@pytest.mark.parametrize("n", [8193, 12288, 20001])
def test_long_rows_of_logits(n):
    """Masked stretches as long as a part, a row that is masked but for its target, a NaN, rows without a target."""
    x, w, b, t = ce_inputs(6, 24, n, 35)
    t[:] = [0, n - 1, 4095, 4096, -1, n]
    b[4097:8192] = -np.inf
    check_ce(x, w, b, t)
    only = np.full(n, -np.inf, np.float32)
    only[4096] = 0.5
    loss, lse = T.dense_cross_entropy(dev(x), dev(w), dev(np.full(6, 4096)), dev(only))
    z = x.astype(np.float64) @ w[:, 4096].astype(np.float64) + 0.5
    assert np.abs(lse.numpy() - z).max() <= 1e-5 and np.abs(loss.numpy()).max() <= 1e-6
    x[2, 3] = np.nan
    loss, lse = T.dense_cross_entropy(dev(x), dev(w), dev(t), dev(b))
    assert np.isnan(lse.numpy()).tolist() == [False, False, True, False, False, False] and np.isnan(loss.numpy()[2])
    lse = T.dense_cross_entropy(dev(x), dev(w), dev(t), dev(np.full(n, -np.inf, np.float32)))[1].numpy()
    assert np.isneginf(lse[[0, 1, 3, 4, 5]]).all() and np.isnan(lse[2])


@gpu
def test_weights_whose_rows_and_columns_differ_in_size():
    """Rows of the weights 2^-30 .. 2^30 against columns of x the other way, a row of zeros, columns 2^-30 below the others."""
    for m, k, n in ((200, 60, 20000), (200, 60, 300)):
        x, w, b, t = ce_inputs(m, k, n, 30)
        e = np.random.default_rng(1).integers(-30, 31, k)
        x, w = np.ldexp(x, e).astype(np.float32), np.ldexp(w, -e[:, None]).astype(np.float32)
        w[7] = 0.0
        w[:, ::9] *= np.float32(2.0 ** -30)
        check_ce_grad(x, w, b, t, np.ones(m, np.float32))


@gpu
def test_memory_that_holds_anything():
    """Scratch comes from a pool of freed tensors: what they held does not show."""
    cx, cw, cb, ct = ce_inputs(150, 75, 333, 26)
    sx, sw, sb, st = ce_inputs(60, 75, 333, 27)
    fx, fw, fb, ft = ce_inputs(60, 75, 11, 27)
    x, wg, wu, bg, bu = gated_inputs(150, 75, 131, 26)
    yx, yg, yu, yb, yc = gated_inputs(40, 75, 131, 26)
    g, u, dout = (np.random.default_rng(i).normal(0, 1, (150, 131)).astype(np.float32) for i in range(3))
    nx, gamma, beta, dy = norm_inputs(300, 261, 26)
    d = [dev(a) for a in (x, wg, wu, bg, bu, g, u, dout, nx, gamma, beta, dy)]
    e = [[dev(a) for a in q] for q in ((cx, cw, ct, cb), (sx, sw, st, sb), (fx, fw, ft, fb))]
    small = [dev(a) for a in (yx, yg, yu, yb, yc)]

    def all_of():
        out = [T.layer_norm(d[8], d[9], d[10]), *T.layer_norm_grad(d[8], d[11], d[9]), T.dense_gated(*d[:5]), T.dense_gated(*small)]
        out += T.dense_gated_grad(*d[:3], *d[5:8], bias=True)
        for cx, cw, ct, cb in e:
            loss, lse = T.dense_cross_entropy(cx, cw, ct, cb)
            out += [loss, lse, *T.dense_cross_entropy_grad(cx, cw, ct, lse, cb)]
        return [a.numpy().tobytes() for a in out]

    want = all_of()
    for value in (math.nan, math.inf, -3e38):
        for size in (1 << 12, 1 << 16, 1 << 20, 1 << 22):
            held = [T.full([size], value) for _ in range(6)]
            T.sync()
            del held
        assert all_of() == want, value


@gpu
@pytest.mark.parametrize("precision", ["3xtf32", "bf16"])
@pytest.mark.parametrize("m,k,n", [(300, 64, 200), (60, 64, 200), (8, 64, 200), (300, 64, 10), (300, 64, 24), (300, 1100, 10), (9, 64, 32)])
def test_padding_rows_may_hold_nan(m, k, n, precision):
    L.check(L.lib.ct_set_precision(L.PREC_BF16 if precision == "bf16" else L.PREC_3XTF32))
    try:
        padding_rows(m, k, n)
    finally:
        L.check(L.lib.ct_set_precision(L.PREC_3XTF32))


def padding_rows(m, k, n):
    """Rows without a target: whatever x holds there, their loss is 0 and they have no part in the gradients."""
    x, w, b, t = ce_inputs(m, k, n, 28)
    t[:] = np.random.default_rng(0).integers(0, n, m)
    t[::5] = -1
    clean = x.copy()
    clean[::5] = 0.0
    x[::5] = np.nan
    x[5 % m] = np.inf if m > 5 else np.nan
    x[0] = np.nan
    mask = t >= 0
    x[mask] = clean[mask]
    dl = np.ones(m, np.float32)
    dl[~mask] = np.nan
    want_loss, want_lse = T.dense_cross_entropy(dev(clean), dev(w), dev(t), dev(b))
    loss, lse = T.dense_cross_entropy(dev(x), dev(w), dev(t), dev(b))
    off = 1e-5 * (1 + np.abs(want_loss.numpy()))
    assert (np.abs(loss.numpy() - want_loss.numpy()) <= off).all() and not loss.numpy()[~mask].any()
    want = T.dense_cross_entropy_grad(dev(clean), dev(w), dev(t), want_lse, dev(b), dev(np.where(mask, dl, 1).astype(np.float32)))
    got = T.dense_cross_entropy_grad(dev(x), dev(w), dev(t), lse, dev(b), dev(dl))
    assert not got[0].numpy()[~mask].any()
    for a, r in zip(got, want):
        r = r.numpy().astype(np.float64)
        assert np.abs(a.numpy() - r).max() <= 1e-5 * np.abs(r).max()


@gpu
def test_two_recordings_replayed_on_two_streams():
    import torch

    def recording(seed):
        x, wg, wu, bg, bu = [dev(a) for a in gated_inputs(200, 96, 260, seed)]
        cx, cw, cb, ct = [dev(a) for a in ce_inputs(200, 96, 700, seed)]
        nx, gamma, beta, dy = [dev(a) for a in norm_inputs(200, 300, seed)]

        def run():
            h, g, u = T.dense_gated(x, wg, wu, bg, bu, keep=True)
            loss, lse = T.dense_cross_entropy(cx, cw, ct, cb)
            return [h, *T.dense_gated_grad(x, wg, wu, g, u, h, bias=True), loss, *T.dense_cross_entropy_grad(cx, cw, ct, lse, cb),
                    T.layer_norm(nx, gamma, beta), *T.layer_norm_grad(nx, dy, gamma)]

        want = [a.numpy().tobytes() for a in run()]
        with T.Graph() as graph:
            graph.keep = run()
        return graph, want, (x, wg, wu, bg, bu, cx, cw, cb, ct, nx, gamma, beta, dy)

    pair = [recording(s) for s in (31, 32)]
    streams = [torch.cuda.Stream() for _ in pair]
    T.sync()
    try:
        for _ in range(10):
            for (graph, _, _), s in zip(pair, streams):
                L.check(L.lib.ct_set_stream(s.cuda_stream))
                graph.launch()
        torch.cuda.synchronize()
    finally:
        L.check(L.lib.ct_set_stream(None))
    T.check_async()
    for graph, want, _ in pair:
        assert [a.numpy().tobytes() for a in graph.keep] == want


@gpu
def test_a_recorded_failure_is_reported():
    """With the time-out word set the products return at once, and the next check says so; after it they compute again."""
    x, wg, wu, bg, bu = [dev(a) for a in gated_inputs(200, 96, 260, 33)]
    want = T.dense_gated(x, wg, wu, bg, bu).numpy().tobytes()
    L.check(L.lib.ct_inject_status(2, 1))
    T.dense_gated(x, wg, wu, bg, bu)
    small = T.wrap_device(x.ptr, L.F32, (40, 96), keep=x)
    T.dense_gated(small, wg, wu, bg, bu)
    with pytest.raises(L.CamelTensorError) as e:
        T.check_async()
    assert e.value.status == L.ERR_TIMEOUT
    assert T.dense_gated(x, wg, wu, bg, bu).numpy().tobytes() == want
    T.check_async()


@gpu
def test_gradients_against_differences():
    """Differences of the forward calls themselves: the slope along a random direction, in steps that float32 losses resolve."""
    rng = np.random.default_rng(41)
    m, k, n, v = 40, 32, 48, 90
    f = lambda s, *shape: rng.normal(0, s, shape).astype(np.float32)  # noqa: E731
    x, wg, wu, wv, gamma, beta = f(1, m, k), f(0.3, k, n), f(0.3, k, n), f(0.3, n, v), 1 + f(0.1, k), f(0.1, k)
    t = rng.integers(0, v, m)

    def loss(x, wg, wu, wv, gamma, beta):
        y = T.layer_norm(dev(x), dev(gamma), dev(beta))
        return T.dense_cross_entropy(T.dense_gated(y, dev(wg), dev(wu), gate="gelu"), dev(wv), dev(t))[0].numpy().astype(np.float64).sum()

    args = [x, wg, wu, wv, gamma, beta]
    y = T.layer_norm(dev(x), dev(gamma), dev(beta))
    h, g, u = T.dense_gated(y, dev(wg), dev(wu), gate="gelu", keep=True)
    _, lse = T.dense_cross_entropy(h, dev(wv), dev(t))
    dh, dwv = T.dense_cross_entropy_grad(h, dev(wv), dev(t), lse)
    dy, dwg, dwu = T.dense_gated_grad(y, dev(wg), dev(wu), g, u, dh, gate="gelu")
    dx, dgamma, dbeta = T.layer_norm_grad(dev(x), dy, dev(gamma))
    for i, grad in enumerate((dx, dwg, dwu, dwv, dgamma, dbeta)):
        grad = grad.numpy().astype(np.float64)
        direction = grad / np.linalg.norm(grad)
        eps = 1e-2
        up, down = ([a if j != i else (a + s * eps * direction).astype(np.float32) for j, a in enumerate(args)] for s in (1, -1))
        step = np.sum((up[i].astype(np.float64) - down[i]) * direction)  # as rounded
        slope = (loss(*up) - loss(*down)) / step
        # the third derivative's part (eps^2 / 6 of it, a few per cent of the slope at most) and 40 losses' rounding over the step
        assert abs(slope - np.linalg.norm(grad)) <= 2e-2 * np.linalg.norm(grad) + 40 * 6 * U * 5 / eps, i
