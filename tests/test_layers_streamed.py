"""Products of 17 to 128 rows whose weights are streamed: few values of k or 2048 columns of weights, 4096 above 32 rows (3000 of many values), 16384
above 64; at any address."""
import numpy as np
import pytest

import camel_b200._lib as L
from camel_b200 import tensor as T
from test_layers import GATES, ce64, ce_inputs, check_ce, check_gated, dev, gated_inputs
from test_layers_calls import Buffer
from test_layers_precision import ce_grad_at_bounds, f64, most, SMALL, SUM, U, within

gpu = pytest.mark.gpu
GATED = [(17, 70, 2049), (20, 1, 2048), (17, 256, 5), (32, 100, 33), (31, 300, 1024), (40, 2100, 1501), (33, 65, 2050), (64, 130, 2115), (40, 200, 3001), (65, 64, 8200), (100, 65, 8193), (128, 33, 8192)]
CE = [(17, 1, 4096), (32, 256, 17), (25, 130, 129), (20, 1000, 2050), (50, 2048, 3001), (30, 130, 4100), (64, 65, 5003), (33, 300, 4601), (65, 40, 16384), (100, 96, 16401), (128, 63, 17002)]


@gpu
@pytest.mark.parametrize("m,k,n", GATED)
def test_gated(m, k, n):
    x, wg, wu, bg, bu = gated_inputs(m, k, n, 71)
    for i, gate in enumerate(GATES):
        check_gated(x, wg, wu, *((bg, bu), (None, bu), (bg, None), (None, None))[i], gate, keep=i % 2 == 0)


@gpu
@pytest.mark.parametrize("shift", [1, 2, 3])
@pytest.mark.parametrize("m,k,n", [(20, 200, 2048), (50, 65, 2050), (64, 33, 2051), (100, 130, 8196)])
def test_gated_at_any_address(m, k, n, shift):
    """The same products of the same terms, wherever they lie: the same bytes."""
    x, wg, wu, bg, bu = gated_inputs(m, k, n, 72)
    t = [Buffer(a.shape, a, (shift + i) % 4) for i, a in enumerate((x, wg, wu, bg, bu))]
    out, g, u = Buffer((m, n), None, shift), Buffer((m, n), None, (shift + 1) % 4), Buffer((m, n), None, 0)
    L.check(L.lib.ct_dense_gated(t[0].ptr, t[1].ptr, t[3].ptr, t[2].ptr, t[4].ptr, m, k, n, L.GATE_SILU, out.ptr, g.ptr, u.ptr))
    T.check_async()
    for a, b in zip((out, g, u), T.dense_gated(*[dev(a) for a in (x, wg, wu, bg, bu)], keep=True)):
        assert a.numpy().tobytes() == b.numpy().tobytes()
    for b in t:
        b.numpy()


@gpu
@pytest.mark.parametrize("decades", [2, 12])
def test_gated_lines_of_many_magnitudes(decades):
    from test_layers_precision import wide

    for m, k, n in ((20, 100, 2050), (64, 300, 2048)):
        rng = np.random.default_rng(decades)
        x, wg, wu = wide(rng, (m, k), decades), wide(rng, (k, n), decades), wide(rng, (k, n), decades)
        _, g, u = (a.numpy() for a in T.dense_gated(dev(x), dev(wg), dev(wu), keep=True))
        for got, w in ((g, wg), (u, wu)):
            a, b = f64(x, w)
            within(got, a @ b, (SUM(k) + U) * (np.abs(a) @ np.abs(b)) + SMALL(k, most(x, 1), most(w, 0)), "kept sum")


@gpu
@pytest.mark.parametrize("m,k,n", [(20, 20000, 2050), (40, 9000, 2048)])
def test_long_sums_of_one_sign(m, k, n):
    import torch

    gen = torch.Generator(device="cuda").manual_seed(k)
    x, w, v = (torch.rand(*s, device="cuda", generator=gen) * 0.5 + 0.5 for s in ((m, k), (k, n), (k, n)))
    out, g, u = (torch.empty(m, n, device="cuda") for _ in range(3))
    torch.cuda.synchronize()
    L.check(L.lib.ct_dense_gated(x.data_ptr(), w.data_ptr(), None, v.data_ptr(), None, m, k, n, L.GATE_RELU, out.data_ptr(), g.data_ptr(), u.data_ptr()))
    T.check_async()
    for got, b in ((g, w), (u, v)):
        want = x.double() @ b.double()
        assert ((got.double() - want).abs() <= (SUM(k) + U) * want).all()


@gpu
@pytest.mark.parametrize("m,k,n", CE)
def test_cross_entropy(m, k, n):
    x, w, b, t = ce_inputs(m, k, n, 73)
    check_ce(x, w, b, t)
    check_ce(x, w, None, t)


@gpu
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
@pytest.mark.parametrize("m,k,n", [(20, 70, 4096), (64, 65, 4098), (100, 40, 16387)])
def test_cross_entropy_and_gradient_without_dx(m, k, n, shift):
    """Without dx the gradient's logits are streamed, too: within the bounds of the call that has it, which has them from planes."""
    x, w, b, t = ce_inputs(m, k, n, 74)
    lse32 = ce64(x, w, b, t)[1].astype(np.float32)
    bx, bw, bb, bt, bl = (Buffer(a.shape, a, (shift + i) % 4, a.dtype.type) for i, a in enumerate((x, w, b, t.astype(np.int64), lse32)))
    loss, lse = Buffer((m,), None, shift), Buffer((m,), None, 3)
    L.check(L.lib.ct_dense_cross_entropy(bx.ptr, bw.ptr, bb.ptr, bt.ptr, m, k, n, loss.ptr, lse.ptr))
    T.check_async()
    plain = T.dense_cross_entropy(dev(x), dev(w), dev(t), dev(b))
    assert loss.numpy().tobytes() == plain[0].numpy().tobytes() and lse.numpy().tobytes() == plain[1].numpy().tobytes()
    _, want = ce_grad_at_bounds(x, w, b, t, lse32)
    dw, db, alone = Buffer((k, n), None, (shift + 1) % 4), Buffer((n,), None, 1), Buffer((n,), None, 2)
    L.check(L.lib.ct_dense_cross_entropy_grad(bx.ptr, bw.ptr, bb.ptr, bt.ptr, bl.ptr, None, m, k, n, None, dw.ptr, db.ptr))
    L.check(L.lib.ct_dense_cross_entropy_grad(bx.ptr, bw.ptr, bb.ptr, bt.ptr, bl.ptr, None, m, k, n, None, None, alone.ptr))
    T.check_async()
    for a, r in ((dw, want[1]), (db, want[2])):
        assert np.abs(a.numpy() - r).max() <= 1e-5 * np.abs(r).max()
    assert alone.numpy().tobytes() == db.numpy().tobytes()
    for q in (bx, bw, bb, bt, bl):
        q.numpy()


@gpu
def test_padding_masked_classes_and_values_that_are_no_numbers():
    m, k, n = 40, 64, 4200
    x, w, b, t = ce_inputs(m, k, n, 75)
    t[:] = np.random.default_rng(0).integers(0, 20, m)
    t[::5] = -1
    x[::5] = np.nan
    b[20:] = -np.inf
    clean = np.where(np.isnan(x), 0.0, x).astype(np.float32)
    _, lse64, loss64, has, _, _ = ce64(clean, w[:, :20], b[:20], t)
    loss, lse = (a.numpy() for a in T.dense_cross_entropy(dev(x), dev(w), dev(t), dev(b)))
    assert np.allclose(loss, loss64, rtol=0, atol=4e-5) and np.allclose(lse[has], lse64[has], rtol=0, atol=2e-5)
    dw, db = T.zeros([k, n]), T.zeros([n])
    d = [dev(a) for a in (x, w, b, t, lse)]
    L.check(L.lib.ct_dense_cross_entropy_grad(d[0].ptr, d[1].ptr, d[2].ptr, d[3].ptr, d[4].ptr, None, m, k, n, None, dw.ptr, db.ptr))
    assert np.isfinite(dw.numpy()).all() and np.isfinite(db.numpy()).all() and not dw.numpy()[:, 20:].any() and not db.numpy()[20:].any()
    x[3, 5] = np.nan
    lse = T.dense_cross_entropy(dev(x), dev(w), dev(t), dev(b))[1].numpy()
    assert np.isnan(lse[3]) and np.isfinite(lse[[r for r in range(m) if has[r] and r != 3]]).all()


@gpu
def test_a_recorded_failure_is_reported():
    """With the time-out word set the streamed product returns at once as well; after the check it computes again."""
    t = [dev(a) for a in gated_inputs(40, 96, 2100, 76)]
    want = T.dense_gated(*t).numpy().tobytes()
    L.check(L.lib.ct_inject_status(2, 1))
    T.dense_gated(*t)
    with pytest.raises(L.CamelTensorError) as e:
        T.check_async()
    assert e.value.status == L.ERR_TIMEOUT
    assert T.dense_gated(*t).numpy().tobytes() == want
    T.check_async()
