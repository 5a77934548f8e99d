"""Embedding lookup, the gated scan and distillation from a teacher's top logits, with their gradients.

Each is compared with its definition in 64 bits.  Bounds are derived, per output value, with U = 2^-24 (half a step of float32, relative):
 * the smaller of a and 1 - a of a gate: 2^-22 of the exponential, and four roundings: 8 U of itself.
 * sums of float32: depth x U of the sum of magnitudes, depth the longest chain of additions; expf and the like 4 U of the value, and of an argument's
   error its slope.
"""
import numpy as np
import pytest

import camel_b200._lib as L
from camel_b200 import tensor as T
from camel_b200._lib import CamelTensorError
from test_layers import U, dev, within
from test_layers_calls import Buffer

gpu = pytest.mark.gpu
TINY = 2.0 ** -149
# The smaller of a and 1 - a: 0 below 2^-126, or (a, of many steps) not below that of the gate -87.33654022, 4.53e-6 short of 126 ln 2: 2^-126 times
# 1 + 4.53e-6, and 7 U of it.  Either way off by less than
FLUSHED = 2.0 ** -126 * (1 + 2.0 ** -17)


# ---- embedding ------------------------------------------------------------------------------------


def embedding_inputs(m, n, k, seed=0):
    rng = np.random.default_rng(seed + 7919 * m + 31 * n + k)
    ids = np.minimum((np.power(n + 1.0, rng.uniform(0, 1, m)) - 1).astype(np.int64), max(n - 1, 0))
    strange = rng.uniform(0, 1, m) < 0.1
    ids[strange] = rng.choice(np.array([-1, n, n + 5, 2 ** 32, -2 ** 63, 2 ** 63 - 1], np.int64), strange.sum())
    return ids, rng.normal(0, 1, (n, k)).astype(np.float32), rng.normal(0, 1, (m, k)).astype(np.float32)


def lookup32(table, ids, scale):
    out = np.zeros((len(ids), table.shape[1]), np.float32)
    has = (ids >= 0) & (ids < len(table))
    out[has] = table[ids[has]] * np.float32(scale)
    return out


def embedding_grad64(ids, dout, n, scale):
    """The sums, and those of the magnitudes."""
    has = (ids >= 0) & (ids < n)
    want, size = np.zeros((n, dout.shape[1])), np.zeros((n, dout.shape[1]))
    s = float(np.float32(scale))
    np.add.at(want, ids[has], dout[has].astype(np.float64) * s)
    np.add.at(size, ids[has], np.abs(dout[has].astype(np.float64) * s))
    return want, size


def embedding_grad_off(want, size, m):
    """One rounding; sums in 64 bits are off by m 2^-53 at most, twice (the oracle's too)."""
    return U * np.abs(want) + (m + 4) * 2.0 ** -51 * size + TINY


EMBEDDING_SHAPES = [(1, 1, 1), (1, 32003, 1024), (5, 3, 2), (7, 10, 16), (33, 50, 31), (64, 100, 771), (300, 37, 1030), (257, 1000, 64), (2, 5, 20001),
                    (1000, 3, 257), (40, 2000, 4096), (1537, 2050, 771)]


@gpu
@pytest.mark.parametrize("m,n,k", EMBEDDING_SHAPES)
def test_embedding(m, n, k):
    ids, table, _ = embedding_inputs(m, n, k)
    for scale in (1.0, float(np.sqrt(k)), -0.3):
        got = T.embedding(dev(table), dev(ids), scale)
        assert got.shape == (m, k) and got.numpy().tobytes() == lookup32(table, ids, scale).tobytes()


@gpu
@pytest.mark.parametrize("m,n,k", EMBEDDING_SHAPES + [(5000, 300, 5), (9000, 70000, 24), (40000, 1000, 8), (3000, 1, 40), (100, 1500000, 2), (70000, 131072, 3),
                                                     (1025, 500, 6), (2049, 500, 70), (8193, 60, 4), (17000, 40, 4), (33000, 300, 3), (140000, 2000, 2), (300000, 70, 1),
                                                     (65, 129, 65), (700, 60, 100), (3000, 200, 60), (1024, 700, 1030), (900, 200000, 12), (2048, 512, 512), (4096, 513, 300),
                                                     (4096, 3, 1000), (1030, 4000, 700), (5, 2, 8388737), (4097, 40, 100), (1025, 4, 300), (1025, 5, 300), (1024, 1, 130),
                                                     (3000, 149 * 4, 129), (2000, 13000, 1300), (60, 600000, 3), (8192, 300, 40)])
def test_embedding_grad(m, n, k):
    ids, _, dout = embedding_inputs(m, n, k, 1)
    want, size = embedding_grad64(ids, dout, n, 3.7)
    got = T.embedding_grad(dev(ids), dev(dout), n, 3.7)
    assert got.shape == (n, k)
    within(got.numpy(), want, embedding_grad_off(want, size, m), "dtable")


@gpu
@pytest.mark.parametrize("m,n,k", [(1, 50, 8), (4000, 50, 8), (20000, 5000, 300), (3000, 4, 2050), (3000, 13, 2050), (5000, 4, 2050)])
@pytest.mark.parametrize("which", ["one", "last", "two", "none", "all", "descending"])
def test_embedding_grad_of_uneven_tokens(m, n, k, which):
    """All tokens one row (it lies across every slice), two rows by turns, none of the table's, every row as often, in the other order."""
    dout = np.random.default_rng(m + k).normal(0, 1, (m, k)).astype(np.float32)
    i = np.arange(m)
    ids = dict(one=0 * i + n // 2, last=0 * i + n - 1, two=np.where(i % 2, 1, n - 1), none=0 * i - 1, all=i % n, descending=(m - 1 - i) * n // m)[which]
    want, size = embedding_grad64(ids, dout, n, 1.0)
    got = T.embedding_grad(dev(ids), dev(dout), n)
    within(got.numpy(), want, embedding_grad_off(want, size, m), which)
    for _ in range(3):
        assert T.embedding_grad(dev(ids), dev(dout), n).numpy().tobytes() == got.numpy().tobytes()


@gpu
@pytest.mark.parametrize("m", [3001, 9001])
def test_embedding_grad_meets_64_bits(m):
    """Terms that cancel: 2^20 and its negative around small ones, which a float32 sum would lose."""
    n, k = 7, 33
    rng = np.random.default_rng(5)
    dout = rng.normal(0, 1, (m, k)).astype(np.float32)
    dout[::3], dout[1::3] = 2.0 ** 20, -2.0 ** 20
    dout[m - 1] = 0.25
    ids = np.zeros(m, np.int64) + 3
    want, size = embedding_grad64(ids, dout, n, 1.0)
    within(T.embedding_grad(dev(ids), dev(dout), n).numpy(), want, embedding_grad_off(want, size, m), "dtable")


@gpu
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
@pytest.mark.parametrize("m,n,k", [(9, 20, 7), (70, 33, 64), (300, 40, 260), (40, 9, 771), (5, 300, 2048), (5000, 40, 771), (2000, 2000, 772), (6000, 300, 64)])
def test_embedding_at_any_address(m, n, k, shift):
    ids, table, dout = embedding_inputs(m, n, k, 2)
    bt, bi, out = Buffer(table.shape, table, shift), Buffer(ids.shape, ids, 1, np.int64), Buffer((m, k), None, (shift * 3) % 4)
    L.check(L.lib.ct_embedding(bt.ptr, bi.ptr, m, n, k, 2.5, out.ptr))
    assert out.numpy().tobytes() == lookup32(table, ids, 2.5).tobytes()
    bd, grad = Buffer(dout.shape, dout, shift), Buffer((n, k), None, (shift + 2) % 4)
    L.check(L.lib.ct_embedding_grad(bi.ptr, bd.ptr, m, n, k, 2.5, grad.ptr))
    want, size = embedding_grad64(ids, dout, n, 2.5)
    within(grad.numpy(), want, embedding_grad_off(want, size, m), "dtable")
    bt.numpy(), bi.numpy(), bd.numpy()


@gpu
def test_embedding_of_nothing():
    table, none = dev(np.ones((5, 8), np.float32)), dev(np.zeros(0, np.int64))
    assert T.embedding(table, none).shape == (0, 8)
    assert not T.embedding_grad(none, dev(np.zeros((0, 8), np.float32)), 5).numpy().any()
    ids = dev(np.array([[0, 4, -1], [2, 9, 2]]))
    assert T.embedding(dev(np.zeros((0, 8), np.float32)), ids).numpy().tobytes() == np.zeros((2, 3, 8), np.float32).tobytes()
    assert T.embedding_grad(ids, dev(np.ones((2, 3, 8), np.float32)), 0).shape == (0, 8)
    got = T.embedding_grad(ids, dev(np.ones((2, 3, 8), np.float32)), 5).numpy()  # ids of any shape
    assert got[:, 0].tolist() == [1, 0, 2, 0, 1]
    assert T.embedding(table, ids).numpy()[..., 0].tolist() == [[1, 1, 0], [1, 0, 1]]


@gpu
def test_embedding_of_infinities_and_nan():
    """They stay in their rows; at padding they are not looked at."""
    table = np.ones((6, 70), np.float32)
    table[1, 3], table[2, 69], table[3] = np.nan, np.inf, -np.inf
    ids = np.array([0, 1, 2, 3, -1, 6])
    got = T.embedding(dev(table), dev(ids), 2.0).numpy()
    np.testing.assert_array_equal(got, lookup32(table, ids, 2.0))
    dout = np.ones((6, 70), np.float32)
    dout[4:], dout[1, 5] = np.nan, np.inf
    got = T.embedding_grad(dev(ids), dev(dout), 6).numpy()
    assert np.isposinf(got[1, 5]) and np.isfinite(np.delete(got.ravel(), 75)).all() and not got[4:].any()


# ---- gated scan -----------------------------------------------------------------------------------


def sides64(gate):
    e = np.exp(-np.abs(gate.astype(np.float64)))
    small, large = e / (1 + e), 1 / (1 + e)
    return np.where(gate >= 0, large, small), np.where(gate >= 0, small, large)  # a, 1 - a


def here_of(lengths, b, t):
    return np.arange(t)[None, :, None] < (np.full(b, t) if lengths is None else lengths)[:, None, None]


def scan64(gate, value, state0, lengths):
    """h, the last state and, by the same recurrence, the largest value so far."""
    b, t, c = gate.shape
    a, rest = sides64(gate)
    here = here_of(lengths, b, t)
    h = np.zeros((b, c)) if state0 is None else state0.astype(np.float64)
    most = np.abs(h)
    out, size = np.zeros((b, t, c)), np.zeros((b, t, c))
    for i in range(t):
        on = here[:, i]
        h = np.where(on, a[:, i] * h + rest[:, i] * np.where(on, value[:, i], 0.0), h)
        most = np.where(on, np.maximum(most, np.abs(np.where(on, value[:, i], 0.0))), most)
        out[:, i], size[:, i] = np.where(on, h, 0.0), np.where(on, most, 0.0)
    return out, h, size, most


# Of the largest value so far (M): the gates' errors, 8 U (1 - a) 2 M a step, are 16 U M in a sum that forgets at that rate; a lane's 16 steps round
# twice each, in 32 U M; the state that they begin with is rounded once, and what pieces of 16 steps do to it is off by less than 2 U per step and value
# that the piece has taken up, again 32 U M at most, twice (1 - a and a value each).  In all 113 U M.
SCAN = 128 * U


def scan_grad64(gate, value, state0, lengths, out, dout, dstate):
    """The gradients, and bounds of their errors."""
    b, t, c = gate.shape
    a, rest = sides64(gate)
    small = np.minimum(a, rest)
    here = here_of(lengths, b, t)
    carry = np.zeros((b, c)) if dstate is None else dstate.astype(np.float64)
    size, off = np.abs(carry), np.zeros((b, c))  # of the same sum of magnitudes, and of what the states between pieces are off by
    first = np.zeros((b, 1, c)) if state0 is None else state0.astype(np.float64)[:, None]
    gap = np.concatenate([first, out[:, :-1].astype(np.float64)], 1) - value
    gap_size = np.abs(np.concatenate([first, out[:, :-1].astype(np.float64)], 1)) + np.abs(value)
    dgate, dvalue, off_gate, off_value = (np.zeros((b, t, c)) for _ in range(4))
    near = np.zeros((16, b, c))  # the last 16 steps' magnitudes
    for i in reversed(range(t)):
        on = here[:, i]
        near[i % 16] = np.where(on, np.abs(dout[:, i]), 0.0)
        d = np.where(on, dout[:, i], 0.0).astype(np.float64)
        g, g_size = d + carry, np.abs(d) + size
        # 16 steps of two roundings, the beginning's, what the state lacks.  The smaller of a and 1 - a, and what it multiplies, is off by FLUSHED
        # of its other factors
        e = off + 40 * U * g_size
        s, p = rest[:, i], a[:, i]
        dvalue[:, i], off_value[:, i] = np.where(on, s * g, 0.0), np.where(on, s * (e + 12 * U * g_size) + FLUSHED * g_size, 0.0)
        with np.errstate(invalid="ignore"):
            dgate[:, i] = np.where(on, p * s * g * gap[:, i], 0.0)
            off_gate[:, i] = np.where(on, p * s * (np.abs(gap[:, i]) * (e + 24 * U * g_size) + U * g_size * gap_size[:, i])
                                      + FLUSHED * g_size * gap_size[:, i], 0.0)
        carry, size = np.where(on, p * g, carry), np.where(on, p * g_size, size)
        # a piece's own sum rounds twice a step (and once more for the gate), what it does to the state is off by its gates' errors
        off = np.where(on, p * off + 3 * U * near.sum(0) + (24 * U * small[:, i] + FLUSHED) * g_size, off)
    return (dgate, dvalue, carry), (off_gate + TINY, off_value + TINY, off + U * size + TINY)


SCAN_SHAPES = [(1, 1, 1), (3, 1, 70), (64, 1, 2048), (2, 2, 5), (2, 5, 33), (3, 17, 40), (1, 129, 32), (4, 300, 40), (1, 2000, 3), (2, 4100, 5), (7, 700, 77),
               (1, 20000, 31), (70, 17, 100), (1, 1025, 513), (33, 130, 257),
               (5, 23, 96), (3, 19, 33), (2, 50, 45), (1, 5000, 260), (3, 2500, 1001), (2, 31, 34), (60, 64, 36)]


def scan_inputs(b, t, c, seed=0):
    rng = np.random.default_rng(seed + 7919 * b + 31 * t + c)
    gate = (rng.normal(0, 1, (b, t, c)) + rng.uniform(-3, 9, c)).astype(np.float32)
    f = lambda *shape: rng.normal(0, 1, shape).astype(np.float32)  # noqa: E731
    lengths = rng.integers(0, t + 1, b)
    lengths[0] = t
    if b > 2:
        lengths[1], lengths[2] = 0, 1
    return gate, f(b, t, c), f(b, c), lengths, f(b, t, c), f(b, c)


def maybe(a):
    return None if a is None else dev(a)


@gpu
@pytest.mark.parametrize("b,t,c", SCAN_SHAPES)
@pytest.mark.parametrize("padded", [False, True])
def test_gated_scan(b, t, c, padded):
    gate, value, state0, lengths, _, _ = scan_inputs(b, t, c)
    given = lengths if padded else None
    for first in (state0, None):
        out, last = T.gated_scan(dev(gate), dev(value), maybe(first), maybe(given))
        want, want_last, size, most = scan64(gate, value, first, given)
        within(out.numpy(), want, SCAN * size, "out")
        within(last.numpy(), want_last, SCAN * most + TINY, "state")


@gpu
@pytest.mark.parametrize("b,t,c", SCAN_SHAPES)
@pytest.mark.parametrize("padded", [False, True])
def test_gated_scan_grad(b, t, c, padded):
    gate, value, state0, lengths, dout, dstate = scan_inputs(b, t, c, 1)
    given = lengths if padded else None
    for first, last in ((state0, dstate), (None, None), (state0, None)):
        out = scan64(gate, value, first, given)[0].astype(np.float32)
        got = T.gated_scan_grad(dev(gate), dev(value), dev(out), dev(dout), maybe(first), maybe(given), maybe(last))
        want, off = scan_grad64(gate, value, first, given, out, dout, last)
        assert len(got) == (2 if first is None else 3)
        for name, x, y, z in zip(("dgate", "dvalue", "dstate0"), got, want, off):
            within(x.numpy(), y, z, name)


def test_the_gradient_is_the_slope():
    """The 64-bit gradient that the kernels are held to, against differences of the 64-bit recurrence, every input by itself."""
    b, t, c = 2, 5, 2
    gate, value, state0, lengths, dout, dstate = scan_inputs(b, t, c, 2)
    lengths[:] = [5, 3]
    args = [a.astype(np.float64) for a in (gate, value, state0)]

    def total(g, v, s):
        out, last, _, _ = scan64(g, v, s, lengths)
        return (out * np.where(here_of(lengths, b, t), dout, 0.0)).sum() + (last * dstate).sum()

    out = scan64(*args, lengths)[0]
    want, _ = scan_grad64(*args, lengths, out, dout, dstate)
    for k, grad in enumerate(want):
        for at in np.ndindex(*grad.shape):
            up, down = ([a.copy() for a in args] for _ in range(2))
            up[k][at] += 1e-5
            down[k][at] -= 1e-5
            assert abs((total(*up) - total(*down)) / 2e-5 - grad[at]) <= 1e-8, (k, at)


@gpu
@pytest.mark.parametrize("gates", [(0.0, 0.0), (40.0, 40.0), (-40.0, -40.0), (100.0, -100.0), (np.inf, -np.inf), (16.0, 17.0), (-1e-30, 1e-30)])
def test_gates_at_their_ends(gates):
    """Gates that keep everything, nothing, or by turns; 1 - a of 2^-24 and below, which 1 - a in float32 would not show."""
    b, t, c = 2, 3000, 40
    _, value, state0, _, dout, dstate = scan_inputs(b, t, c, 3)
    gate = np.empty((b, t, c), np.float32)
    gate[:, ::2], gate[:, 1::2] = gates
    out, last = T.gated_scan(dev(gate), dev(value), dev(state0))
    want, want_last, size, most = scan64(gate, value, state0, None)
    within(out.numpy(), want, SCAN * size, "out")
    within(last.numpy(), want_last, SCAN * most, "state")
    o32 = want.astype(np.float32)
    got = T.gated_scan_grad(dev(gate), dev(value), dev(o32), dev(dout), dev(state0), None, dev(dstate))
    for name, x, y, z in zip(("dgate", "dvalue", "dstate0"), got, *scan_grad64(gate, value, state0, None, o32, dout, dstate)):
        within(x.numpy(), y, z, name)


@gpu
def test_a_state_that_only_decays_keeps_its_digits():
    """Values of 0: h is a product of gates, and as exact as its factors (8 U (1 - a) / a or 8 U each, and three roundings) however small it gets."""
    b, t, c = 2, 60, 33
    gate, _, state0, _, _, _ = scan_inputs(b, t, c, 4)
    value = np.zeros_like(gate)
    out, _ = T.gated_scan(dev(gate), dev(value), dev(state0))
    want = scan64(gate, value, state0, None)[0]
    a, rest = sides64(gate)
    off = np.cumsum(8 * U * np.minimum(1.0, rest / a) + 3 * U, 1)
    # pieces: 1 - the product of a has as many roundings as steps, and is subtracted from 1 where it is below 1/2
    within(out.numpy(), want, (2 * off + 40 * U) * np.abs(want) + 2.0 ** -120, "out")


@gpu
def test_padding_may_hold_anything():
    b, t, c = 5, 700, 37
    gate, value, state0, lengths, dout, dstate = scan_inputs(b, t, c, 5)
    lengths[:] = [0, 1, 699, 350, 700]
    here = here_of(lengths, b, t)
    want = [a.numpy().tobytes() for a in T.gated_scan(dev(gate), dev(value), dev(state0), dev(lengths))]
    out = scan64(gate, value, state0, lengths)[0].astype(np.float32)
    want_grad = [a.numpy().tobytes() for a in T.gated_scan_grad(dev(gate), dev(value), dev(out), dev(dout), dev(state0), dev(lengths), dev(dstate))]
    for bad in (np.nan, np.inf, -3e38):
        g, v, o, d = (np.where(here, a, np.float32(bad)) for a in (gate, value, out, dout))
        assert [a.numpy().tobytes() for a in T.gated_scan(dev(g), dev(v), dev(state0), dev(lengths))] == want
        assert [a.numpy().tobytes() for a in T.gated_scan_grad(dev(g), dev(v), dev(o), dev(d), dev(state0), dev(lengths), dev(dstate))] == want_grad
    # lengths beyond the ends are the ends
    wide = lengths.copy()
    wide[0], wide[4] = -2 ** 63, 2 ** 63 - 1
    assert [a.numpy().tobytes() for a in T.gated_scan(dev(gate), dev(value), dev(state0), dev(wide))] == want


@gpu
@pytest.mark.parametrize("cuts", [[1, 299], [150, 150], [297, 1, 1, 1], [17, 283]])
def test_the_state_carries_from_call_to_call(cuts):
    b, c = 3, 50
    gate, value, state0, _, _, _ = scan_inputs(b, 300, c, 6)
    want, want_last, size, most = scan64(gate, value, state0, None)
    state, at, parts = dev(state0), 0, []
    for n in cuts:
        out, state = T.gated_scan(dev(gate[:, at:at + n]), dev(value[:, at:at + n]), state)
        parts.append(out.numpy())
        at += n
    within(np.concatenate(parts, 1), want, (SCAN + len(cuts) * U) * size, "out")
    within(state.numpy(), want_last, (SCAN + len(cuts) * U) * most, "state")


@gpu
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
@pytest.mark.parametrize("b,t,c", [(2, 1, 64), (3, 40, 36), (1, 700, 64), (2, 513, 33)])
def test_gated_scan_at_any_address(b, t, c, shift):
    gate, value, state0, lengths, dout, dstate = scan_inputs(b, t, c, 7)
    bg, bv, bs = Buffer(gate.shape, gate, shift), Buffer(value.shape, value, (shift + 1) % 4), Buffer(state0.shape, state0, (shift + 2) % 4)
    bl, out, last = Buffer(lengths.shape, lengths, 1, np.int64), Buffer(gate.shape, None, (shift * 3) % 4), Buffer(state0.shape, None, shift)
    L.check(L.lib.ct_gated_scan(bg.ptr, bv.ptr, bs.ptr, bl.ptr, b, t, c, out.ptr, last.ptr))
    want = T.gated_scan(dev(gate), dev(value), dev(state0), dev(lengths))
    assert out.numpy().tobytes() == want[0].numpy().tobytes() and last.numpy().tobytes() == want[1].numpy().tobytes()
    bd, be = Buffer(dout.shape, dout, (shift + 3) % 4), Buffer(dstate.shape, dstate, shift)
    dg, dv, ds = Buffer(gate.shape, None, shift), Buffer(gate.shape, None, (shift + 2) % 4), Buffer(state0.shape, None, 1)
    L.check(L.lib.ct_gated_scan_grad(bg.ptr, bv.ptr, bs.ptr, bl.ptr, out.ptr, bd.ptr, be.ptr, b, t, c, dg.ptr, dv.ptr, ds.ptr))
    grads = T.gated_scan_grad(dev(gate), dev(value), want[0], dev(dout), dev(state0), dev(lengths), dev(dstate))
    for x, y in zip((dg, dv, ds), grads):
        assert x.numpy().tobytes() == y.numpy().tobytes()
    for x in (bg, bv, bs, bl, bd, be, out):
        x.numpy()
    # outputs one at a time, and states in place
    for alone in range(3):
        outs = [Buffer(s, None, 0) if i == alone else None for i, s in enumerate((gate.shape, gate.shape, state0.shape))]
        L.check(L.lib.ct_gated_scan_grad(bg.ptr, bv.ptr, bs.ptr, bl.ptr, out.ptr, bd.ptr, be.ptr, b, t, c, *[None if o is None else o.ptr for o in outs]))
        assert outs[alone].numpy().tobytes() == grads[alone].numpy().tobytes()
    only = Buffer(gate.shape, None, 0)
    L.check(L.lib.ct_gated_scan(bg.ptr, bv.ptr, bs.ptr, bl.ptr, b, t, c, only.ptr, None))
    assert only.numpy().tobytes() == want[0].numpy().tobytes()
    L.check(L.lib.ct_gated_scan(bg.ptr, bv.ptr, bs.ptr, bl.ptr, b, t, c, None, bs.ptr))
    assert bs.numpy().tobytes() == want[1].numpy().tobytes()
    bs = Buffer(state0.shape, state0, 0)
    L.check(L.lib.ct_gated_scan_grad(bg.ptr, bv.ptr, bs.ptr, bl.ptr, out.ptr, bd.ptr, be.ptr, b, t, c, None, None, be.ptr))
    assert be.numpy().tobytes() == grads[2].numpy().tobytes()


@gpu
def test_scans_of_nothing():
    e = np.zeros((2, 0, 5), np.float32)
    s = np.arange(10, dtype=np.float32).reshape(2, 5)
    out, last = T.gated_scan(dev(e), dev(e), dev(s))
    assert out.shape == (2, 0, 5) and last.numpy().tobytes() == s.tobytes()
    assert not T.gated_scan(dev(e), dev(e))[1].numpy().any()
    assert T.gated_scan_grad(dev(e), dev(e), dev(e), dev(e), dev(s), None, dev(s + 1))[2].numpy().tobytes() == (s + 1).tobytes()
    for shape in ((0, 3, 5), (2, 3, 0)):
        z = np.zeros(shape, np.float32)
        out, last = T.gated_scan(dev(z), dev(z))
        assert out.shape == shape and last.shape == (shape[0], shape[2])
        T.gated_scan_grad(dev(z), dev(z), dev(z), dev(z))
    T.check_async()


@gpu
def test_infinite_values_and_nan_stay_in_their_chains():
    b, t, c = 2, 400, 40
    gate, value, state0, _, _, _ = scan_inputs(b, t, c, 8)
    want = T.gated_scan(dev(gate), dev(value), dev(state0))[0].numpy()
    value[0, 200, 7], gate[1, 100, 9], value[1, 399, 3] = np.inf, np.nan, np.nan
    got = T.gated_scan(dev(gate), dev(value), dev(state0))[0].numpy()
    bad = np.zeros((b, t, c), bool)
    bad[0, 200:, 7], bad[1, 100:, 9], bad[1, 399, 3] = True, True, True
    assert not np.isfinite(got[bad]).any() and got[~bad].tobytes() == want[~bad].tobytes()


# ---- distillation ---------------------------------------------------------------------------------


def distill_inputs(m, n, top, seed=0):
    rng = np.random.default_rng(seed + 7919 * m + 31 * n + top)
    z = rng.normal(0, 3, (m, n)).astype(np.float32)
    ids = rng.integers(0, n, (m, top))  # the same class twice, now and then
    teacher = (rng.normal(0, 2, (m, top)) + 5).astype(np.float32)
    ids[rng.uniform(0, 1, (m, top)) < 0.1] = -1
    ids[rng.uniform(0, 1, (m, top)) < 0.05] = n
    ids[1::5] = -1  # rows of padding
    return z, ids, teacher, rng.uniform(0.5, 2, m).astype(np.float32)


def distill64(z, ids, teacher, temperature):
    """p, lse, loss and bounds of lse and loss."""
    m, n = z.shape
    w = float(np.float32(temperature))
    x = z.astype(np.float64) / w
    has = (ids >= 0) & (ids < n)
    at = np.where(has, ids, 0)
    some = has.any(1)
    top = x.max(1, keepdims=True)
    e = np.exp(x - top)
    lse = (top + np.log(e.sum(1, keepdims=True)))[:, 0]
    # a term is off by the roundings of its argument (3 U of it) and 2^-22 + U of itself; the sum by a chain of n / 4096 groups of 16 terms, six
    # additions each, and eleven joins of four roundings and an exponential
    rel = U * ((e * (3 * np.abs(x - top) + 5)).sum(1) / e.sum(1) + 6 * (n / 4096 + 1) + 11 * 9)
    off_lse = rel + U * (4 * np.abs(np.log(e.sum(1))) + 2 * np.abs(top[:, 0]) + np.abs(lse)) + TINY
    u = np.where(has, teacher.astype(np.float64) / w, -np.inf)
    u = u - np.where(some, u.max(1), 0.0)[:, None]
    eu = np.exp(u)
    total = np.where(some, eu.sum(1), 1.0)[:, None]
    p = eu / total
    gap = np.where(has, np.where(has, u, 0.0) - np.log(total) - (np.take_along_axis(x, at, 1) - lse[:, None]), 0.0)
    loss = w * w * (p * gap).sum(1)
    depth = ids.shape[1] / 32 + 6
    arg = np.where(has, np.abs(u), 0.0)
    rel_p = U * (3 * arg + (p * 3 * arg).sum(1, keepdims=True) + depth + 12)
    off_gap = U * (3 * arg + 5 * np.abs(np.log(total)) + 3 * np.abs(np.take_along_axis(x, at, 1)) + 3 * np.abs(gap)) + off_lse[:, None]
    off = w * w * (p * off_gap + p * np.abs(gap) * (rel_p + depth * U)).sum(1) + 4 * U * np.abs(loss) + TINY
    return p, lse, np.where(some, loss, 0.0), off_lse, np.where(some, off, 0.0)


def distill_grad64(z, ids, p, lse, dloss, temperature):
    """dlogits and bounds, with the lse that the kernel was given."""
    m, n = z.shape
    w = float(np.float32(temperature))
    x = z.astype(np.float64) / w
    has = (ids >= 0) & (ids < n)
    some = has.any(1)[:, None]
    q = np.where(some, np.exp(x - lse.astype(np.float64)[:, None]), 0.0)
    weights, terms = np.zeros((m, n)), np.zeros((m, n))
    rows = np.repeat(np.arange(m)[:, None], ids.shape[1], 1)
    np.add.at(weights, (rows[has], ids[has]), p[has])
    with np.errstate(divide="ignore"):
        arg = np.where(p > 0, np.abs(np.log(np.where(p > 0, p, 1.0))), 0.0)
    rel_p = 3 * arg + (p * 3 * arg).sum(1, keepdims=True) + 3 * np.log(ids.shape[1] + 1) + ids.shape[1] / 32 + 20
    np.add.at(terms, (rows[has], ids[has]), (p * rel_p)[has])
    scale = np.where(some, w * np.asarray(dloss, np.float64)[:, None], 0.0)
    # of q: two roundings of z / T (in two parts) minus lse, its product with log2 e, the exponential, the factor; of the weights as in the loss
    rel_q = 2 * np.abs(x) + np.abs(lse)[:, None] + 4 * np.abs(x - lse[:, None]) + 10
    off = np.abs(scale) * U * (q * rel_q + terms + 4 * (q + weights)) + TINY
    return scale * (q - weights), off


DISTILL_SHAPES = [(1, 1, 1), (3, 2, 1), (5, 10, 5), (40, 10, 3), (9, 32, 32), (7, 33, 4), (70, 130, 20), (6, 512, 64), (6, 513, 64), (5, 2050, 7), (300, 1025, 1),
                  (2, 32003, 20), (64, 5000, 40), (1, 131072, 64), (3, 50257, 128), (2, 700, 1024), (2, 9, 100), (700, 4099, 9), (1500, 6000, 3),
                  (33, 20, 30), (31, 100, 50), (30, 300, 100), (3, 200, 200), (2500, 1500, 20), (2500, 5000, 33), (600, 9000, 40), (3, 25000, 5), (4000, 33, 2)]


@gpu
@pytest.mark.parametrize("m,n,top", DISTILL_SHAPES)
def test_distill(m, n, top):
    z, ids, teacher, dloss = distill_inputs(m, n, top)
    for temperature in (1.0, 2.0, 0.7):
        loss, lse = T.distill(dev(z), dev(ids), dev(teacher), temperature)
        p, want_lse, want, off_lse, off = distill64(z, ids, teacher, temperature)
        within(lse.numpy(), want_lse, off_lse, "lse")
        within(loss.numpy(), want, off, "loss")
        l32 = want_lse.astype(np.float32)
        for d in (dloss, None):
            got = T.distill_grad(dev(z), dev(ids), dev(teacher), dev(l32), temperature, maybe(d))
            grad, off_grad = distill_grad64(z, ids, p, l32, np.ones(m) if d is None else d, temperature)
            within(got.numpy(), grad, off_grad, "dlogits")


@gpu
@pytest.mark.parametrize("shift", [0, 1, 2, 3])
@pytest.mark.parametrize("m,n,top", [(5, 10, 3), (20, 300, 9), (3, 2050, 30), (2, 20001, 70), (400, 1024, 5)])
def test_distill_at_any_address(m, n, top, shift):
    z, ids, teacher, dloss = distill_inputs(m, n, top, 1)
    bz, bi, bt = Buffer(z.shape, z, shift), Buffer(ids.shape, ids, 1, np.int64), Buffer(teacher.shape, teacher, (shift + 1) % 4)
    loss, lse, bd = Buffer((m,), None, shift), Buffer((m,), None, (shift + 2) % 4), Buffer((m,), dloss, (shift + 3) % 4)
    L.check(L.lib.ct_distill(bz.ptr, bi.ptr, bt.ptr, m, n, top, 2.0, loss.ptr, lse.ptr))
    p, want_lse, want, off_lse, off = distill64(z, ids, teacher, 2.0)
    within(lse.numpy(), want_lse, off_lse, "lse")
    within(loss.numpy(), want, off, "loss")
    want, off = distill_grad64(z, ids, p, lse.numpy(), dloss, 2.0)
    for gshift in (shift, (shift + 1) % 4):  # the same distance from 16 bytes as the logits, and another
        grad = Buffer(z.shape, None, gshift)
        L.check(L.lib.ct_distill_grad(bz.ptr, bi.ptr, bt.ptr, lse.ptr, bd.ptr, m, n, top, 2.0, grad.ptr))
        within(grad.numpy(), want, off, "dlogits")
    bz.numpy()
    L.check(L.lib.ct_distill_grad(bz.ptr, bi.ptr, bt.ptr, lse.ptr, bd.ptr, m, n, top, 2.0, bz.ptr))  # in place
    within(bz.numpy(), want, off, "dlogits in place")
    for x in (bi, bt, bd, lse):
        x.numpy()
    one, other = Buffer((m,), None, 0), Buffer((m,), None, 0)
    bz = Buffer(z.shape, z, shift)
    L.check(L.lib.ct_distill(bz.ptr, bi.ptr, bt.ptr, m, n, top, 2.0, one.ptr, None))
    L.check(L.lib.ct_distill(bz.ptr, None, None, m, n, top, 2.0, None, other.ptr))
    assert one.numpy().tobytes() == loss.numpy().tobytes() and other.numpy().tobytes() == lse.numpy().tobytes()


@gpu
@pytest.mark.parametrize("n", [12, 400, 3000, 40000])
def test_distill_of_infinities_and_nan(n):
    z, ids, teacher, _ = distill_inputs(8, n, 6, 2)
    ids[:] = np.arange(6) * (n // 6)
    ids[3] = -1
    z[0, 1] = -np.inf                 # a class that is out, no entry's
    z[1, ids[1, 2]] = -np.inf         # out, and an entry's: log q is -infinity
    z[2, n - 1] = np.nan
    z[3] = np.nan                     # padding
    z[4, :] = -np.inf
    z[4, ids[4, 0]] = 1.5             # nothing but one class, all of the teacher's weight
    teacher[4, 1:] = -np.inf
    teacher[5, 2] = -np.inf           # an entry of weight 0 whose class is out
    z[5, ids[5, 2]] = -np.inf
    z[6, 0] = np.inf
    teacher[7, 3] = np.nan
    loss, lse = T.distill(dev(z), dev(ids), dev(teacher), 2.0)
    loss, l32 = loss.numpy(), lse.numpy()
    rows = [0, 5]
    with np.errstate(invalid="ignore"):
        t, l64 = np.where(np.isneginf(teacher), -1e30, teacher), None
        y = np.where(np.isneginf(z), np.float32(-1e30), z)
        p, want_lse, want, off_lse, off = distill64(y[rows], ids[rows], t[rows], 2.0)
    within(l32[rows], want_lse, U * (np.abs(want_lse) + 200), "lse")
    # (the bound of the entry of weight 0 is not one: its logit was replaced)
    assert (np.abs(loss[rows] - want) <= 2e-5 * (1 + np.abs(want))).all()
    assert np.isposinf(loss[1]) and np.isnan(loss[[2, 6, 7]]).all() and np.isnan(l32[[2, 3, 6]]).all()
    assert loss[3] == 0 and abs(loss[4]) <= 1e-6 and l32[4] == 0.75
    grad = T.distill_grad(dev(z), dev(ids), dev(teacher), lse, 2.0).numpy()
    assert not grad[3].any() and np.isfinite(grad[[0, 1, 4, 5]]).all() and np.isnan(grad[2]).all() and np.isnan(grad[6]).all()
    assert grad[0, 1] == 0 and np.abs(grad[4]).max() <= 1e-6


@gpu
def test_a_class_in_every_entry():
    """All entries the same class: its weight is 1, whatever their logits."""
    for n, top in ((10, 9), (300, 200), (5000, 1024)):
        z, ids, teacher, _ = distill_inputs(2, n, top, 3)
        ids[:] = n - 1
        loss, lse = T.distill(dev(z), dev(ids), dev(teacher), 1.0)
        p, want_lse, want, off_lse, off = distill64(z, ids, teacher, 1.0)
        within(loss.numpy(), want, off, "loss")
        l32 = want_lse.astype(np.float32)
        within(T.distill_grad(dev(z), dev(ids), dev(teacher), dev(l32)).numpy(), *distill_grad64(z, ids, p, l32, np.ones(2), 1.0), "dlogits")


@gpu
def test_distill_of_nothing():
    none = dev(np.zeros((0, 7), np.float32))
    loss, lse = T.distill(none, dev(np.zeros((0, 2), np.int64)), dev(np.zeros((0, 2), np.float32)))
    assert loss.shape == (0,) and T.distill_grad(none, dev(np.zeros((0, 2), np.int64)), dev(np.zeros((0, 2), np.float32)), lse).shape == (0, 7)
    for n in (7, 700):
        z = np.random.default_rng(1).normal(0, 1, (3, n)).astype(np.float32)
        loss, lse = T.distill(dev(z), dev(np.zeros((3, 0), np.int64)), dev(np.zeros((3, 0), np.float32)))
        assert not loss.numpy().any()
        within(lse.numpy(), *[distill64(z, np.full((3, 1), -1), np.zeros((3, 1), np.float32), 1.0)[i] for i in (1, 3)], "lse")
        assert not T.distill_grad(dev(z), dev(np.zeros((3, 0), np.int64)), dev(np.zeros((3, 0), np.float32)), lse).numpy().any()


# ---- refusals -------------------------------------------------------------------------------------


def view(shape, dtype=L.F32):
    return T.wrap_device(1 << 40, dtype, shape)  # nothing reads it: the call is refused


REFUSED = [
    lambda: T.embedding(view((5,)), view((3,), L.I64)),
    lambda: T.embedding(view((5, 2), L.I64), view((3,), L.I64)),
    lambda: T.embedding(view((5, 2)), view((3,))),
    lambda: T.embedding(view((5, 2)), None),
    lambda: T.embedding_grad(view((3,)), view((3, 2)), 5),
    lambda: T.embedding_grad(view((3,), L.I64), view((4, 2)), 5),
    lambda: T.embedding_grad(view((3,), L.I64), view((3,)), 5),
    lambda: T.embedding_grad(view((3,), L.I64), view((3, 2)), -1),
    lambda: T.gated_scan(view((2, 3)), view((2, 3))),
    lambda: T.gated_scan(view((2, 3, 4)), view((2, 3, 5))),
    lambda: T.gated_scan(view((2, 3, 4)), view((2, 3, 4), L.I64)),
    lambda: T.gated_scan(view((2, 3, 4)), view((2, 3, 4)), view((2, 5))),
    lambda: T.gated_scan(view((2, 3, 4)), view((2, 3, 4)), None, view((3,), L.I64)),
    lambda: T.gated_scan(view((2, 3, 4)), view((2, 3, 4)), None, view((2,))),
    lambda: T.gated_scan_grad(view((2, 3, 4)), view((2, 3, 4)), view((2, 3, 4)), view((2, 4, 4))),
    lambda: T.gated_scan_grad(view((2, 3, 4)), view((2, 3, 4)), view((2, 3, 4)), view((2, 3, 4)), dstate=view((3, 4))),
    lambda: T.distill(view((4, 9)), view((4, 2)), view((4, 2))),
    lambda: T.distill(view((4, 9)), view((4, 3), L.I64), view((4, 2))),
    lambda: T.distill(view((4, 9)), view((5, 2), L.I64), view((5, 2))),
    lambda: T.distill(view((4,)), view((4, 2), L.I64), view((4, 2))),
    lambda: T.distill_grad(view((4, 9)), view((4, 2), L.I64), view((4, 2)), None),
    lambda: T.distill_grad(view((4, 9)), view((4, 2), L.I64), view((4, 2)), view((3,))),
    lambda: T.distill_grad(view((4, 9)), view((4, 2), L.I64), view((4, 2)), view((4,)), 1.0, view((5,))),
]


@pytest.mark.parametrize("n", range(len(REFUSED)))
def test_refusals(n):
    with pytest.raises(CamelTensorError) as e:
        REFUSED[n]()
    assert e.value.status == L.ERR_INVALID


BIG = (1 << 29) + 1
REFUSED_BY_THE_LIBRARY = [
    (L.ERR_INVALID, lambda p: L.lib.ct_embedding(p, p, -1, 2, 2, 1.0, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_embedding(None, p, 2, 2, 2, 1.0, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_embedding(p, None, 2, 2, 2, 1.0, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_embedding(p, p, 2, 2, 2, 1.0, None)),
    (L.ERR_INVALID, lambda p: L.lib.ct_embedding(p, p, 2, 2, 2, float("nan"), p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_embedding(p, p, 2, 2, 2, 1e39, p)),
    (L.ERR_TOO_LARGE, lambda p: L.lib.ct_embedding(p, p, BIG, 0, 0, 1.0, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_embedding_grad(p, None, 2, 2, 2, 1.0, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_embedding_grad(None, p, 2, 2, 2, 1.0, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_embedding_grad(p, p, 2, 2, 2, 1.0, None)),
    (L.ERR_INVALID, lambda p: L.lib.ct_embedding_grad(p, p, 2, 2, 2, float("inf"), p)),
    (L.ERR_TOO_LARGE, lambda p: L.lib.ct_embedding_grad(p, p, 0, BIG, 0, 1.0, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_gated_scan(None, p, None, None, 1, 1, 1, p, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_gated_scan(p, None, None, None, 1, 1, 1, p, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_gated_scan(p, p, None, None, 1, -1, 1, p, p)),
    (L.ERR_TOO_LARGE, lambda p: L.lib.ct_gated_scan(p, p, None, None, 1 << 17, 0, 1 << 16, p, p)),
    (L.ERR_TOO_LARGE, lambda p: L.lib.ct_gated_scan(p, p, None, None, 0, BIG, 0, p, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_gated_scan_grad(p, p, None, None, None, p, None, 1, 1, 1, p, p, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_gated_scan_grad(p, p, None, None, p, None, None, 1, 1, 1, p, p, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_distill(p, p, p, 1, 0, 1, 1.0, p, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_distill(p, p, p, 1, 5, 1, 0.0, p, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_distill(p, p, p, 1, 5, 1, float("nan"), p, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_distill(p, p, p, 1, 5, 1, 1e7, p, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_distill(None, p, p, 1, 5, 1, 1.0, p, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_distill(p, None, p, 1, 5, 1, 1.0, p, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_distill(p, p, p, 1, 5, -1, 1.0, p, p)),
    (L.ERR_TOO_LARGE, lambda p: L.lib.ct_distill(p, p, p, 1, 5, 1025, 1.0, p, p)),
    (L.ERR_TOO_LARGE, lambda p: L.lib.ct_distill(p, p, p, 0, BIG, 1, 1.0, p, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_distill_grad(p, p, p, None, p, 1, 5, 1, 1.0, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_distill_grad(p, p, None, p, p, 1, 5, 1, 1.0, p)),
    (L.ERR_INVALID, lambda p: L.lib.ct_distill_grad(p, p, p, p, p, 1, 5, 1, 1.0, None)),
]


@gpu
@pytest.mark.parametrize("n", range(len(REFUSED_BY_THE_LIBRARY)))
def test_refusals_of_the_library(n):
    """Nothing is launched: what lies there stays."""
    status, call = REFUSED_BY_THE_LIBRARY[n]
    held = dev(np.arange(64, dtype=np.float32))
    assert call(held.ptr) == status and L.lib.ct_last_error()
    assert held.numpy().tolist() == list(range(64))


def test_without_a_device_the_entry_points_refuse():
    import torch

    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    for _, call in REFUSED_BY_THE_LIBRARY:
        assert call(0) == L.ERR_NO_DEVICE
