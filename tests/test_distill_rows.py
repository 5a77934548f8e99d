"""Distillation where its rows are hard: any temperature that is accepted, logits far from zero, classes and entries that are masked."""
import numpy as np
import pytest

import camel_b200._lib as L
from camel_b200 import tensor as T
from test_layers import U, dev, within
from test_sequences import distill64, distill_grad64, distill_inputs

gpu = pytest.mark.gpu


def exact(z, ids, teacher, temperature):
    """loss, lse and p from the definition, in 80 bits: at a temperature of 10^6 a sum of 64 bits is off by 10^12 2^-53 in the loss."""
    w = np.longdouble(np.float32(temperature))
    z, ids, teacher = np.atleast_2d(z), np.atleast_2d(ids), np.atleast_2d(teacher)
    has = (ids >= 0) & (ids < z.shape[1])
    with np.errstate(invalid="ignore"):
        x, u = z.astype(np.longdouble) / w, np.where(has, teacher.astype(np.longdouble) / w, -np.inf)
        x_top, u_top = x.max(1, keepdims=True), u.max(1, keepdims=True)
        log_sum = np.log(np.exp(x - x_top).sum(1, keepdims=True))
        log_p = u - u_top - np.log(np.exp(u - u_top).sum(1, keepdims=True))
        log_q = np.take_along_axis(x, np.where(has, ids, 0), 1) - x_top - log_sum
        p = np.exp(log_p)
        loss = w * w * np.where(p > 0, p * (log_p - log_q), 0).sum(1)
    return loss, (x_top + log_sum)[:, 0], p.astype(np.float64)


def loss_off(loss, temperature):
    """In 32 bits the divergence is off by some 16 U = 2^-20: 4 U (2^-22) of each of two exponentials, their sums' and logarithm's roundings, and 3 U of
    the mean argument, which is around 1.  That counts T^2 times, 2^-16 at T = 4; above, a divergence below 1/16 is taken in 64 bits, off by a few 2^-52, and a
    larger one is off by 16 of 2^-20 of itself."""
    return 2.0 ** -16 * np.maximum(1, np.abs(loss.astype(np.float64))) + 2.0 ** -49 * temperature ** 2


# a row's entries are all its classes: 8 and 16 threads to a row, a warp, a block
COVERED = [(41, 10), (5, 2), (9, 16), (19, 32), (7, 60), (6, 128), (5, 700), (3, 1024)]


@gpu
@pytest.mark.parametrize("temperature", [1e-6, 0.01, 1.0, 4.0, 4.001, 20.0, 100.0, 1e3, 1e4, 1e6])
@pytest.mark.parametrize("m,n", COVERED)
def test_loss_of_all_classes_at_any_temperature(m, n, temperature):
    rng = np.random.default_rng(n)
    for offset in (0, 1000, -70000):
        z = (rng.normal(0, 2, (m, n)) + offset).astype(np.float32)
        ids = np.argsort(rng.uniform(0, 1, (m, n)), 1)
        near = rng.choice([0.0, 0.01, 2.0], (m, 1))  # the teacher's answer itself, one near it, another one
        teacher = (np.take_along_axis(z, ids, 1) + near * rng.normal(0, 1, (m, n)) - offset / 3).astype(np.float32)
        want, want_lse, p = exact(z, ids, teacher, temperature)
        loss, lse = T.distill(dev(z), dev(ids), dev(teacher), temperature)
        within(loss.numpy(), want.astype(np.float64), loss_off(want, temperature), "loss")
        # lse = top / T + log(sum), three roundings, and 2^-20 of the sum as above
        within(lse.numpy(), want_lse.astype(np.float64), U * (3 * np.abs(want_lse.astype(np.float64)) + 16 + 3 * np.log(n)), "lse")
        if temperature >= 0.01:
            grad = T.distill_grad(dev(z), dev(ids), dev(teacher), lse, temperature)
            want, off = distill_grad64(z, ids, p, lse.numpy(), np.ones(m), temperature)
            # q is 0 below 2^-126, the smallest that ex2.approx.ftz gives: off by less than that times T
            within(grad.numpy(), want, off + temperature * 2.0 ** -126, "dlogits")


# rows of which a mask leaves `left` classes, all of them entries: a warp, a block, two and four blocks to a row
MASKED = [(3, 1000, 40), (2400, 1030, 9), (4, 6001, 300), (50, 30000, 20), (2, 32003, 1000)]


@gpu
@pytest.mark.parametrize("mask", [-np.inf, np.finfo(np.float32).min, -1e9])
@pytest.mark.parametrize("temperature", [2.0, 20.0, 1e3])
@pytest.mark.parametrize("m,n,left", MASKED)
def test_loss_of_masked_classes(m, n, left, temperature, mask):
    rng = np.random.default_rng(n + left)
    z = np.full((m, n), mask, np.float32)
    ids = np.stack([rng.choice(n, left, False) for _ in range(m)])
    some = rng.normal(0, 2, (m, left)).astype(np.float32)
    np.put_along_axis(z, ids, some, 1)
    teacher = (some + rng.choice([0.0, 0.01, 2.0], (m, 1)) * rng.normal(0, 1, (m, left))).astype(np.float32)
    ids[::3, left // 2] = -1  # one of the classes is none of the row's entries
    loss, lse = T.distill(dev(z), dev(ids), dev(teacher), temperature)
    want, want_lse, p = exact(z, ids, teacher, temperature)
    within(loss.numpy(), want.astype(np.float64), loss_off(want, temperature), "loss")
    within(lse.numpy(), want_lse.astype(np.float64), U * (3 * np.abs(want_lse.astype(np.float64)) + 16 + 3 * np.log(n)), "lse")


PATHS = [(9, 10, 5), (9, 100, 20), (9, 400, 50), (9, 800, 100), (9, 5000, 200), (9, 40000, 7)]  # 8 and 16 threads to a row, a warp, a block, several


@gpu
@pytest.mark.parametrize("m,n,top", PATHS)
def test_entries_masked_with_infinity(m, n, top):
    """Entries whose teacher is -infinity are none: a row of nothing else has loss 0 and a gradient of zeros, whatever its logits hold."""
    rng = np.random.default_rng(n)
    z = rng.normal(0, 2, (m, n)).astype(np.float32)
    ids = np.stack([rng.choice(n, top, False) for _ in range(m)])
    teacher = rng.normal(0, 2, (m, top)).astype(np.float32)
    teacher[0] = teacher[3] = -np.inf
    ids[3, 1:] = -1
    teacher[4, 1:] = -np.inf
    teacher[5, :2] = -np.inf
    teacher[6] = -np.inf
    z[6] = np.nan
    ids[7], teacher[7, 0] = -1, np.nan
    rows = np.array([1, 2, 4, 5, 8])
    for temperature in (2.0, 20.0):
        loss, lse = T.distill(dev(z), dev(ids), dev(teacher), temperature)
        grad = T.distill_grad(dev(z), dev(ids), dev(teacher), lse, temperature).numpy()
        loss, lse = loss.numpy(), lse.numpy()
        assert not loss[[0, 3, 6, 7]].any() and not grad[[0, 3, 6, 7]].any()
        want, _, p = exact(z[rows], ids[rows], teacher[rows], temperature)
        within(loss[rows], want.astype(np.float64), loss_off(want, temperature), "loss")
        within(grad[rows], *distill_grad64(z[rows], ids[rows], p, lse[rows], np.ones(len(rows)), temperature), "dlogits")
        some = np.where(np.isneginf(teacher), -1, ids)  # the same rows without these entries
        other, _ = T.distill(dev(z), dev(some), dev(teacher), temperature)
        assert other.numpy().tobytes() == loss.tobytes()


@gpu
@pytest.mark.parametrize("m,n,top", PATHS)
def test_no_class_left(m, n, top):
    """Logits that are all -infinity are no distribution: lse is -infinity, loss and gradient are NaN; 0 where the row has no entries."""
    rng = np.random.default_rng(n)
    z = np.full((m, n), -np.inf, np.float32)
    z[1] = 0
    ids = np.stack([rng.choice(n, top, False) for _ in range(m)])
    ids[2] = -1
    for temperature in (1e-3, 2.0, 20.0):
        loss, lse = T.distill(dev(z), dev(ids), dev(rng.normal(0, 2, (m, top)).astype(np.float32)), temperature)
        grad = T.distill_grad(dev(z), dev(ids), dev(np.zeros((m, top), np.float32)), lse, temperature).numpy()
        loss = loss.numpy()
        assert np.isneginf(np.delete(lse.numpy(), 1)).all() and np.isfinite(loss[1]) and np.isfinite(grad[1]).all()
        assert loss[2] == 0 and not grad[2].any()
        assert np.isnan(loss[[0, *range(3, m)]]).all() and np.isnan(grad[[0, *range(3, m)]]).all()


@gpu
@pytest.mark.parametrize("order", ["first", "last", "rising", "falling"])
@pytest.mark.parametrize("m,n", [(1, 2 ** 27), (700, 2 ** 17), (3, 2 ** 22 + 3)])
def test_sums_of_long_rows(m, n, order):
    """lse does not depend on how many classes a row has, nor on where its likeliest one stands."""
    import torch

    z = torch.full((n,), -1.2345, device="cuda")
    if order in ("rising", "falling"):
        z = torch.linspace(-30, 0, n, device="cuda")
    if order == "falling":
        z = z.flip(0)
    if order in ("first", "last"):
        z[0 if order == "first" else -1] = 0
    # in pieces: a sum of 2^27 doubles, as torch adds them up, is off by less than 2^-40
    want = torch.logsumexp(torch.stack([torch.logsumexp(p.double(), 0) for p in z.split(2 ** 22)]), 0).item()
    rows = z.expand(m, n).contiguous()
    lse = torch.empty(m, device="cuda")
    torch.cuda.synchronize()
    L.check(L.lib.ct_distill(rows.data_ptr(), None, None, m, n, 0, 1.0, None, lse.data_ptr()))
    T.check_async()
    # an exponential 4 U, its argument's 3 U of up to 2 in the mean, 16 terms 6 U, four moves and eleven joins of 4 U and two roundings each; lse three roundings
    off = U * (4 + 6 + 6 + 15 * 6 + 3 * abs(want))
    within(lse.cpu().numpy(), np.full(m, want), off, "lse")


@gpu
@pytest.mark.parametrize("m,n,top", [(1479, 3001, 5), (1480, 3001, 5), (1480, 6000, 128), (1480, 6001, 9), (2959, 7001, 20), (2960, 7001, 20), (2960, 12000, 3),
                                     (2960, 12001, 3), (2960, 7000, 129)])
def test_rows_where_warps_and_blocks_meet(m, n, top):
    z, ids, teacher, dloss = distill_inputs(m, n, top, 4)
    loss, lse = T.distill(dev(z), dev(ids), dev(teacher), 2.0)
    p, want_lse, want, off_lse, off = distill64(z, ids, teacher, 2.0)
    within(lse.numpy(), want_lse, off_lse, "lse")
    within(loss.numpy(), want, off, "loss")
    got = T.distill_grad(dev(z), dev(ids), dev(teacher), lse, 2.0, dev(dloss))
    within(got.numpy(), *distill_grad64(z, ids, p, lse.numpy(), dloss, 2.0), "dlogits")
