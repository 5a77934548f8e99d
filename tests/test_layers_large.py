"""Layer norm, the gated dense layer and the cross entropy of a dense layer on matrices of more than 2^31 values, whose last rows and columns lie
beyond what 32 bits count.  Checked there, against 64 bits on the device; bounds as in test_layers_calls (by the largest value)."""
import math

import pytest

import camel_b200._lib as L
from camel_b200 import tensor as T

gpu = pytest.mark.gpu
EDGE = 40  # rows or columns that are looked at, at both ends


@pytest.fixture
def torch():
    import torch

    T.sync()
    yield torch
    T.sync()
    torch.cuda.empty_cache()


def normal(torch, seed, *shape, std=1.0):
    out = torch.empty(*shape, device="cuda")
    return out.normal_(0.0, std, generator=torch.Generator(device="cuda").manual_seed(seed))


def near(got, want, off):
    want = want.double()
    assert ((got.double() - want).abs().max() <= off * want.abs().max()).item()


def ends(count):
    return list(range(EDGE)) + list(range(count - EDGE, count))


@gpu
@pytest.mark.parametrize("rows,cols", [(2200001, 1000), (3000000, 785), (270000, 8193), (60000, 40000)])
def test_layer_norm(torch, rows, cols):
    x, dy, gamma = normal(torch, 1, rows, cols), normal(torch, 2, rows, cols), normal(torch, 3, cols)
    out, dx, dg, db = torch.empty_like(x), torch.empty_like(x), torch.empty(cols, device="cuda"), torch.empty(cols, device="cuda")
    torch.cuda.synchronize()
    L.check(L.lib.ct_layer_norm(x.data_ptr(), gamma.data_ptr(), None, rows, cols, 1e-5, out.data_ptr()))
    L.check(L.lib.ct_layer_norm_grad(x.data_ptr(), gamma.data_ptr(), dy.data_ptr(), rows, cols, 1e-5, dx.data_ptr(), dg.data_ptr(), db.data_ptr()))
    T.check_async()
    r = ends(rows)
    d = x[r].double()
    d -= d.mean(1, keepdim=True)
    rstd = 1 / (d.square().mean(1, keepdim=True) + 1e-5).sqrt()
    h, g = d * rstd, dy[r].double() * gamma.double()
    near(out[r], h * gamma.double(), 1e-6)
    near(dx[r], rstd * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True)), 2e-6)
    near(db, sum(part.double().sum(0) for part in dy.split(1 << 16)), 1e-5)
    del out, dx
    near(dg, sum((b.double() * (a.double() - a.double().mean(1, keepdim=True)) / (a.double().var(1, correction=0, keepdim=True) + 1e-5).sqrt()).sum(0)
                 for a, b in zip(x.split(1 << 16), dy.split(1 << 16))), 1e-5)


def silu(z):
    s = z.sigmoid()
    return z * s, s * (1 + z * (1 - s))


@gpu
@pytest.mark.parametrize("m,k,n", [(2, 60000, 40000), (20, 60000, 40000), (200, 60000, 36000), (70000, 8, 32800)])
def test_dense_gated(torch, m, k, n):
    x, wg, wu = normal(torch, 1, m, k), normal(torch, 2, k, n, std=1 / math.sqrt(k)), normal(torch, 3, k, n, std=1 / math.sqrt(k))
    out, g, u = (torch.empty(m, n, device="cuda") for _ in range(3))
    torch.cuda.synchronize()
    L.check(L.lib.ct_dense_gated(x.data_ptr(), wg.data_ptr(), None, wu.data_ptr(), None, m, k, n, L.GATE_SILU, out.data_ptr(), g.data_ptr(), u.data_ptr()))
    T.check_async()
    r, c = (ends(m) if m > 2 * EDGE else list(range(m))), ends(n)
    a, b = x[r].double() @ wg[:, c].double(), x[r].double() @ wu[:, c].double()
    near(g[r][:, c], a, 1e-5)
    near(u[r][:, c], b, 1e-5)
    near(out[r][:, c], silu(a)[0] * b, 1e-5)


@gpu
@pytest.mark.parametrize("m,k,n", [(2, 60000, 40000), (20, 60000, 40000), (70000, 8, 32800)])
def test_dense_gated_grad(torch, m, k, n):
    x, wg, wu = normal(torch, 1, m, k), normal(torch, 2, k, n, std=1 / math.sqrt(k)), normal(torch, 3, k, n, std=1 / math.sqrt(k))
    g, u, dout = normal(torch, 4, m, n), normal(torch, 5, m, n), normal(torch, 6, m, n)
    dx, dwg, dwu, dbg, dbu = torch.empty_like(x), torch.empty_like(wg), torch.empty_like(wu), torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
    torch.cuda.synchronize()
    p = lambda a: a.data_ptr()  # noqa: E731
    L.check(L.lib.ct_dense_gated_grad(p(x), p(wg), p(wu), p(g), p(u), p(dout), m, k, n, L.GATE_SILU, p(dx), p(dwg), p(dwu), p(dbg), p(dbu)))
    T.check_async()
    r, c, j = (ends(m) if m > 2 * EDGE else list(range(m))), ends(n), (ends(k) if k > 2 * EDGE else list(range(k)))
    value, slope = silu(g[:, c].double())
    du, dg = dout[:, c].double() * value, dout[:, c].double() * u[:, c].double() * slope
    near(dwg[:, c], x.double().T @ dg, 2e-5)
    near(dwu[:, c], x.double().T @ du, 2e-5)
    near(dbg[c], dg.sum(0), 2e-5)
    near(dbu[c], du.sum(0), 2e-5)
    value, slope = silu(g[r].double())
    du, dg = dout[r].double() * value, dout[r].double() * u[r].double() * slope
    near(dx[r][:, j], dg @ wg[j].double().T + du @ wu[j].double().T, 2e-5)


@gpu
@pytest.mark.parametrize("m", [2, 20, 200])
def test_cross_entropy(torch, m):
    k, n = 8192, 300001
    x, w = normal(torch, 1, m, k), normal(torch, 2, k, n, std=1 / math.sqrt(k))
    t = torch.randint(n, (m,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    t[0], t[1] = n - 1, -1
    loss, lse, dx, dw, db = torch.empty(m, device="cuda"), torch.empty(m, device="cuda"), torch.empty_like(x), torch.empty_like(w), torch.empty(n, device="cuda")
    torch.cuda.synchronize()
    p = lambda a: a.data_ptr()  # noqa: E731
    L.check(L.lib.ct_dense_cross_entropy(p(x), p(w), None, p(t), m, k, n, p(loss), p(lse)))
    L.check(L.lib.ct_dense_cross_entropy_grad(p(x), p(w), None, p(t), p(lse), None, m, k, n, p(dx), p(dw), p(db)))
    T.check_async()
    z = torch.cat([x.double() @ part.double() for part in w.split(1 << 14, 1)], 1)
    want = torch.logsumexp(z, 1)
    assert ((lse.double() - want).abs().max() <= 1e-5).item()
    has = t >= 0
    assert ((loss.double() - torch.where(has, want - z.gather(1, t.clamp_min(0)[:, None])[:, 0], 0.0)).abs().max() <= 2e-5).item()
    d = (z - lse.double()[:, None]).exp()
    d.scatter_add_(1, t.clamp_min(0)[:, None], -torch.ones(m, 1, device="cuda", dtype=torch.float64))
    d *= has[:, None]
    c, j = ends(n), ends(k)
    near(dw[:, c], x.double().T @ d[:, c], 2e-5)
    near(db, d.sum(0), 2e-5)
    near(dx[:, j], d @ w[j].double().T, 2e-5)
