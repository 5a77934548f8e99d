"""Embedding lookup, the gated scan and distillation on arrays of more than 2^31 values, whose last ones lie beyond what 32 bits count.  Checked there, against
64 bits on the device, by the largest value."""
import pytest

import camel_b200._lib as L
from camel_b200 import tensor as T
from test_layers_large import normal, near, torch  # noqa: F401

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("n,k", [(1100000, 2048), (1100000, 2050), (30000001, 75)])
def test_embedding(torch, n, k):  # noqa: F811
    m = 3000
    table, dout = normal(torch, 1, n, k), normal(torch, 2, m, k)
    ids = torch.randint(n, (m,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    ids[:4] = torch.tensor([n - 1, 0, n, n - 1], device="cuda")
    ids[100:200] = n - 2
    out, grad = torch.empty(m, k, device="cuda"), torch.full((n, k), 7.0, device="cuda")
    torch.cuda.synchronize()
    L.check(L.lib.ct_embedding(table.data_ptr(), ids.data_ptr(), m, n, k, 1.5, out.data_ptr()))
    L.check(L.lib.ct_embedding_grad(ids.data_ptr(), dout.data_ptr(), m, n, k, 1.5, grad.data_ptr()))
    T.check_async()
    has = ids < n
    assert torch.equal(out[has], table[ids[has]] * 1.5) and not out[~has].any()
    rows, at = torch.unique(ids[has], return_inverse=True)
    want = torch.zeros(len(rows), k, dtype=torch.float64, device="cuda").index_add_(0, at, dout[has].double() * 1.5)
    near(grad[rows], want, 1e-7)
    del table
    grad[rows] = 0.0
    assert not any(part.any().item() for part in grad.split(1 << 18))


@gpu
def test_embedding_of_many_tokens(torch):  # noqa: F811
    m, n, k = 8500000, 1000, 256
    ids = torch.randint(-1, n, (m,), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    table, dout = normal(torch, 1, n, k), normal(torch, 2, m, k)
    out, grad = torch.empty(m, k, device="cuda"), torch.empty(n, k, device="cuda")
    torch.cuda.synchronize()
    L.check(L.lib.ct_embedding(table.data_ptr(), ids.data_ptr(), m, n, k, 1.0, out.data_ptr()))
    L.check(L.lib.ct_embedding_grad(ids.data_ptr(), dout.data_ptr(), m, n, k, 1.0, grad.data_ptr()))
    T.check_async()
    end = slice(m - 1000, m)
    assert torch.equal(out[end], torch.where(ids[end, None] >= 0, table[ids[end].clamp_min(0)], 0.0))
    want = torch.zeros(n, k, dtype=torch.float64, device="cuda")
    for i in range(0, m, 1 << 19):
        has = ids[i:i + (1 << 19)] >= 0
        want.index_add_(0, ids[i:i + (1 << 19)][has], dout[i:i + (1 << 19)][has].double())
    near(grad, want, 1e-7)


def scan(torch, gate, value, state, out, dout, dstate):  # noqa: F811
    """h and the gradients in 64 bits of a few chains and steps; out: what the forward call left."""
    a, rest = torch.sigmoid(gate.double()), torch.sigmoid(-gate.double())
    h, now = torch.empty_like(a), state
    for t in range(a.shape[1]):
        now = a[:, t] * now + rest[:, t] * value[:, t].double()
        h[:, t] = now
    g, carry = torch.empty_like(a), dstate
    for t in reversed(range(a.shape[1])):
        g[:, t] = dout[:, t].double() + carry
        carry = a[:, t] * g[:, t]
    before = torch.cat([state[:, None], out[:, :-1].double()], 1)
    return h, now, g * a * rest * (before - value.double()), g * rest


@gpu
@pytest.mark.parametrize("b,t,c", [(70000, 32, 1000), (70001, 10, 3100), (1, 4300000, 512), (2, 2100001, 517), (1, 1 << 28, 9)])
def test_gated_scan(torch, b, t, c):  # noqa: F811
    """Gates below 0: 300 steps forget what was before them to 2^-300."""
    gate, value = normal(torch, 1, b, t, c), normal(torch, 2, b, t, c)
    gate.sub_(4.0)
    gate.clamp_(max=0.0)
    out, state = torch.empty_like(gate), torch.empty(b, c, device="cuda")
    torch.cuda.synchronize()
    L.check(L.lib.ct_gated_scan(gate.data_ptr(), value.data_ptr(), None, None, b, t, c, out.data_ptr(), state.data_ptr()))
    T.check_async()
    dout = normal(torch, 3, b, t, c)
    dgate, dvalue = torch.empty_like(gate), torch.empty_like(gate)
    torch.cuda.synchronize()
    L.check(L.lib.ct_gated_scan_grad(gate.data_ptr(), value.data_ptr(), None, None, out.data_ptr(), dout.data_ptr(), None, b, t, c, dgate.data_ptr(),
                                     dvalue.data_ptr(), None))
    T.check_async()
    r, steps = slice(max(0, b - 40), b), min(t, 300)
    zero = torch.zeros(len(range(*r.indices(b))), c, dtype=torch.float64, device="cuda")
    for s, skip_h, skip_g in ((slice(0, steps), 0, 100 if t > 300 else 0), (slice(t - steps, t), 100 if t > 300 else 0, 0)):
        part = [x[r, s] for x in (gate, value, out, dout)]
        h, last, dg, dv = scan(torch, part[0], part[1], zero, part[2], part[3], zero)
        keep_h, keep_g = slice(skip_h, steps), slice(0, steps - skip_g)
        near(out[r, s][:, keep_h], h[:, keep_h], 1e-5)
        lo = max(1, skip_h) if s.start else 0  # the first step's state before it is not zero in the middle of a sequence
        near(dgate[r, s][:, lo:steps - skip_g], dg[:, lo:steps - skip_g], 1e-5)
        near(dvalue[r, s][:, keep_g], dv[:, keep_g], 1e-5)
        if s.stop == t:
            near(state[r], last, 1e-5)


@gpu
@pytest.mark.parametrize("m,n", [(17000, 131072), (66000, 33001), (430000, 5001), (4300000, 501), (5, 500000003)])
def test_distill(torch, m, n):  # noqa: F811
    top = 7
    z = normal(torch, 1, m, n)
    ids = torch.randint(n, (m, top), device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    ids[:, 0] = n - 1
    teacher = normal(torch, 2, m, top)
    loss, lse = torch.empty(m, device="cuda"), torch.empty(m, device="cuda")
    torch.cuda.synchronize()
    L.check(L.lib.ct_distill(z.data_ptr(), ids.data_ptr(), teacher.data_ptr(), m, n, top, 2.0, loss.data_ptr(), lse.data_ptr()))
    grad = torch.empty_like(z)
    L.check(L.lib.ct_distill_grad(z.data_ptr(), ids.data_ptr(), teacher.data_ptr(), lse.data_ptr(), None, m, n, top, 2.0, grad.data_ptr()))
    T.check_async()
    for i in sorted({0, 1, m // 2, m - 2, m - 1}):
        q = z[i].double() / 2
        want = torch.logsumexp(q, 0)
        assert abs(lse[i].item() - want.item()) <= 1e-5 * abs(want.item())
        log_p = torch.log_softmax(teacher[i].double() / 2, 0)
        ref = 4 * (log_p.exp() * (log_p - (q[ids[i]] - want))).sum()
        assert abs(loss[i].item() - ref.item()) <= 1e-5 * abs(ref.item())
        d = 2 * torch.exp(q - lse[i].double())
        d.index_add_(0, ids[i], -2 * log_p.exp())
        near(grad[i], d, 1e-6)
