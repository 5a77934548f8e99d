"""Embedding lookup, the gated scan and distillation from a teacher's top logits, with their gradients: what a network over sequences of
tokens calls around its dense layers, measured against their plain forms.

Every case goes through the C ABI (include/camel_tensor_b200.h) on device buffers that the program owns.  Sizes are those of the
benchmark's own data sets (60000 x 10, 1537 x 771 x 2050) and generic ones; `draw` spreads over the same ranges.
"""
import math

import numpy as np
import torch

own = False

# ---- the cases --------------------------------------------------------------------------------------


def listed():
    return [
        # the token that a network answered last, on its way in again: latency alone
        dict(name="embedding_1", kind="embed", m=1, n=32003, k=1024),
        # the tokens of a large training batch
        dict(name="embedding_32768", kind="embed", m=32768, n=50257, k=2048),
        # a small batch, sizes that fit no vector access
        dict(name="embedding_grad_ragged", kind="embed_grad", m=1537, n=2050, k=771),
        # a training batch over a large vocabulary: most rows of the gradient are zeros, a few have a thousand terms
        dict(name="embedding_grad_16384", kind="embed_grad", m=16384, n=50257, k=2048),
        # one token of each of 64 sequences that are being answered: the state moves one step
        dict(name="scan_step", kind="scan", batch=64, steps=1, channels=2048, lengths=False, state=True),
        # one long document
        dict(name="scan_long", kind="scan", batch=1, steps=65536, channels=512, lengths=False, state=False),
        # a padded batch of odd sizes on the way back
        dict(name="scan_grad_ragged", kind="scan_grad", batch=7, steps=1537, channels=771, lengths=True, state=True),
        # a training batch on the way back
        dict(name="scan_grad_2048", kind="scan_grad", batch=8, steps=2048, channels=2048, lengths=False, state=False),
        # the loss of a short evaluation batch over a vocabulary that no tile divides
        dict(name="distill_64", kind="distill", m=64, n=32003, top=20, temperature=2.0),
        # a training batch over a large vocabulary
        dict(name="distill_4096", kind="distill", m=4096, n=131072, top=64, temperature=1.0),
        # a small classifier that learns an image data set from a larger one: few classes, many rows
        dict(name="distill_grad_60000", kind="distill_grad", m=60000, n=10, top=5, temperature=4.0),
        # a training batch over an odd vocabulary on the way back
        dict(name="distill_grad_4096", kind="distill_grad", m=4096, n=50257, top=64, temperature=2.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(["embed", "embed_grad", "scan", "scan_grad", "distill", "distill_grad"])
    if kind in ("embed", "embed_grad"):
        k = _log_int(rng, 16, 4096)
        return dict(kind=kind, m=_log_int(rng, 1, min(131072, (1 << (26 if kind == "embed" else 25)) // k)),
                    n=_log_int(rng, 10, min(131072, 50257 * 2048 // k)), k=k)
    if kind in ("scan", "scan_grad"):
        channels = _log_int(rng, 16, 4096)
        batch = _log_int(rng, 1, 64)
        return dict(kind=kind, batch=batch, steps=_log_int(rng, 1, min(65536, (1 << 25) // (batch * channels))), channels=channels,
                    lengths=rng.random() < 0.5, state=rng.random() < 0.5)
    m = _log_int(rng, 1, 60000)
    n = _log_int(rng, 10, min(131072, (131072 if kind == "distill" else 50257) * 4096 // m))
    return dict(kind=kind, m=m, n=n, top=_log_int(rng, 1, min(n, 128)), temperature=rng.choice([1.0, 2.0, 4.0]))


# ---- inputs -----------------------------------------------------------------------------------------


def _normal(g, std, *shape):
    return torch.randn(*shape, device="cuda", generator=g) * std


def _rand(g, *shape):
    return torch.rand(*shape, device="cuda", generator=g)


def _out(*shape):
    return torch.empty(*shape, device="cuda")


def _scale(k):
    """sqrt(k), as the library takes it: rounded to 32 bits."""
    return float(np.float32(math.sqrt(k)))


def _here(s, t):
    """Which steps belong to their sequence: behind its end nothing changes the state."""
    if s["lengths"] is None:
        return torch.ones((), dtype=torch.bool, device="cuda")
    return torch.arange(t, device="cuda")[None, :, None] < s["lengths"][:, None, None]


def _inputs(case, seed):
    """The tensors a program holds, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind = case["kind"]
    if kind in ("embed", "embed_grad"):
        m, n, k = case["m"], case["n"], case["k"]
        # words by their rank: the first is drawn as often as the second and third together, and so on; some padding
        ids = (torch.pow(float(n + 1), _rand(g, m).double()) - 1.0).long().clamp_(0, n - 1)
        s = dict(ids=torch.where(_rand(g, m) < 0.02, torch.full_like(ids, -1), ids))
        if kind == "embed":
            s["table"] = _normal(g, 1.0 / math.sqrt(k), n, k)
        else:
            s["dout"] = _normal(g, 1.0 / m, m, k)
        return s
    if kind in ("scan", "scan_grad"):
        b, t, c = case["batch"], case["steps"], case["channels"]
        # channels that forget at once beside channels that remember hundreds of steps
        s = dict(gate=_normal(g, 1.0, b, t, c) + 5.0 * _rand(g, c), value=_normal(g, 1.0, b, t, c),
                 state0=_normal(g, 0.3, b, c) if case["state"] else None,
                 lengths=(t // 2 + (_rand(g, b) * (t - t // 2 + 1)).long()).clamp_(max=t) if case["lengths"] else None)
        if kind == "scan_grad":
            s.update(dout=_normal(g, 1.0 / (b * t), b, t, c), dstate=_normal(g, 1.0 / (b * t), b, c) if case["state"] else None)
            s["out"] = _plain_scan(s)["out"]
        return s
    m, n, top = case["m"], case["n"], case["top"]
    z = _normal(g, 2.0, m, n)
    # the teacher's classes, likeliest first; the student has learned some of it; rows with fewer classes, and rows of padding
    step = (_rand(g, m) * (n // top)).long().clamp_(0, n // top - 1) + 1
    ids = ((_rand(g, m) * n).long().clamp_(0, n - 1)[:, None] + step[:, None] * torch.arange(top, device="cuda")) % n
    teacher = torch.sort(_normal(g, 2.0, m, top), 1, descending=True).values + 8.0
    z.scatter_add_(1, ids, 0.5 * teacher)
    given = torch.where(_rand(g, m) < 0.05, (_rand(g, m) * top).long(), torch.full_like(step, top))
    given = torch.where(_rand(g, m) < 0.02, torch.zeros_like(given), given)
    s = dict(logits=z, ids=torch.where(torch.arange(top, device="cuda") < given[:, None], ids, torch.full_like(ids, -1)), teacher=teacher)
    if kind == "distill_grad":
        s["lse"] = _out(m)
        for i, j in _pieces(m, n):
            s["lse"][i:j] = torch.logsumexp(z[i:j].double() / case["temperature"], 1).float()
        s["dloss"] = (0.5 + _rand(g, m)) / m
    return s


def prepare(case, seed):
    s, kind = _inputs(case, seed), case["kind"]
    s["case"] = case
    if kind == "embed":
        s["out"] = _out(case["m"], case["k"])
    elif kind == "embed_grad":
        s["dtable"] = _out(case["n"], case["k"])
    elif kind == "scan":
        s.update(out=torch.empty_like(s["value"]), state=_out(case["batch"], case["channels"]))
    elif kind == "scan_grad":
        s.update(dgate=torch.empty_like(s["value"]), dvalue=torch.empty_like(s["value"]),
                 dstate0=_out(case["batch"], case["channels"]) if case["state"] else None)
    elif kind == "distill":
        s.update(loss=_out(case["m"]), lse=_out(case["m"]))
    else:
        s["dlogits"] = torch.empty_like(s["logits"])
    return s


# ---- one pass ---------------------------------------------------------------------------------------


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from camel_b200 import _lib as L

    lib, case = L.lib, s["case"]
    kind = case["kind"]
    p = lambda key: None if s[key] is None else s[key].data_ptr()  # noqa: E731
    if kind == "embed":
        L.check(lib.ct_embedding(p("table"), p("ids"), case["m"], case["n"], case["k"], _scale(case["k"]), p("out")))
        return s["out"]
    if kind == "embed_grad":
        L.check(lib.ct_embedding_grad(p("ids"), p("dout"), case["m"], case["n"], case["k"], _scale(case["k"]), p("dtable")))
        return s["dtable"]
    if kind == "scan":
        L.check(lib.ct_gated_scan(p("gate"), p("value"), p("state0"), p("lengths"), case["batch"], case["steps"], case["channels"], p("out"),
                                  p("state")))
        return dict(out=s["out"], state=s["state"])
    if kind == "scan_grad":
        L.check(lib.ct_gated_scan_grad(p("gate"), p("value"), p("state0"), p("lengths"), p("out"), p("dout"), p("dstate"), case["batch"],
                                       case["steps"], case["channels"], p("dgate"), p("dvalue"), p("dstate0")))
        grads = dict(dgate=s["dgate"], dvalue=s["dvalue"])
        return dict(grads, dstate0=s["dstate0"]) if case["state"] else grads
    if kind == "distill":
        L.check(lib.ct_distill(p("logits"), p("ids"), p("teacher"), case["m"], case["n"], case["top"], case["temperature"], p("loss"), p("lse")))
        return dict(loss=s["loss"], lse=s["lse"])
    L.check(lib.ct_distill_grad(p("logits"), p("ids"), p("teacher"), p("lse"), p("dloss"), case["m"], case["n"], case["top"], case["temperature"],
                                p("dlogits")))
    return s["dlogits"]


# The plain forms, in 32 bits.


def _gates(x):
    """(a, 1 - a) of the gate's pre-activation, each with its own digits."""
    e = torch.exp(-x.abs())
    small, large = e / (1.0 + e), 1.0 / (1.0 + e)
    return torch.where(x >= 0, large, small), torch.where(x >= 0, small, large)


def _recur(s, h):
    """y[t] = (1 - s[t]) y[t - 1] + h[t] along axis 1, in rounds of doubled reach; of s as it is, since what 1 - s loses of a small s grows with
    every step."""
    reach = 1
    while reach < h.shape[1]:
        h2, s2 = h.clone(), s.clone()
        h2[:, reach:] += h[:, :-reach] - s[:, reach:] * h[:, :-reach]
        s2[:, reach:] += s[:, :-reach] * (1.0 - s[:, reach:])
        h, s, reach = h2, s2, 2 * reach
    return h


def _plain_scan(s):
    t = s["value"].shape[1]
    here = _here(s, t)
    a, keep = _gates(s["gate"])
    zero = torch.zeros((), device="cuda")
    a, keep = torch.where(here, a, zero + 1.0), torch.where(here, keep, zero)
    h = torch.where(here, keep * s["value"], zero)
    if s["state0"] is not None:
        h[:, 0] += a[:, 0] * s["state0"]
    h = _recur(keep, h)
    return dict(out=torch.where(here, h, zero), state=h[:, -1].clone())


def _plain_scan_grad(s):
    t = s["value"].shape[1]
    here = _here(s, t)
    a, keep = _gates(s["gate"])
    zero = torch.zeros((), device="cuda")
    a, keep = torch.where(here, a, zero + 1.0), torch.where(here, keep, zero)
    dout = torch.where(here, s["dout"], zero)
    # c[t] = a[t] (dout[t] + c[t + 1]) is what reaches step t - 1, along the reversed axis
    c = a * dout
    if s["dstate"] is not None:
        c[:, -1] += a[:, -1] * s["dstate"]
    c = _recur(keep.flip(1), c.flip(1)).flip(1)
    after = torch.cat([c[:, 1:], (torch.zeros_like(c[:, :1]) if s["dstate"] is None else s["dstate"][:, None])], 1)
    grad = dout + after
    first = torch.zeros_like(c[:, :1]) if s["state0"] is None else s["state0"][:, None]
    before = torch.cat([first, s["out"][:, :-1]], 1)
    grads = dict(dgate=torch.where(here, a * keep * grad * (before - s["value"]), zero), dvalue=torch.where(here, keep * grad, zero))
    return dict(grads, dstate0=c[:, 0].clone()) if s["case"]["state"] else grads


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "embed":
        has = s["ids"] >= 0
        rows = s["table"][torch.where(has, s["ids"], torch.zeros_like(s["ids"]))] * _scale(case["k"])
        return torch.where(has[:, None], rows, torch.zeros_like(rows))
    if kind == "embed_grad":
        has = s["ids"] >= 0
        rows = torch.where(has[:, None], s["dout"], torch.zeros_like(s["dout"]))
        return torch.zeros(case["n"], case["k"], device="cuda").index_add_(0, torch.where(has, s["ids"], torch.zeros_like(s["ids"])), rows) * _scale(case["k"])
    if kind == "scan":
        return _plain_scan(s)
    if kind == "scan_grad":
        return _plain_scan_grad(s)
    warm = case["temperature"]
    has = s["ids"] >= 0
    at = torch.where(has, s["ids"], torch.zeros_like(s["ids"]))
    u = torch.where(has, s["teacher"] / warm, torch.full_like(s["teacher"], -math.inf))
    some = has.any(1)
    u = u - torch.where(some, u.max(1).values, torch.zeros_like(u[:, 0]))[:, None]
    e = torch.exp(u)
    total = e.sum(1, keepdim=True)
    p = torch.where(has, e / total, torch.zeros_like(e))
    z = s["logits"] / warm
    if kind == "distill":
        top = z.max(1, keepdim=True).values
        lse = (top + torch.log(torch.exp(z - top).sum(1, keepdim=True)))[:, 0]
        gap = u - torch.log(total) - (z.gather(1, at) - lse[:, None])
        loss = warm * warm * torch.where(has, p * gap, torch.zeros_like(p)).sum(1)
        return dict(loss=torch.where(some, loss, torch.zeros_like(loss)), lse=lse)
    scale = torch.where(some, s["dloss"] * warm, torch.zeros_like(s["dloss"]))[:, None]
    d = torch.exp(z - s["lse"][:, None]) * scale
    return d.scatter_add_(1, at, -scale * p)


# ---- what a pass cannot do without ------------------------------------------------------------------


def _distinct(m, n):
    """Of m tokens drawn as above, how many differ."""
    v = np.arange(n, dtype=np.float64)
    return float((1.0 - (1.0 - np.log1p(1.0 / (v + 1.0)) / math.log(n + 1.0)) ** (0.98 * m)).sum())


def work(case):
    kind = case["kind"]
    if kind in ("embed", "embed_grad"):
        m, n, k = case["m"], case["n"], case["k"]
        if kind == "embed":
            return dict(bytes=4 * (_distinct(m, n) * k + m * k) + 8 * m, flops=m * k)
        return dict(bytes=4 * (m * k + n * k) + 8 * m, flops=m * k)
    if kind in ("scan", "scan_grad"):
        lanes = case["batch"] * case["channels"]
        count = lanes * case["steps"]
        here = 0.75 if case["lengths"] else 1.0  # padding is not read; it is written, as zeros
        if kind == "scan":
            return dict(bytes=4 * (count * (2 * here + 1) + lanes * (2 if case["state"] else 1)), flops=10 * count)
        return dict(bytes=4 * (count * (4 * here + 2) + lanes * (3 if case["state"] else 0)), flops=16 * count)
    m, n, top = case["m"], case["n"], case["top"]
    if kind == "distill":
        return dict(bytes=4 * (m * n + 2 * m) + 12 * m * top, flops=4 * m * n)
    return dict(bytes=4 * (2 * m * n + 2 * m) + 12 * m * top, flops=4 * m * n)


# ---- the same in 64 bits, from the definitions -------------------------------------------------------


def _pieces(rows, values_per_row):
    step = max(1, (1 << 27) // values_per_row)
    return [(i, min(rows, i + step)) for i in range(0, rows, step)]


def _exact_scan(v, steps):
    a, b = torch.sigmoid(v["gate"]), torch.sigmoid(-v["gate"]) * v["value"]
    state = torch.zeros_like(a[:, 0]) if v["state0"] is None else v["state0"].clone()
    out = torch.zeros_like(a)
    if v["lengths"] is None:
        for t in range(steps):
            torch.addcmul(b[:, t], a[:, t], state, out=state)
            out[:, t] = state
    else:
        for t in range(steps):
            on = (v["lengths"] > t).double()[:, None]
            new = a[:, t] * state + b[:, t]
            state = on * new + (1.0 - on) * state
            out[:, t] = on * new
    return dict(out=out, state=state)


def _exact_scan_grad(v, steps, with_state):
    a, rest = torch.sigmoid(v["gate"]), torch.sigmoid(-v["gate"])
    carry = torch.zeros_like(a[:, 0]) if v["dstate"] is None else v["dstate"].clone()
    g = torch.zeros_like(a)
    for t in reversed(range(steps)):
        new = v["dout"][:, t] + carry
        if v["lengths"] is None:
            g[:, t] = new
            carry = a[:, t] * new
        else:
            on = (v["lengths"] > t).double()[:, None]
            g[:, t] = on * new
            carry = on * a[:, t] * new + (1.0 - on) * carry
    before = torch.roll(v["out"], 1, 1)
    before[:, 0] = 0.0 if v["state0"] is None else v["state0"]
    grads = dict(dgate=g * a * rest * (before - v["value"]), dvalue=g * rest)
    return dict(grads, dstate0=carry) if with_state else grads


def exact(case, seed):
    s, kind = _inputs(case, seed), case["kind"]
    if kind in ("embed", "embed_grad"):
        has = torch.nonzero(s["ids"] >= 0)[:, 0]
        if kind == "embed":
            out = torch.zeros(case["m"], case["k"], dtype=torch.float64, device="cuda")
            out[has] = s["table"][s["ids"][has]].double() * _scale(case["k"])
            return out
        out = torch.zeros(case["n"], case["k"], dtype=torch.float64, device="cuda")
        return out.index_add_(0, s["ids"][has], s["dout"][has].double(), alpha=_scale(case["k"]))
    if kind in ("scan", "scan_grad"):
        v = {key: t.double() if t is not None and t.is_floating_point() else t for key, t in s.items()}
        return _exact_scan(v, case["steps"]) if kind == "scan" else _exact_scan_grad(v, case["steps"], case["state"])
    warm, m = case["temperature"], case["m"]
    rows = torch.nonzero((s["ids"] >= 0).any(1))[:, 0]
    u = torch.where(s["ids"] >= 0, s["teacher"].double() / warm, -math.inf)
    if kind == "distill":
        lse, loss = torch.empty(m, dtype=torch.float64, device="cuda"), torch.zeros(m, dtype=torch.float64, device="cuda")
        for i, j in _pieces(m, case["n"]):
            lse[i:j] = torch.logsumexp(s["logits"][i:j].double() / warm, 1)
        log_p = torch.log_softmax(u[rows], 1)
        log_q = s["logits"][rows[:, None], s["ids"][rows].clamp_min(0)].double() / warm - lse[rows, None]
        loss[rows] = warm ** 2 * torch.nan_to_num(log_p.exp() * (log_p - log_q), nan=0.0).sum(1)
        return dict(loss=loss, lse=lse)
    d = torch.zeros(s["logits"].shape, dtype=torch.float64, device="cuda")
    for i, j in _pieces(m, case["n"]):
        some = rows[(rows >= i) & (rows < j)]
        q = torch.exp(s["logits"][some].double() / warm - s["lse"][some].double()[:, None])
        q.scatter_add_(1, s["ids"][some].clamp_min(0), -torch.softmax(u[some], 1))
        d[some] = q * (warm * s["dloss"][some].double())[:, None]
    return d
