"""Layer norm, the gated dense layer and the cross entropy of a dense layer, with their gradients: the calls that a network
trained over a large vocabulary makes, measured against their plain forms.

Every case goes through the C ABI (include/camel_tensor_b200.h) on device buffers that the program owns.  Sizes are those of the
benchmark's own data sets (60000 x 785 x 10, 1537 x 771 x 2050) and generic ones; `draw` spreads over the same ranges.
"""
import math

import torch

own = False

# ---- the cases --------------------------------------------------------------------------------------


def listed():
    return [
        # one token on its way through a network that answers: latency alone
        dict(name="layer_norm_1", kind="norm", rows=1, cols=1024),
        # the activations of a large training batch
        dict(name="layer_norm_16384", kind="norm", rows=16384, cols=4096),
        # an image data set with its bias column: rows that no vector access divides
        dict(name="layer_norm_grad_785", kind="norm_grad", rows=60000, cols=785),
        # the same large batch on the way back
        dict(name="layer_norm_grad_16384", kind="norm_grad", rows=16384, cols=4096),
        # one token through the gated layer: the weights are read once
        dict(name="gated_1", kind="gated", m=1, k=1024, n=4096, gate="silu", bias=True, keep=False),
        # a training batch, with what the gradient needs kept
        dict(name="gated_8192", kind="gated", m=8192, k=2048, n=5504, gate="silu", bias=False, keep=True),
        # sizes that fit no tile, with biases
        dict(name="gated_grad_ragged", kind="gated_grad", m=1537, k=771, n=2050, gate="gelu", bias=True),
        # the training batch on the way back
        dict(name="gated_grad_8192", kind="gated_grad", m=8192, k=2048, n=5504, gate="silu", bias=False),
        # the loss of a short evaluation batch over a vocabulary that no tile divides
        dict(name="cross_entropy_64", kind="ce", m=64, k=1024, n=32003, bias=True),
        # a training batch over a large vocabulary
        dict(name="cross_entropy_8192", kind="ce", m=8192, k=1024, n=131072, bias=False),
        # softmax regression on the image data set: few classes, many rows
        dict(name="cross_entropy_grad_60000", kind="ce_grad", m=60000, k=785, n=10, bias=True),
        # a training batch over an odd vocabulary on the way back
        dict(name="cross_entropy_grad_4096", kind="ce_grad", m=4096, k=1024, n=50257, bias=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


GATES = ("sigmoid", "relu", "silu", "gelu")


def draw(rng):
    kind = rng.choice(["norm", "norm_grad", "gated", "gated_grad", "ce", "ce_grad"])
    if kind in ("norm", "norm_grad"):
        cols = _log_int(rng, 16, 16384)
        return dict(kind=kind, rows=_log_int(rng, 1, min(100000, (1 << 26) // cols)), cols=cols)
    if kind in ("gated", "gated_grad"):
        return dict(kind=kind, m=_log_int(rng, 1, 8192), k=_log_int(rng, 64, 2048), n=_log_int(rng, 64, 5504), gate=rng.choice(GATES),
                    bias=rng.random() < 0.5, **(dict(keep=rng.random() < 0.5) if kind == "gated" else {}))
    m, k = _log_int(rng, 1, 8192), _log_int(rng, 64, 1024)
    return dict(kind=kind, m=m, k=k, n=_log_int(rng, 10, 131072 if kind == "ce" else 50257 * 4096 // max(m, 4096)), bias=rng.random() < 0.5)


# ---- inputs -----------------------------------------------------------------------------------------

EPS = 1e-5


def _normal(g, std, *shape):
    return torch.randn(*shape, device="cuda", generator=g) * std


def _out(*shape):
    return torch.empty(*shape, device="cuda")


def _logsumexp64(x, w, b):
    """Of the logits, as the forward pass leaves it: rounded to 32 bits."""
    w, out = w.double(), _out(x.shape[0])
    step = max(1, (1 << 27) // w.shape[1])
    for i in range(0, x.shape[0], step):
        z = x[i:i + step].double() @ w
        out[i:i + step] = torch.logsumexp(z if b is None else z + b.double(), 1).float()
    return out


def _inputs(case, seed):
    """The tensors a program holds, from the seed alone."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind = case["kind"]
    if kind in ("norm", "norm_grad"):
        r, c = case["rows"], case["cols"]
        # activations: rows of different means and widths
        s = dict(x=_normal(g, 1.0, r, c) * (0.5 + torch.rand(r, 1, device="cuda", generator=g)) + _normal(g, 1.0, r, 1),
                 gamma=1.0 + _normal(g, 0.1, c), beta=_normal(g, 0.1, c))
        if kind == "norm_grad":
            s["dout"] = _normal(g, 1.0 / r, r, c)
        return s
    if kind in ("gated", "gated_grad"):
        m, k, n = case["m"], case["k"], case["n"]
        s = dict(x=_normal(g, 1.0, m, k), wg=_normal(g, 1.0 / math.sqrt(k), k, n), wu=_normal(g, 1.0 / math.sqrt(k), k, n))
        if kind == "gated":
            s.update(bg=_normal(g, 0.1, n) if case["bias"] else None, bu=_normal(g, 0.1, n) if case["bias"] else None)
        else:
            s.update(gate_pre=_normal(g, 1.0, m, n), up_pre=_normal(g, 1.0, m, n), dout=_normal(g, 1.0 / m, m, n))
        return s
    m, k, n = case["m"], case["k"], case["n"]
    s = dict(x=_normal(g, 1.0, m, k), w=_normal(g, 2.0 / math.sqrt(k), k, n), b=_normal(g, 0.5, n) if case["bias"] else None)
    t = torch.randint(n, (m,), device="cuda", generator=g)
    s["targets"] = torch.where(torch.rand(m, device="cuda", generator=g) < 0.05, torch.full_like(t, -1), t)  # padding has no target
    if kind == "ce_grad":
        s["lse"] = _logsumexp64(s["x"], s["w"], s["b"])
        s["dloss"] = (0.5 + torch.rand(m, device="cuda", generator=g)) / m
    return s


def prepare(case, seed):
    s, kind = _inputs(case, seed), case["kind"]
    s["case"] = case
    if kind == "norm":
        s["out"] = _out(case["rows"], case["cols"])
    elif kind == "norm_grad":
        s.update(dx=_out(case["rows"], case["cols"]), dgamma=_out(case["cols"]), dbeta=_out(case["cols"]))
    elif kind == "gated":
        s["out"] = _out(case["m"], case["n"])
        s.update(keep_gate=_out(case["m"], case["n"]) if case["keep"] else None, keep_up=_out(case["m"], case["n"]) if case["keep"] else None)
    elif kind == "gated_grad":
        m, k, n = case["m"], case["k"], case["n"]
        s.update(dx=_out(m, k), dwg=_out(k, n), dwu=_out(k, n), dbg=_out(n) if case["bias"] else None, dbu=_out(n) if case["bias"] else None)
    elif kind == "ce":
        s.update(loss=_out(case["m"]), lse=_out(case["m"]))
    else:
        m, k, n = case["m"], case["k"], case["n"]
        s.update(dx=_out(m, k), dw=_out(k, n), db=_out(n) if case["bias"] else None)
    return s


# ---- one pass ---------------------------------------------------------------------------------------


def run(s):
    return _own(s) if own else _plain(s)


def _own(s):
    from camel_b200 import _lib as L

    lib, case = L.lib, s["case"]
    kind = case["kind"]
    p = lambda key: None if s[key] is None else s[key].data_ptr()  # noqa: E731
    if kind == "norm":
        L.check(lib.ct_layer_norm(p("x"), p("gamma"), p("beta"), case["rows"], case["cols"], EPS, p("out")))
        return s["out"]
    if kind == "norm_grad":
        L.check(lib.ct_layer_norm_grad(p("x"), p("gamma"), p("dout"), case["rows"], case["cols"], EPS, p("dx"), p("dgamma"), p("dbeta")))
        return dict(dx=s["dx"], dgamma=s["dgamma"], dbeta=s["dbeta"])
    m, k, n = case["m"], case["k"], case["n"]
    if kind == "gated":
        gate = dict(sigmoid=L.GATE_SIGMOID, relu=L.GATE_RELU, silu=L.GATE_SILU, gelu=L.GATE_GELU)[case["gate"]]
        L.check(lib.ct_dense_gated(p("x"), p("wg"), p("bg"), p("wu"), p("bu"), m, k, n, gate, p("out"), p("keep_gate"), p("keep_up")))
        return dict(out=s["out"], gate=s["keep_gate"], up=s["keep_up"]) if case["keep"] else s["out"]
    if kind == "gated_grad":
        gate = dict(sigmoid=L.GATE_SIGMOID, relu=L.GATE_RELU, silu=L.GATE_SILU, gelu=L.GATE_GELU)[case["gate"]]
        L.check(lib.ct_dense_gated_grad(p("x"), p("wg"), p("wu"), p("gate_pre"), p("up_pre"), p("dout"), m, k, n, gate, p("dx"), p("dwg"),
                                        p("dwu"), p("dbg"), p("dbu")))
        grads = dict(dx=s["dx"], dwg=s["dwg"], dwu=s["dwu"])
        return dict(grads, dbg=s["dbg"], dbu=s["dbu"]) if case["bias"] else grads
    if kind == "ce":
        L.check(lib.ct_dense_cross_entropy(p("x"), p("w"), p("b"), p("targets"), m, k, n, p("loss"), p("lse")))
        return dict(loss=s["loss"], lse=s["lse"])
    L.check(lib.ct_dense_cross_entropy_grad(p("x"), p("w"), p("b"), p("targets"), p("lse"), p("dloss"), m, k, n, p("dx"), p("dw"), p("db")))
    return dict(dx=s["dx"], dw=s["dw"], db=s["db"]) if case["bias"] else dict(dx=s["dx"], dw=s["dw"])


# The plain forms, in 32 bits.


def _activation(gate, g):
    """(a(g), a'(g))"""
    if gate == "relu":
        on = (g > 0).to(g.dtype)
        return g * on, on
    if gate == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * (torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi)))
    sig = 1.0 / (1.0 + torch.exp(-g))
    if gate == "sigmoid":
        return sig, sig * (1.0 - sig)
    return g * sig, sig * (1.0 + g * (1.0 - sig))


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind in ("norm", "norm_grad"):
        x = s["x"]
        d = x - x.mean(1, keepdim=True)
        rstd = 1.0 / torch.sqrt((d * d).mean(1, keepdim=True) + EPS)
        xh = d * rstd
        if kind == "norm":
            return xh * s["gamma"] + s["beta"]
        g = s["dout"] * s["gamma"]
        dx = rstd * (g - g.mean(1, keepdim=True) - xh * (g * xh).mean(1, keepdim=True))
        return dict(dx=dx, dgamma=(s["dout"] * xh).sum(0), dbeta=s["dout"].sum(0))
    if kind == "gated":
        g, u = s["x"] @ s["wg"], s["x"] @ s["wu"]
        if case["bias"]:
            g, u = g + s["bg"], u + s["bu"]
        out = _activation(case["gate"], g)[0] * u
        return dict(out=out, gate=g, up=u) if case["keep"] else out
    if kind == "gated_grad":
        a, slope = _activation(case["gate"], s["gate_pre"])
        dg, du = s["dout"] * s["up_pre"] * slope, s["dout"] * a
        grads = dict(dx=dg @ s["wg"].T + du @ s["wu"].T, dwg=s["x"].T @ dg, dwu=s["x"].T @ du)
        return dict(grads, dbg=dg.sum(0), dbu=du.sum(0)) if case["bias"] else grads
    z = s["x"] @ s["w"]
    if case["bias"]:
        z = z + s["b"]
    has = s["targets"] >= 0
    at = torch.where(has, s["targets"], torch.zeros_like(s["targets"]))[:, None]
    if kind == "ce":
        top = z.max(1, keepdim=True).values
        lse = (top + torch.log(torch.exp(z - top).sum(1, keepdim=True)))[:, 0]
        return dict(loss=torch.where(has, lse - z.gather(1, at)[:, 0], torch.zeros_like(lse)), lse=lse)
    scale = torch.where(has, s["dloss"], torch.zeros_like(s["dloss"]))[:, None]
    d = torch.exp(z - s["lse"][:, None]) * scale
    d.scatter_add_(1, at, -scale)
    grads = dict(dx=d @ s["w"].T, dw=s["x"].T @ d)
    return dict(grads, db=d.sum(0)) if case["bias"] else grads


# ---- what a pass cannot do without ------------------------------------------------------------------


def work(case):
    kind = case["kind"]
    if kind in ("norm", "norm_grad"):
        r, c = case["rows"], case["cols"]
        return dict(bytes=4 * (2 * r * c + 2 * c), flops=8 * r * c) if kind == "norm" else dict(bytes=4 * (3 * r * c + 3 * c), flops=16 * r * c)
    m, k, n = case["m"], case["k"], case["n"]
    if kind == "gated":
        return dict(bytes=4 * (m * k + 2 * k * n + m * n * (3 if case["keep"] else 1) + (2 * n if case["bias"] else 0)), flops=4 * m * k * n)
    if kind == "gated_grad":
        return dict(bytes=4 * (2 * m * k + 4 * k * n + 3 * m * n + (2 * n if case["bias"] else 0)), flops=8 * m * k * n)
    b = n if case["bias"] else 0
    if kind == "ce":
        return dict(bytes=4 * (m * k + k * n + b + 2 * m) + 8 * m, flops=2 * m * k * n)
    return dict(bytes=4 * (2 * m * k + 2 * k * n + 2 * b + 2 * m) + 8 * m, flops=6 * m * k * n)  # the logits again, and two products


# ---- the same in 64 bits, from the definitions -------------------------------------------------------


def _pieces(rows, values_per_row):
    step = max(1, (1 << 27) // values_per_row)
    return [(i, min(rows, i + step)) for i in range(0, rows, step)]


def _gate64(gate, g):
    return dict(sigmoid=torch.special.expit, relu=lambda v: v.clamp_min(0.0), silu=lambda v: v * torch.special.expit(v),
                gelu=lambda v: v * torch.special.ndtr(v))[gate](g)


def _slope64(gate, g):
    if gate == "relu":
        return torch.heaviside(g, torch.zeros((), dtype=g.dtype, device=g.device))
    if gate == "gelu":
        return torch.special.ndtr(g) + g * torch.exp(-g.square() / 2) / math.sqrt(2 * math.pi)
    e = torch.special.expit(g)
    return e * torch.special.expit(-g) if gate == "sigmoid" else e + g * e * torch.special.expit(-g)


def exact(case, seed):
    s, kind = _inputs(case, seed), case["kind"]
    v = {key: t.double() if t is not None and t.is_floating_point() else t for key, t in s.items()}
    if kind in ("norm", "norm_grad"):
        var, mean = torch.var_mean(v["x"], 1, correction=0, keepdim=True)
        xh = (v["x"] - mean) / (var + EPS).sqrt()
        if kind == "norm":
            return torch.addcmul(v["beta"], xh, v["gamma"])
        g = v["gamma"] * v["dout"]
        cols = case["cols"]
        dx = (g - (g.sum(1, keepdim=True) + xh * (g * xh).sum(1, keepdim=True)) / cols) / (var + EPS).sqrt()
        return dict(dx=dx, dgamma=torch.einsum("rc,rc->c", v["dout"], xh), dbeta=v["dout"].sum(0))
    if kind == "gated":
        g = v["x"] @ v["wg"] + (v["bg"] if case["bias"] else 0.0)
        u = v["x"] @ v["wu"] + (v["bu"] if case["bias"] else 0.0)
        out = _gate64(case["gate"], g) * u
        return dict(out=out, gate=g, up=u) if case["keep"] else out
    if kind == "gated_grad":
        du = _gate64(case["gate"], v["gate_pre"]) * v["dout"]
        dg = _slope64(case["gate"], v["gate_pre"]) * v["up_pre"] * v["dout"]
        both = torch.cat([dg, du], 1)
        dw = v["x"].mT @ both
        n = case["n"]
        grads = dict(dx=both @ torch.cat([v["wg"], v["wu"]], 1).mT, dwg=dw[:, :n], dwu=dw[:, n:])
        return dict(grads, dbg=dg.sum(0), dbu=du.sum(0)) if case["bias"] else grads
    m, n = case["m"], case["n"]
    targets = s["targets"]
    if kind == "ce":
        loss, lse = torch.zeros(m, dtype=torch.float64, device="cuda"), torch.empty(m, dtype=torch.float64, device="cuda")
        for i, j in _pieces(m, n):
            z = v["x"][i:j] @ v["w"] + (v["b"] if case["bias"] else 0.0)
            lse[i:j] = torch.logsumexp(z, 1)
            rows = torch.nonzero(targets[i:j] >= 0)[:, 0]
            loss[i + rows] = lse[i + rows] - z[rows, targets[i + rows]]
        return dict(loss=loss, lse=lse)
    dx = torch.empty_like(v["x"])
    dw, db = torch.zeros_like(v["w"]), torch.zeros(n, dtype=torch.float64, device="cuda")
    for i, j in _pieces(m, n):
        d = (v["x"][i:j] @ v["w"] + (v["b"] if case["bias"] else 0.0) - v["lse"][i:j, None]).exp()
        rows = torch.nonzero(targets[i:j] >= 0)[:, 0]
        d[rows, targets[i + rows]] -= 1.0
        d *= torch.where(targets[i:j] >= 0, v["dloss"][i:j], 0.0)[:, None]
        dx[i:j] = d @ v["w"].mT
        dw += v["x"][i:j].mT @ d
        db += d.sum(0)
    return dict(dx=dx, dw=dw, db=db) if case["bias"] else dict(dx=dx, dw=dw)
