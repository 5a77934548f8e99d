"""Embedding lookup, the gated scan and distillation as programs call them: one after the other over buffers that are rewritten, recorded and
replayed, on other streams, from scratch memory that holds anything, and together as a network over sequences of tokens."""
import math

import numpy as np
import pytest

import camel_b200._lib as L
from camel_b200 import tensor as T
from test_layers import U, dev, within
from test_sequences import (SCAN, distill64, distill_grad64, distill_inputs, embedding_grad64, embedding_grad_off, embedding_inputs, lookup32, scan64,
                            scan_grad64, scan_inputs)

gpu = pytest.mark.gpu


def all_operators(seed, m=900, n=300, k=70, b=3, t=200, c=45, classes=1500, top=20):
    """Every entry point on inputs of a seed: a function that runs them and returns the outputs, and what it holds."""
    ids, table, dout = [dev(a) for a in embedding_inputs(m, n, k, seed)]
    gate, value, state0, lengths, dy, dstate = [dev(a) for a in scan_inputs(b, t, c, seed)]
    z, entries, teacher, dloss = [dev(a) for a in distill_inputs(m, classes, top, seed)]
    small = [dev(a) for a in distill_inputs(m, 40, 5, seed)]
    more_ids, _, more = [dev(a) for a in embedding_inputs(9 * m, n, 30, seed)]
    step_gate, step_value = [dev(a[:, :1]) for a in scan_inputs(b, t, c, seed)[:2]]

    def run():
        out, last = T.gated_scan(gate, value, state0, lengths)
        loss, lse = T.distill(z, entries, teacher, 2.0)
        loss2, lse2 = T.distill(*small[:3], 2.0)
        return [T.embedding(table, ids, 3.0), T.embedding_grad(ids, dout, n, 3.0), T.embedding_grad(more_ids, more, n), out, last,
                *T.gated_scan_grad(gate, value, out, dy, state0, lengths, dstate), *T.gated_scan(step_gate, step_value, last),
                loss, lse, T.distill_grad(z, entries, teacher, lse, 2.0, dloss), loss2, lse2, T.distill_grad(*small[:3], lse2, 2.0)]

    return run, (ids, table, dout, gate, value, state0, lengths, dy, dstate, z, entries, teacher, dloss, small, more_ids, more, step_gate, step_value)


def bytes_of(tensors):
    return [a.numpy().tobytes() for a in tensors]


@gpu
def test_two_recordings_replayed_on_two_streams():
    import torch

    pair = []
    for seed in (31, 32):
        run, held = all_operators(seed)
        want = bytes_of(run())
        with T.Graph() as graph:
            graph.keep = run()
        pair.append((graph, want, held))
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
        assert bytes_of(graph.keep) == want


@gpu
def test_calls_on_two_streams_at_once():
    import torch

    pair = []
    for seed in (33, 34):
        run, held = all_operators(seed)
        pair.append((run, bytes_of(run()), held, torch.cuda.Stream()))
    T.sync()
    for _ in range(5):
        got = []
        try:
            for run, _, _, s in pair:
                L.check(L.lib.ct_set_stream(s.cuda_stream))
                got.append(run())
            torch.cuda.synchronize()
        finally:
            L.check(L.lib.ct_set_stream(None))
        for outputs, (_, want, _, _) in zip(got, pair):
            assert bytes_of(outputs) == want


@gpu
def test_memory_that_holds_anything():
    """Scratch comes from a pool of freed tensors: what they held does not show."""
    run, _ = all_operators(35)
    want = bytes_of(run())
    for value in (math.nan, math.inf, -3e38):
        for size in (1 << 10, 1 << 14, 1 << 18, 1 << 21):
            held = [T.full([size], value) for _ in range(6)]
            T.sync()
            del held
        assert bytes_of(run()) == want, value


def rewritten(rng, m, n, k):
    """name -> (the float inputs of an operator, its call, its outputs)"""
    f = lambda *s: dev(rng.normal(0, 0.5, s).astype(np.float32))  # noqa: E731
    z = lambda *s: T.zeros(list(s))  # noqa: E731
    ids, entries, p = dev(rng.integers(-1, n, m)), dev(rng.integers(-1, n, (m, 5))), L.lib
    b, t, c = 3, m, k
    table, dout, dtable, rows = f(n, k), f(m, k), z(n, k), z(m, k)
    gate, value, dy, out = f(b, t, c), f(b, t, c), f(b, t, c), f(b, t, c)
    h, dgate, dvalue, state, last, dlast = z(b, t, c), z(b, t, c), z(b, t, c), f(b, c), z(b, c), z(b, c)
    logits, teacher, lse, loss, dz = f(m, n), f(m, 5), f(m), z(m), z(m, n)
    return {
        "embedding": ([table], lambda: p.ct_embedding(table.ptr, ids.ptr, m, n, k, 2.0, rows.ptr), [rows]),
        "embedding_grad": ([dout], lambda: p.ct_embedding_grad(ids.ptr, dout.ptr, m, n, k, 2.0, dtable.ptr), [dtable]),
        "gated_scan": ([gate, value, state], lambda: p.ct_gated_scan(gate.ptr, value.ptr, state.ptr, None, b, t, c, h.ptr, last.ptr), [h, last]),
        "gated_scan_in_place": ([gate, value, state], lambda: p.ct_gated_scan(gate.ptr, value.ptr, state.ptr, None, b, t, c, h.ptr, state.ptr), [h, state]),
        "gated_scan_grad": ([gate, value, out, dy, state],
                            lambda: p.ct_gated_scan_grad(gate.ptr, value.ptr, state.ptr, None, out.ptr, dy.ptr, None, b, t, c, dgate.ptr, dvalue.ptr, dlast.ptr),
                            [dgate, dvalue, dlast]),
        "distill": ([logits, teacher], lambda: p.ct_distill(logits.ptr, entries.ptr, teacher.ptr, m, n, 5, 2.0, loss.ptr, last.ptr if m <= b * c else lse.ptr), [loss]),
        "distill_grad": ([logits, teacher, lse], lambda: p.ct_distill_grad(logits.ptr, entries.ptr, teacher.ptr, lse.ptr, None, m, n, 5, 2.0, dz.ptr), [dz]),
        "distill_grad_in_place": ([logits, teacher, lse],
                                  lambda: p.ct_distill_grad(logits.ptr, entries.ptr, teacher.ptr, lse.ptr, None, m, n, 5, 2.0, logits.ptr), [logits]),
    }


@gpu
@pytest.mark.parametrize("m,n,k", [(1, 300, 40), (2, 40, 64), (16, 2000, 512), (300, 77, 33), (700, 3000, 128), (6000, 700, 24)])
@pytest.mark.parametrize("name", ["embedding", "embedding_grad", "gated_scan", "gated_scan_in_place", "gated_scan_grad", "distill", "distill_grad",
                                  "distill_grad_in_place"])
def test_operator_on_rewritten_inputs(name, m, n, k):
    """The operator, its inputs doubled in place, the operator again: the same bytes as with pauses between."""
    inputs, call, outputs = rewritten(np.random.default_rng(m + n + k), m, n, k)[name]
    kept = [a.numpy() for a in inputs]

    def run(wait):
        for a, v in zip(inputs, kept):
            L.check(L.lib.ct_h2d(a.ptr, v.ctypes.data, v.nbytes))
        L.check(call())
        for a in inputs:
            if wait:
                T.sync()
            L.check(L.lib.ct_binary(L.ADD, L.F32, a.ptr, L.F32, a.ptr, a.numel, a.ptr))
        if wait:
            T.sync()
        L.check(call())
        T.check_async()
        return [o.numpy().tobytes() for o in outputs]

    want = run(True)
    assert [run(False) == want for _ in range(10)] == [True] * 10


PART = 1 << 18  # values; a buffer has four, operands are different parts of different buffers


def any_call(rng, buffers, ids):
    i, j, l, o = rng.permutation(len(buffers))[:4]
    at = lambda b, part=0: buffers[b].ptr + part * PART * 4  # noqa: E731
    log = lambda most: max(1, int(round(np.exp(rng.uniform(0, np.log(most))))))  # noqa: E731
    while True:
        m, n, k, b, t = log(20000), log(3000), log(600), log(20), log(600)
        top = log(40)
        if max(m * k, n * k, m * n, b * t * k) <= PART and m * top <= ids.numel:
            break
    x, y, v, w, out, p = at(i), at(j, 1), at(l, 2), at(i, 3), [at(o, q) for q in range(4)], L.lib
    return [
        lambda: p.ct_embedding(x, ids.ptr, m, n, k, 0.5, out[0]),
        lambda: p.ct_embedding_grad(ids.ptr, x, m, n, k, 0.5, out[0]),
        lambda: p.ct_gated_scan(x, y, v, None, b, t, k, out[0], out[1]),
        lambda: p.ct_gated_scan(x, y, None, ids.ptr, b, t, k, out[0], out[1]),
        lambda: p.ct_gated_scan(x, y, v, None, b, 1, k, None, v),
        lambda: p.ct_gated_scan_grad(x, y, v, None, w, at(j, 3), at(l, 3), b, t, k, out[0], out[1], out[2]),
        lambda: p.ct_distill(x, ids.ptr, y, m, n, top if m * top <= PART else 1, 2.0, out[0], out[0] + 4 * m),
        lambda: p.ct_distill_grad(x, ids.ptr, y, v, None, m, n, top if m * top <= PART else 1, 2.0, out[0]),
        lambda: p.ct_distill_grad(x, ids.ptr, y, v, None, m, n, top if m * top <= PART else 1, 2.0, x),
        lambda: p.ct_layer_norm(x, None, None, m, k, 1e-5, out[0]),
        lambda: p.ct_matmul(L.F32, x, L.F32, y, m, k, n, out[0]),
        lambda: p.ct_binary(L.ADD, L.F32, x, L.F32, y, m * k, out[0]),
        lambda: p.ct_fill(L.F32, 0.25, m, out[0]),
    ][int(rng.integers(0, 13))]


@gpu
@pytest.mark.parametrize("seed", range(3))
def test_sequences_without_pauses(seed):
    """Sequences of up to 14 operators leave the same bytes in all buffers as with a pause behind each, and recorded and replayed, too."""
    rng = np.random.default_rng(seed)
    first = [dev(rng.normal(0, 0.3, 4 * PART).astype(np.float32)) for _ in range(5)]
    buffers, kept = [T.zeros([4 * PART]) for _ in first], [T.zeros([4 * PART]) for _ in first]
    ids = dev(rng.integers(-1, 300, 1 << 16))

    def copy(to, source):
        for a, b in zip(to, source):
            L.check(L.lib.ct_d2d(a.ptr, b.ptr, a.nbytes))
        T.sync()

    def same():
        equal = [T.Tensor(L.BOOL, (2 * PART,)) for _ in buffers]
        for e, a, b in zip(equal, buffers, kept):  # two values as an int64: NaN equals itself
            L.check(L.lib.ct_compare(L.EQ, L.I64, a.ptr, L.I64, b.ptr, 2 * PART, e.ptr))
        return all(e.numpy().all() for e in equal)

    for number in range(150):
        calls = [any_call(rng, buffers, ids) for _ in range(int(rng.integers(3, 15)))]
        copy(buffers, first)
        for call in calls:
            L.check(call())
            T.sync()
        copy(kept, buffers)
        for again in range(3):
            copy(buffers, first)
            for call in calls:
                L.check(call())
            T.check_async()
            assert same(), (number, again)
        with T.Graph() as graph:
            for call in calls:
                L.check(call())
        copy(buffers, first)
        graph.launch()
        T.check_async()
        assert same(), (number, "recorded")
        del graph  # not while the next one records


# ---- a network over sequences of tokens, which learns from a larger one's answers ---------------------


def network(ids, lengths, entries, teacher, p, state=None, temperature=2.0):
    """Losses, the states behind the sequences, and what the way back needs."""
    b, t = ids.shape
    k, c = p["table"].shape[1], p["w_gate"].shape[1]
    x = T.embedding(p["table"], ids, math.sqrt(k))
    rows = T.reshape(x, (b * t, k))
    y = T.layer_norm(rows, p["gamma"], p["beta"])
    gate, value = T.dense(y, p["w_gate"]), T.dense(y, p["w_value"])
    h, last = T.gated_scan(T.reshape(gate, (b, t, c)), T.reshape(value, (b, t, c)), state, lengths)
    hidden = T.reshape(h, (b * t, c))
    up, g, u = T.dense_gated(hidden, p["v_gate"], p["v_up"], keep=True)
    logits = T.dense(up, p["w_out"])
    loss, lse = T.distill(logits, entries, teacher, temperature)
    return loss, last, (rows, y, gate, value, h, hidden, up, g, u, logits, lse)


def network_grad(ids, lengths, entries, teacher, p, kept, state=None, temperature=2.0):
    rows, y, gate, value, h, hidden, up, g, u, logits, lse = kept
    (b, t), (k, c) = ids.shape, p["w_gate"].shape
    dlogits = T.distill_grad(logits, entries, teacher, lse, temperature)
    d = {"w_out": T.matmul_tn(up, dlogits)}
    dup = T.matmul(dlogits, T.transpose(p["w_out"]))
    dhidden, d["v_gate"], d["v_up"] = T.dense_gated_grad(hidden, p["v_gate"], p["v_up"], g, u, dup)
    shape = (b, t, c)
    dgate, dvalue, *first = T.gated_scan_grad(T.reshape(gate, shape), T.reshape(value, shape), h, T.reshape(dhidden, shape), state, lengths)
    dgate, dvalue = T.reshape(dgate, (b * t, c)), T.reshape(dvalue, (b * t, c))
    d["w_gate"], d["w_value"] = T.matmul_tn(y, dgate), T.matmul_tn(y, dvalue)
    dy = T.add(T.matmul(dgate, T.transpose(p["w_gate"])), T.matmul(dvalue, T.transpose(p["w_value"])))
    drows, d["gamma"], d["beta"] = T.layer_norm_grad(rows, dy, p["gamma"])
    d["table"] = T.embedding_grad(ids, T.reshape(drows, (b, t, k)), p["table"].shape[0], math.sqrt(k))
    return d, first


def network_inputs(seed=0, b=5, t=23, vocabulary=170, k=36, c=40, n=48, top=6):
    rng = np.random.default_rng(seed)
    f = lambda s, *shape: rng.normal(0, s, shape).astype(np.float32)  # noqa: E731
    p = dict(table=f(1 / math.sqrt(k), vocabulary, k), gamma=1 + f(0.1, k), beta=f(0.1, k), w_gate=f(2 / math.sqrt(k), k, c), w_value=f(1 / math.sqrt(k), k, c),
             v_gate=f(1 / math.sqrt(c), c, n), v_up=f(1 / math.sqrt(c), c, n), w_out=f(1 / math.sqrt(n), n, vocabulary))
    lengths = rng.integers(1, t + 1, b)
    lengths[0] = t
    ids = np.where(np.arange(t) < lengths[:, None], rng.integers(0, vocabulary, (b, t)), -1)
    entries = np.where((ids >= 0).reshape(-1, 1), rng.integers(0, vocabulary, (b * t, top)), -1)
    return ids, lengths, entries, f(2, b * t, top), p, f(0.5, b, c)


def network_torch(ids, lengths, entries, teacher, p, state, temperature=2.0):
    """The same in 64 bits, with torch's own gradients."""
    import torch

    w = {key: torch.tensor(v, dtype=torch.float64, requires_grad=True) for key, v in p.items()}
    first = torch.tensor(state, dtype=torch.float64, requires_grad=True)
    ids, entries = torch.tensor(ids), torch.tensor(entries)
    b, t = ids.shape
    k = w["table"].shape[1]
    x = torch.where(ids[..., None] >= 0, w["table"][ids.clamp_min(0)] * float(np.float32(math.sqrt(k))), 0.0)
    y = torch.nn.functional.layer_norm(x, (k,), w["gamma"], w["beta"], 1e-5)
    a, value, h, out = torch.sigmoid(y @ w["w_gate"]), y @ w["w_value"], first, []
    for i in range(t):
        on = torch.tensor(lengths > i)[:, None]
        h = torch.where(on, a[:, i] * h + (1 - a[:, i]) * value[:, i], h)
        out.append(torch.where(on, h, torch.zeros_like(h)))
    hidden = torch.stack(out, 1).reshape(b * t, -1)
    up = torch.nn.functional.silu(hidden @ w["v_gate"]) * (hidden @ w["v_up"])
    log_q = torch.log_softmax(up @ w["w_out"] / temperature, 1)
    some = (entries >= 0).any(1)
    scores = torch.where(entries >= 0, torch.tensor(teacher, dtype=torch.float64) / temperature, -torch.inf)[some]
    log_p = torch.log_softmax(scores, 1)
    terms = torch.where(entries[some] >= 0, log_p.exp() * (log_p - log_q[some].gather(1, entries[some].clamp_min(0))), torch.zeros(()))
    loss = temperature ** 2 * terms.nan_to_num(0.0).sum(1)
    loss.sum().backward()
    full = torch.zeros(b * t, dtype=torch.float64)
    full[some] = loss.detach()
    return full.numpy(), h.detach().numpy(), {key: v.grad.numpy() for key, v in w.items()}, first.grad.numpy()


@gpu
@pytest.mark.parametrize("sizes", [dict(), dict(b=1, t=1), dict(b=2, t=300, vocabulary=700, k=33), dict(b=30, t=9, c=100, top=40)])
def test_a_network_over_tokens(sizes):
    """Losses, last states and every gradient, by the largest of each: products are within 2^-20 of theirs, and some ten operators follow one another."""
    ids, lengths, entries, teacher, p, state = network_inputs(**sizes)
    d = {key: dev(v) for key, v in p.items()}
    args = dev(ids), dev(lengths), dev(entries), dev(teacher), d
    loss, last, kept = network(*args, dev(state))
    grads, (dstate,) = network_grad(*args, kept, dev(state))
    want_loss, want_last, want, want_state = network_torch(ids, lengths, entries, teacher, p, state)
    near = lambda got, ref, what: within(got, ref, np.full(ref.shape, 5e-5 * np.abs(ref).max() + 1e-12), what)  # noqa: E731
    near(loss.numpy(), want_loss, "loss")
    near(last.numpy(), want_last, "state")
    near(dstate.numpy(), want_state, "dstate")
    for key, ref in want.items():
        near(grads[key].numpy(), ref, key)


@gpu
def test_a_recorded_training_step():
    """The same step eager and recorded, twice each: the same bytes."""
    ids, lengths, entries, teacher, p, state = [dev(a) if isinstance(a, np.ndarray) else a for a in network_inputs(3)]
    p = {key: dev(v) for key, v in p.items()}
    T.set_weight_cache(False)
    try:
        def step():
            loss, last, kept = network(ids, lengths, entries, teacher, p, state)
            grads, first = network_grad(ids, lengths, entries, teacher, p, kept, state)
            moved = [T.scaled_sub(p[key], grads[key], 0.01) for key in sorted(p)]
            return [loss, last, *first, *moved]

        want = bytes_of(step())
        assert bytes_of(step()) == want
        with T.Graph() as graph:
            graph.keep = step()
        for _ in range(2):
            graph.launch()
            T.check_async()
            assert bytes_of(graph.keep) == want
    finally:
        T.set_weight_cache(True)


@gpu
def test_answering_token_by_token():
    """The network on whole sequences, and on one token after the other with the states carried along: the same logits within the scan's bound."""
    _, _, _, _, p, state = network_inputs(4, b=3, t=40)
    rng = np.random.default_rng(1)
    ids = rng.integers(0, p["table"].shape[0], (3, 40))
    d = {key: dev(v) for key, v in p.items()}
    none, scores = dev(np.full((120, 1), -1)), dev(np.zeros((120, 1), np.float32))
    _, last, kept = network(dev(ids), None, none, scores, d, dev(state))
    whole = kept[9].numpy().reshape(3, 40, -1)
    now, worst = dev(state), 0.0
    for i in range(40):
        _, now, step = network(dev(ids[:, i:i + 1]), None, dev(np.full((3, 1), -1)), dev(np.zeros((3, 1), np.float32)), d, now)
        worst = max(worst, np.abs(step[9].numpy() - whole[:, i]).max())
    assert worst <= 2e-5 * np.abs(whole).max()
    assert np.abs(now.numpy() - last.numpy()).max() <= (SCAN + 40 * U) * max(np.abs(state).max(), np.abs(kept[3].numpy()).max())
