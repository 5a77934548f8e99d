"""The operators that use clusters of more than 8 blocks, without them: what a device has by itself that has no room for larger ones."""
import os
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest

from camel_b200 import tensor as T
from test_layers import U, dev

gpu = pytest.mark.gpu
GRADIENTS = [(9000, 700, 24), (17000, 3, 6), (40000, 50000, 4), (70000, 131072, 3), (140000, 2000, 2), (300000, 70, 5)]  # tokens, rows, columns
SCANS = [(1, 20000, 512), (2, 5000, 33)]


def calls():
    rng = np.random.default_rng(11)
    out = {}
    for m, n, k in GRADIENTS:
        ids = np.minimum((np.power(n + 1.0, rng.uniform(0, 1, m)) - 1).astype(np.int64), n - 1)
        ids[rng.uniform(0, 1, m) < 0.1] = -1
        out[f"gradient {m} {n} {k}"] = T.embedding_grad(dev(ids), dev(rng.normal(0, 1, (m, k)).astype(np.float32)), n).numpy()
    for shape in SCANS:
        gate, value, dout = (dev(rng.normal(0, 1, shape).astype(np.float32)) for _ in range(3))
        h, state = T.gated_scan(gate, value)
        dgate, dvalue = T.gated_scan_grad(gate, value, h, dout)
        for name, t in (("out", h), ("state", state), ("dgate", dgate), ("dvalue", dvalue)):
            out[f"scan {shape} {name}"] = t.numpy()
    T.check_async()
    return out


@gpu
def test_clusters_of_eight_blocks(tmp_path):
    to = tmp_path / "portable.npz"
    code = "import sys; sys.path[:0] = sys.argv[2:]; import numpy as np; from test_portable_clusters import calls; np.savez(sys.argv[1], **calls())"
    tests = Path(__file__).resolve().parent
    subprocess.run([sys.executable, "-c", code, str(to), str(tests), str(tests.parent)], check=True, timeout=300,
                   env={**os.environ, "CAMEL_TENSOR_PORTABLE_CLUSTERS": "1"})
    got, want = np.load(to), calls()
    assert set(got.files) == set(want)
    for name, a in want.items():
        b = got[name]
        if name.startswith("gradient"):
            assert a.tobytes() == b.tobytes(), name  # the same order of the same tokens
        else:  # in other pieces: each value is a few roundings of the largest so far from its definition
            assert np.abs(a - b).max() <= 32 * U * np.abs(a).max(), name
