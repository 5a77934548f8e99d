"""The walk of a scan's blocks along the steps (camel_b200/csrc/scan_walk.cuh) with threads of the host in place of warps, and with waits that run out.

On the GPU no input makes a wait run out, and nothing is broken on purpose there: here a warp is late, a copy does not come, or comes too late.  The block
that cannot go on has to say so, all have to end, and none may do what the machine leaves undefined (tests/scan_walk/machine.h)."""
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest

import camel_b200._lib as L
from camel_b200 import tensor as T

HERE = Path(__file__).resolve().parent
WALK = HERE.parent / "camel_b200" / "csrc" / "scan_walk.cuh"


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if not shutil.which("g++"):
        pytest.skip("no g++")
    to = tmp_path_factory.mktemp("scan_walk")
    shutil.copy(WALK, to)
    for name in ("common.cuh", "tc_ptx.cuh", "tmap.cuh"):  # the machine in their place
        (to / name).write_text('#include "machine.h"\n')
    for name in ("machine.h", "walk.cpp"):
        shutil.copy(HERE / "scan_walk" / name, to)
    r = subprocess.run(["g++", "-std=c++17", "-O1", "-pthread", "walk.cpp", "-o", "walk"], cwd=to, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return to / "walk"


def run(program, tiles, what, when=6):
    return subprocess.run([program, str(tiles), what, str(when)], capture_output=True, text=True, timeout=60, check=True).stdout.splitlines()


@pytest.mark.parametrize("tiles", [1, 2, 3, 4, 5, 40])
def test_all_blocks_have_the_state(program, tiles):
    assert run(program, tiles, "nothing") == [f"block {b} right" for b in range(3)]


@pytest.mark.parametrize("what", ["slow", "lost", "late"])
@pytest.mark.parametrize("tiles,when", [(40, 6), (40, 0), (40, 39), (5, 3), (1, 0)])
def test_a_wait_that_runs_out(program, what, tiles, when):
    out = run(program, tiles, what, when)
    assert not [line for line in out if line.startswith("violation")]
    assert len(out) == 3 and "block 1 reported" in out  # on the device the blocks report in one word


@pytest.mark.gpu
def test_the_record_of_a_wait_stays_until_it_is_checked():
    """As if a block of a scan had given up, written from the host: the scans behind it run, and ct_check reports it once."""
    rng = np.random.default_rng(5)
    gate, value = (T.from_numpy(rng.normal(0, 1, (2, 3000, 64)).astype(np.float32)) for _ in range(2))  # blocks of a cluster
    out, state = T.gated_scan(gate, value)
    T.check_async()
    L.check(L.lib.ct_inject_status(2, 8))
    again, last = T.gated_scan(gate, value)
    assert again.numpy().tobytes() == out.numpy().tobytes() and last.numpy().tobytes() == state.numpy().tobytes()
    assert L.lib.ct_check() == L.ERR_TIMEOUT and "block 7" in L.lib.ct_last_error().decode()
    assert L.lib.ct_check() == 0
