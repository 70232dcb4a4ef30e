"""CPU proof of the paged attention's index math: tests/paged_plan_sim.c runs
every wave's walk and the merge with the kernels' own header
(laii_amd/csrc/paged_q4.h).  No GPU needed."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
U32P = C.POINTER(C.c_uint32)


@pytest.fixture(scope="module")
def sim(tmp_path_factory):
    out = str(tmp_path_factory.mktemp("plan") / "libpagedsim.so")
    subprocess.run(["gcc", "-O2", "-std=c11", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC",
                    "-I", os.path.join(ROOT, "laii_amd", "csrc"), os.path.join(ROOT, "tests", "paged_plan_sim.c"),
                    "-o", out], check=True)
    lib = C.CDLL(out)
    lib.plan_check.restype = C.c_int
    lib.plan_check.argtypes = [C.c_uint32, U32P, U32P] + [C.c_uint32] * 8 + [C.c_int, C.c_char_p, C.c_size_t]

    def check(pos, n_rows, mul, nkv, window=0, capacity=1 << 20, cols=16, shift=5, waves=2048, rows=None, mutant=0):
        pos = np.ascontiguousarray(pos, np.uint32)
        rows = None if rows is None else np.ascontiguousarray(rows, np.uint32)
        msg = C.create_string_buffer(256)
        rc = lib.plan_check(pos.size, pos.ctypes.data_as(U32P), None if rows is None else rows.ctypes.data_as(U32P),
                            n_rows, mul, nkv, window, capacity, cols, shift, waves, mutant, msg, 256)
        return rc, msg.value.decode()

    check.lib = lib
    lib.share.argtypes = [C.c_uint32] * 3 + [U32P] * 2
    return check


@pytest.mark.parametrize("seed", range(8))
def test_random_batches(sim, seed):
    rng = np.random.default_rng(seed)
    for i in range(150):
        n = int(rng.integers(1, 150))
        n_rows = int(rng.choice([1, 1, 2, 5, 8, 40, 200]))
        mul, nkv = int(rng.integers(1, 9)), int(rng.integers(1, 9))
        cols, shift = (4, 6) if n_rows * mul <= 4 and rng.random() < 0.7 else (int(rng.choice([8, 16, 32])), 5)
        capacity = int(rng.choice([32, 64, 1024, 32768]))
        pos = rng.integers(0, int(capacity * 1.1) + 1, n)
        rows = rng.integers(0, n_rows + 2, n) if rng.random() < 0.5 else None
        window = int(rng.choice([0, 0, 1, 31, 33, 300]))
        waves = 4 * int(rng.integers(1, 513))
        rc, msg = sim(pos, n_rows, mul, nkv, window, capacity, cols, shift, waves, rows)
        assert rc == 0, (i, rc, msg)


@pytest.mark.parametrize("pos,rows,n_rows", [
    ([0], None, 1), ([0], [0], 1), ([0xFFFFFFFF, 5], None, 4), ([2 ** 31 - 2], None, 8), ([0] * 300, [0] * 300, 1),
    ([0] * 299 + [2 ** 20], [0] * 299 + [1], 1), ([2 ** 31 - 1, 2 ** 31], None, 2)])
def test_ends(sim, pos, rows, n_rows):
    """Nothing to do, one key, the last positions a table can reach, one long sequence behind many empty ones."""
    for window in (0, 1, 2 ** 31, 0xFFFFFFFF):
        for waves in (4, 2048):
            rc, msg = sim(pos, n_rows, 4, 1, window, 2 ** 31, 16, 5, waves, rows)
            assert rc == 0, (window, waves, rc, msg)


@pytest.mark.parametrize("units,n_steps,k", [(128, 129, 4), (8, 2049, 256), (24, 77, 84), (3, 1000, 680), (512, 9, 4)])
def test_equal_units_are_cut_at_their_ends(sim, units, n_steps, k):
    """k waves for each of equal units: none holds the end of one and the start of the next."""
    waves, k = -(-units * k // 4) * 4, min(k, n_steps)  # a wave has a step at least
    for u in range(units):
        for g in (u * k, u * k + k - 1):
            t0, t1 = C.c_uint32(), C.c_uint32()
            sim.lib.share(g, units * n_steps, units * k, C.byref(t0), C.byref(t1))
            assert u * n_steps <= t0.value < t1.value <= (u + 1) * n_steps
            assert g != u * k or t0.value == u * n_steps
    assert sim([n_steps * 32 - 1] * units, 1, 4, 1, 0, 1 << 20, 16, 5, waves)[0] == 0


@pytest.mark.parametrize("mutant", [1, 2, 3])
def test_checks_find_mistakes(sim, mutant):
    assert sim([3000, 70, 9000], 1, 4, 2, 0, 1 << 20, 16, 5, 256, None, mutant)[0] != 0
