"""Forks of the 8-bit cache: refusals that need no GPU, and the plain pool that the GPU tests compare with."""
import ctypes

import numpy as np

import q4hip
from kv8_fork_ref import SharedPool


def test_null_arguments():
    one = ctypes.c_int(0)
    p = ctypes.addressof(one)
    assert q4hip.lib().q4hip_kv8_fork(None, p, p, None, None) == q4hip.EINVAL


def test_plain_pool_loses_no_page():
    rng = np.random.default_rng(1)
    pool = SharedPool(5, 200, 22)
    lens = [0] * 5
    done = {"plan": 0, "fork": 0}
    for _ in range(400):
        if rng.random() < 0.5:
            f = rng.integers(0, 5, 5).tolist()
            k = [int(rng.integers(0, lens[s] + 1)) for s in f]
            if pool.fork(f, k) is not None:
                lens = k
                done["fork"] += 1
        else:
            have = [int(rng.integers(0, n + 1)) if rng.random() < 0.2 else n for n in lens]
            add = [int(rng.integers(0, min(40, 201 - h))) if rng.random() < 0.5 else 0 for h in have]
            if pool.plan(have, add, sum(add)) is not None:
                lens = [h + a for h, a in zip(have, add)]
                done["plan"] += 1
        held = {p for t in pool.tables for p in t}
        assert sorted(list(held) + pool.stack) == list(range(22)) and [len(t) for t in pool.tables] == [-(-n // 32) for n in lens]
        # a page that may be written to belongs to one sequence, unless its sequence was cut back to within it
        n = pool.holders()
        assert all(n[p] > 0 for p in held)
    assert min(done.values()) > 60
