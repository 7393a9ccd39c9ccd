"""Plans and forks whose sequences have more pages in all than 32-bit sums over them hold, while some share any: refused as a whole."""
import numpy as np
import pytest
import torch

import q4hip
from test_gpu_kv8 import ints

pytestmark = pytest.mark.gpu

B, W = 70000, 61000             # B * W = 2^32 - 24,967,296: taken pages that counted as less than none


@pytest.fixture(scope="module")
def cache():
    if torch.cuda.mem_get_info()[0] < 64 << 30:
        pytest.skip("two tables of 17 GB")
    kv = q4hip.Kv8(1, 1, 1, 64, B, 32 * W, W + 20, 64)
    yield kv
    kv.close()


def plan(kv, have):
    h, a = ints(have), torch.zeros(B, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    kv.plan(h.data_ptr(), a.data_ptr(), 0)


def fork(kv, source, keep):
    f, k = ints(source), ints(keep)
    torch.cuda.synchronize()
    kv.fork(f.data_ptr(), k.data_ptr())


def only(**held):
    lens = np.zeros(B, np.int64)
    for b, n in held.items():
        lens[int(b[1:])] = n
    return lens


def test_a_plan_that_takes_more(cache):
    plan(cache, only(b0=70))
    fork(cache, np.zeros(B, np.int64), only(b0=70, b1=70))
    assert cache.status() == (0, W + 20 - 4)
    with pytest.raises(q4hip.Q4Error) as e:
        plan(cache, np.full(B, 32 * W))
    assert e.value.code == q4hip.ECONTEXT
    plan(cache, only(b0=70, b1=70))                 # nothing has changed
    assert cache.status() == (0, W + 20 - 4)
    plan(cache, only())
    assert cache.status() == (0, W + 20)


def test_a_fork_that_shares_more(cache):
    plan(cache, only(b0=32 * W))
    with pytest.raises(q4hip.Q4Error) as e:
        fork(cache, np.zeros(B, np.int64), np.where(np.arange(B) == 0, 32 * W, 32 * 17000))      # 1.19e9 pages
    assert e.value.code == q4hip.ECONTEXT
    plan(cache, only(b0=32 * W))
    assert cache.status() == (0, 20)
    fork(cache, np.zeros(B, np.int64), only(b0=32 * W, b9=32 * 300))
    assert cache.status() == (0, 20)
    plan(cache, only(b9=32 * 300))                  # the pages in common stay
    assert cache.status() == (0, W + 20 - 300)
    plan(cache, only())
    assert cache.status() == (0, W + 20)
