"""Rows of rotary positions and of logits that take more threads than one launch has."""
import numpy as np
import pytest
import torch

import q4hip

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()


def room(gib):
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"{gib} GiB")


@pytest.mark.parametrize("rows", [2 ** 25 + 3, 2 ** 26 + 5, 2 ** 31 - 1])
def test_rope(rows):
    """Pairs of one column each in place; row t at position t.  In bf16 (1, 0) becomes (cos, sin) and (0, 1) (-sin, cos)."""
    room(40)
    r = q4hip.Rope(2, 2, "halves", [0.25])
    x = torch.zeros(rows, 2, dtype=torch.bfloat16, device="cuda")
    x[::2, 0] = 1
    x[1::2, 1] = 1
    pos = torch.arange(rows, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    r.run(x.data_ptr(), x.data_ptr(), 1, q4hip.BF16, 2, 2, pos.data_ptr(), rows)
    ends = [0, 2 ** 25 - 1, 2 ** 25, 2 ** 26, 2 ** 30, rows - 1]
    for at in [e for e in ends if e < rows] + np.random.default_rng(1).integers(0, rows, 20).tolist():
        lo, hi = max(0, at - 500), min(rows, at + 500)
        t = np.arange(lo, hi) * 0.25
        even = np.arange(lo, hi) % 2 == 0
        want = np.stack([np.where(even, np.cos(t), -np.sin(t)), np.where(even, np.sin(t), np.cos(t))], 1)
        got = x[lo:hi].double().cpu().numpy()
        assert (np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 9 * 2.0 ** -24).all(), at


def test_logits():
    """The best token of 2^20 rows of 8 pieces: the only one above the others."""
    room(140)
    rows, V = 2 ** 20, 7 * 8192 + 1
    lg = q4hip.Logits(V, rows)
    x = torch.full((rows, V), -1.0, dtype=torch.bfloat16, device="cuda")
    want = (torch.arange(rows, device="cuda") * 7919) % V
    for r in range(0, rows, 65536):
        x[r:r + 65536].scatter_(1, want[r:r + 65536, None], 1.0)
    params = np.zeros(rows, q4hip.LOGITS_ROW)
    params["repetition"], params["mask"] = 1.0, -1
    p = torch.from_numpy(params.view(np.int32).reshape(rows, 8)).cuda()
    best = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    for _ in range(2):
        lg.run(x.data_ptr(), x.data_ptr(), q4hip.BF16, V, V, rows, p.data_ptr(), best=best.data_ptr())
        assert torch.equal(best, want.int())
        best.fill_(-7)
        torch.cuda.synchronize()
    for r in (0, rows // 2, rows - 1000):                    # the rest as it was
        assert (x[r:r + 1000].float().sum(1) == 2 - V).all()
    lg.close()
