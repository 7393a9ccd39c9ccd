"""The paged 8-bit cache: a capture changes nothing for the calls outside of it."""
import numpy as np
import pytest
import torch

import q4hip
from test_gpu_kv8 import Both, ints

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [3, 0, 40])
def test_calls_between_a_plan_and_their_own(rows):
    """A plan of 20 rows, then a step of `rows` rows captured, then the append and attention of the 20; the graph afterwards."""
    rng = np.random.default_rng(rows)
    H, KVH, hd = 4, 2, 64
    w = (H + 2 * KVH) * hd
    t = Both(H, KVH, hd, 2, 300, 20, 300)
    t.plan([0, 0], [30, 5])
    t.fill(rng, "f32")
    have, add = ints([40, 15]), ints([rows // 2, rows - rows // 2])
    x, out = torch.randn(64, w, device="cuda"), torch.full((64, H * hd), 7.0, device="cuda")
    t.plan([30, 5], [10, 10])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        s = torch.cuda.current_stream().cuda_stream
        t.kv.plan(have.data_ptr(), add.data_ptr(), rows, stream=s)
        t.kv.append(0, x[:, H * hd:].data_ptr(), x[:, (H + KVH) * hd:].data_ptr(), q4hip.F32, w, w, s)
        t.kv.attend(0, x.data_ptr(), out.data_ptr(), q4hip.F32, w, H * hd, s)
        out.add_(0)                                # a graph is never empty
    t.fill(rng, "f32")
    t.check_values()
    t.attend(rng, "f32")
    assert t.kv.status() == (20, len(t.pool.stack))
    for _ in range(3):
        out.fill_(7.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        t.have, t.add = [40, 15], [rows // 2, rows - rows // 2]
        _, _, t.slots, _, t.seq = t.pool.plan(t.have, t.add, rows)
        y = x[:rows].cpu().numpy()
        for c, at in ((0, H), (1, H + KVH)):
            t.ref[0][c].append(y[:, at * hd:(at + KVH) * hd].reshape(rows, KVH, hd), t.slots)
        assert t.kv.status() == (rows, len(t.pool.stack)) and (out[rows:] == 7).all()
        t.check_values()
        if rows:
            t.compare(out[:rows].double().cpu().numpy().reshape(rows, H, hd), y[:, :H * hd].reshape(rows, H, hd), "f32")


def test_two_captures_of_different_rows():
    """Each graph's append and attend count with its own plan."""
    rng = np.random.default_rng(2)
    H, KVH, hd, w = 4, 2, 64, 8 * 64
    t = Both(H, KVH, hd, 1, 300, 20, 300)
    t.plan([0], [50])
    t.fill(rng, "f32")
    add, have = ints([0]), ints([50])
    x, out = torch.randn(64, w, device="cuda"), torch.full((64, H * hd), 7.0, device="cuda")
    graphs = {}
    torch.cuda.synchronize()
    for rows in (24, 2):
        graphs[rows] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[rows], stream=torch.cuda.Stream()):
            s = torch.cuda.current_stream().cuda_stream
            t.kv.plan(have.data_ptr(), add.data_ptr(), rows, stream=s)
            t.kv.append(0, x[:, H * hd:].data_ptr(), x[:, (H + KVH) * hd:].data_ptr(), q4hip.F32, w, w, s)
            t.kv.attend(0, x.data_ptr(), out.data_ptr(), q4hip.F32, w, H * hd, s)
    for rows in (24, 2, 24, 2):
        add.copy_(ints([rows]))
        out.fill_(7.0)
        torch.cuda.synchronize()
        graphs[rows].replay()
        torch.cuda.synchronize()
        assert t.kv.status()[0] == rows and (out[rows:] == 7).all()
        t.have, t.add = [50], [rows]
        _, _, t.slots, _, t.seq = t.pool.plan([50], [rows], rows)
        y = x[:rows].cpu().numpy()
        for c, at in ((0, H), (1, H + KVH)):
            t.ref[0][c].append(y[:, at * hd:(at + KVH) * hd].reshape(rows, KVH, hd), t.slots)
        t.check_values()
        t.compare(out[:rows].double().cpu().numpy().reshape(rows, H, hd), y[:, :H * hd].reshape(rows, H, hd), "f32")
