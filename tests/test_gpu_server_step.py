"""A server's step on buffers of its own: plan, rotary positions, append, attention of forked chats, logits' rules, captured in one
graph and replayed as chats grow, fork and end; every part against its own plain form."""
import numpy as np
import pytest
import torch

import q4hip
import test_gpu_logits as lt
import test_gpu_rope as rt
from test_gpu_kv8 import TYPES, ints
from test_gpu_kv8_fork import Forked

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,order,rot,join", [("f32", "halves", 64, "0"), ("bf16", "pairs", 32, "0"), ("f16", "halves", 48, None)])
def test_steps_of_a_server(monkeypatch, dtype, order, rot, join):
    if join is not None:
        monkeypatch.setenv("Q4HIP_KV8_JOINT_SAVES", join)
    rng = np.random.default_rng(rot)
    typ, tt = TYPES[dtype]
    H, KVH, hd, B, V, most = 6, 2, 64, 7, 3001, 12
    w = (H + 2 * KVH) * hd
    t = Forked(H, KVH, hd, B, 900, 120, 700, 2)
    t.grow(rng, [0] * B, [600] + [0] * (B - 1), dtype)
    t.fork([0] * B, [600, 600, 590, 300, 0, 600, 600])
    lens = [600, 600, 590, 300, 0, 600, 600]
    freq, amplitude = q4hip.rope_frequencies(rot, 1e4, "bands", 4.0, 512, 1.0, 4.0)
    rope, logits = q4hip.Rope(hd, rot, order, freq, amplitude), q4hip.Logits(V, most)
    head = (torch.randn(H * hd, V, device="cuda") / 8).to(tt)
    have, add, positions = ints([0] * B), ints([0] * B), ints([0] * most)
    starts = ints([0] * (B + 1))
    x0, x = (torch.zeros(most, w, dtype=tt, device="cuda") for _ in range(2))
    outs = [torch.zeros(most, H * hd, dtype=tt, device="cuda") for _ in range(2)]
    lg = torch.zeros(most, V, dtype=tt, device="cuda")
    best = ints([0] * most)
    p, h, b, mask, allowed = lt.rules(rng, most, V, history=200, biases=9, masks=3)
    dp, dh, db, dm = (lt.device(a) for a in (p, h, b, mask))
    before = torch.zeros_like(lg)

    def step(s):
        x.copy_(x0)
        t.kv.plan(have.data_ptr(), add.data_ptr(), most, starts.data_ptr(), positions.data_ptr(), 0, 0, s)
        rope.run(x.data_ptr(), x.data_ptr(), H + KVH, typ, w, w, positions.data_ptr(), most, starts[B:].data_ptr(), s)
        for layer in range(2):
            t.kv.append(layer, x[:, H * hd:].data_ptr(), x[:, (H + KVH) * hd:].data_ptr(), typ, w, w, s)
            t.kv.attend(layer, x.data_ptr(), outs[layer].data_ptr(), typ, w, H * hd, s)
        lg.copy_((outs[1].float() @ head.float()).to(tt))
        before.copy_(lg)
        logits.run(lg.data_ptr(), lg.data_ptr(), typ, V, V, most, dp.data_ptr(), dh.data_ptr(), len(h), db.data_ptr(), len(b), dm.data_ptr(),
                   len(mask), best.data_ptr(), s)

    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):                 # the libraries' own first calls, outside of the capture
        (outs[1].float() @ head.float()).to(tt)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        step(torch.cuda.current_stream().cuda_stream)
    for turn in range(6):
        if turn in (2, 4):
            source = [0, 1, 1, 3, 5, 0, 6]
            keep = [lens[s] if s != 3 else 0 for s in source]
            t.fork(source, keep)
            lens = keep
        more = rng.integers(0, 3, B).tolist()
        more[turn] = 1
        n = sum(more)
        have.copy_(ints(lens))
        add.copy_(ints(more))
        x0.copy_(torch.randn(most, w, device="cuda"))
        for out in outs:
            out.fill_(7.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        t.have, t.add = lens, more
        st, pos, t.slots, _, t.seq = t.pool.plan(lens, more, most)
        assert np.array_equal(starts.cpu(), st) and np.array_equal(positions.cpu()[:n], pos) and t.kv.status() == (n, len(t.pool.stack))
        # rotary positions: of q and k, of the step's rows alone
        turned = (H + KVH) * hd
        rt.check(x[:n, :turned], x0[:n, :turned], dtype, pos, freq, amplitude, H + KVH, hd, rot, order)
        assert torch.equal(x[n:], x0[n:]) and torch.equal(x[:, turned:], x0[:, turned:])
        y = x[:n].float().cpu().numpy()
        for layer in range(2):
            for c, at in ((0, H), (1, H + KVH)):
                t.ref[layer][c].append(y[:, at * hd:(at + KVH) * hd].reshape(n, KVH, hd), t.slots)
            t.check_values(layer)
            t.compare(outs[layer][:n].double().cpu().numpy().reshape(n, H, hd), y[:, :H * hd].reshape(n, H, hd), dtype, layer)
            assert (outs[layer][n:] == 7).all()
        want, _, top = lt.plain(before.float().cpu().numpy(), p, h, b, allowed)
        assert torch.equal(lg.cpu().float(), torch.from_numpy(want).to(tt).float()) and np.array_equal(best.cpu().numpy(), top)
        lens = [a + c for a, c in zip(lens, more)]
