"""Attention of sequences that begin with the same pages, which one pass serves for all, against kv8_ref.py; its rows' bound holds
for any split of the positions."""
import numpy as np
import pytest
import torch

import q4hip
from test_gpu_kv8 import ints
from test_gpu_kv8_fork import Forked

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def join_all(monkeypatch):
    """However little it saves."""
    monkeypatch.setenv("Q4HIP_KV8_JOINT_SAVES", "0")


def grown(rng, H, KVH, hd, prefixes, dtype, own=40, spare=0, layers=1, max_rows=4000):
    """Groups of sequences: prefixes is [(positions, sequences)]; every sequence then adds up to `own` rows of its own."""
    B = sum(n for _, n in prefixes) + spare
    longest = max(p for p, _ in prefixes) + own + 300
    pages = sum(-(-p // 32) for p, _ in prefixes) + B * (-(-(own + 300) // 32) + 2)
    t = Forked(H, KVH, hd, B, longest, pages, max(max_rows, sum(p for p, _ in prefixes)), layers)
    lead, keep, first = list(range(B)), [0] * B, [0] * B
    at = 0
    for p, n in prefixes:
        first[at] = p
        for b in range(at, at + n):
            lead[b], keep[b] = at, p
        at += n
    t.grow(rng, [0] * B, first, dtype)
    t.fork(lead, keep)
    add = [int(rng.integers(0, own + 1)) if k else 0 for k in keep]
    t.grow(rng, keep, add, dtype)
    return t, [k + a for k, a in zip(keep, add)]


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (4, 1, 128), (3, 3, 64), (16, 1, 64), (12, 2, 128), (15, 1, 128)])
@pytest.mark.parametrize("prefixes", [[(300, 2)], [(256, 5), (999, 3)], [(289, 33)]])
def test_one_token_each(dtype, H, KVH, hd, prefixes):
    rng = np.random.default_rng(H + hd)
    t, lens = grown(rng, H, KVH, hd, prefixes, dtype)
    t.grow(rng, lens, [1] * t.B, dtype)
    first = t.attend(rng, dtype)
    assert torch.isfinite(first).all()
    t.check_values()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("H,KVH,hd", [(2, 2, 64), (4, 2, 128), (10, 2, 64), (20, 1, 64)])
def test_rows_of_every_kind(dtype, H, KVH, hd):
    """Sequences that add no row, one, up to a unit's and many, behind two prefixes, beside one without a prefix."""
    rng = np.random.default_rng(H)
    t, lens = grown(rng, H, KVH, hd, [(480, 9), (257, 6)], dtype, spare=2)
    for step in range(3):
        add = rng.choice([0, 1, 1, 2, 3, 16 * KVH // H + 1, 40], t.B).tolist()
        add[1] = add[2] = 1
        t.grow(rng, lens, add, dtype)
        t.attend(rng, dtype)
        lens = [n + a for n, a in zip(lens, add)]


def test_prompts_in_tiles_beside_joints():
    """Enough rows for tiles, units and joints in one launch."""
    rng = np.random.default_rng(9)
    t, lens = grown(rng, 20, 20, 64, [(300, 12)], "f16", own=10, spare=4)
    add = [1] * 12 + [257, 130, 290, 200]
    t.grow(rng, lens, add, "f16")
    t.attend(rng, "f16")


@pytest.mark.parametrize("dtype", ["f32", "f16"])
@pytest.mark.parametrize("H,KVH,hd,positions", [(14, 2, 64, 9000), (8, 1, 128, 20000), (8, 8, 128, 3500)])
def test_long_prefixes(dtype, H, KVH, hd, positions):
    """Pages in common, and of units, shared among workgroups: up to sixteens of parts."""
    rng = np.random.default_rng(positions)
    t, lens = grown(rng, H, KVH, hd, [(positions, 5)], dtype, own=2000, max_rows=30000)
    t.grow(rng, lens, [1, 2, 1, 1, 0] if 16 * KVH >= 2 * H else [1, 1, 1, 1, 0], dtype)
    t.attend(rng, dtype)
    t.attend(rng, dtype, scale=0.01)
    t.attend(rng, dtype, size=30.0)


def test_forks_of_forks():
    """Prefixes of several lengths in one group: what all have in common counts."""
    rng = np.random.default_rng(11)
    B = 12
    t = Forked(4, 2, 64, B, 2000, 200, 3000)
    lens = [700] + [0] * (B - 1)
    t.grow(rng, [0] * B, lens)
    for step in range(6):
        alive = [b for b in range(B) if lens[b] > 400]
        lead = [int(rng.choice(alive)) if rng.random() < 0.5 or not lens[b] else b for b in range(B)]
        keep = [int(rng.integers(350, lens[a] + 1)) if a != b else lens[b] for b, a in enumerate(lead)]
        t.fork(lead, keep)
        t.grow(rng, keep, [1] * B)
        t.attend(rng, "f32")
        add = rng.integers(0, 90, B).tolist()
        t.grow(rng, [k + 1 for k in keep], add)
        t.attend(rng, "f32")
        lens = [k + 1 + a for k, a in zip(keep, add)]


@pytest.mark.parametrize("hd", [64, 128])
def test_faint_and_large_pages(hd):
    """Scales that lie far apart on the two sides of a joint, zeros, a dominant key in the prefix or behind it."""
    rng = np.random.default_rng(hd)
    B, KVH = 4, 1
    t = Forked(2, KVH, hd, B, 600, 60, 700)
    t.plan([0] * B, [320, 0, 0, 0])
    k, v = rng.standard_normal((320, KVH, hd)).astype(np.float32), rng.standard_normal((320, KVH, hd)).astype(np.float32)
    v[:64], v[64:128] = 0, v[64:128] * 2.0 ** 40
    k[200] *= 50
    t.append(k, v, "f32")
    t.fork([0] * B, [320] * B)
    t.plan([320] * B, [40] * B)
    k, v = (rng.standard_normal((40 * B, KVH, hd)).astype(np.float32) for _ in range(2))
    v[:40], v[40:80] = v[:40] * 2.0 ** 60, 0
    k[100] *= 60
    t.append(k, v, "f32")
    t.grow(rng, [360] * B, [1] * B)
    t.attend(rng, "f32")
    t.attend(rng, "f32", size=100.0)
    t.attend(rng, "bf16")


@pytest.mark.parametrize("seqs", [40, 1100])
def test_many_sequences_and_no_room(seqs):
    """More joints than a step has room for (their group is attended to as without), more sequences than shared memory holds."""
    rng = np.random.default_rng(seqs)
    t, lens = grown(rng, 16, 1, 64, [(256, seqs)], "bf16", own=3)
    t.grow(rng, lens, [1] * seqs, "bf16")
    t.attend(rng, "bf16")


def test_the_same_bits_every_time():
    rng = np.random.default_rng(13)
    t, lens = grown(rng, 14, 2, 64, [(5000, 40)], "f32", own=600, max_rows=25000)
    t.grow(rng, lens, [1] * t.B)
    x = torch.randn(t.B, 14 * 64, device="cuda")
    outs = [torch.empty_like(x) for _ in range(6)]
    h, a = ints(lens), ints([1] * t.B)
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        if i % 2:
            t.kv.plan(h.data_ptr(), a.data_ptr(), t.B)
        t.kv.attend(0, x.data_ptr(), out.data_ptr(), q4hip.F32, x.stride(0), out.stride(0))
    for out in outs[1:]:
        assert torch.equal(out.view(torch.int32), outs[0].view(torch.int32))


@pytest.mark.parametrize("late", [False, True])
def test_captured(late):
    """A decode step captured before the first fork, or after it, and replayed as sequences grow and trade places."""
    rng = np.random.default_rng(14)
    H, KVH, hd, B, w = 4, 2, 64, 6, 8 * 64
    t = Forked(H, KVH, hd, B, 700, 120, 800)
    t.grow(rng, [0] * B, [400, 350, 0, 0, 0, 0])
    x, out, have, add = torch.randn(B, w, device="cuda"), torch.empty(B, H * hd, device="cuda"), ints([0] * B), ints([1] * B)

    def step(s):
        t.kv.plan(have.data_ptr(), add.data_ptr(), B, stream=s)
        t.kv.append(0, x[:, H * hd:].data_ptr(), x[:, (H + KVH) * hd:].data_ptr(), q4hip.F32, w, w, s)
        t.kv.attend(0, x.data_ptr(), out.data_ptr(), q4hip.F32, w, H * hd, s)

    def capture():
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=torch.cuda.Stream()):
            step(torch.cuda.current_stream().cuda_stream)
        return g

    torch.cuda.synchronize()
    g = None if late else capture()
    lens = [400, 350, 0, 0, 0, 0]
    for lead, keep in [([0, 1, 0, 0, 1, 1], [400, 350, 300, 400, 350, 333]), ([0, 0, 0, 0, 0, 0], None), ([1, 2, 3, 4, 5, 0], None)]:
        keep = keep or [lens[a] for a in lead]
        t.fork(lead, keep)
        g = g or capture()
        lens = keep
        for _ in range(3):
            have.copy_(ints(lens))
            x.copy_(torch.randn(B, w, device="cuda"))
            torch.cuda.synchronize()
            g.replay()
            torch.cuda.synchronize()
            t.have, t.add = lens, [1] * B
            _, _, t.slots, _, t.seq = t.pool.plan(lens, [1] * B, B)
            y = x.cpu().numpy()
            for c, at in ((0, H), (1, H + KVH)):
                t.ref[0][c].append(y[:, at * hd:(at + KVH) * hd].reshape(B, KVH, hd), t.slots)
            t.check_values()
            t.compare(out.double().cpu().numpy().reshape(B, H, hd), y[:, :H * hd].reshape(B, H, hd), "f32")
            t.plan(lens, [1] * B)
            t.attend(rng, "f32")
            lens = [n + 1 for n in lens]


@pytest.mark.parametrize("H,KVH,hd,positions,seqs", [(20, 20, 64, 700, 40), (4, 2, 64, 300, 3)])
def test_by_what_it_saves(monkeypatch, H, KVH, hd, positions, seqs):
    """As a program has it: one case that is worth it, one that is not."""
    monkeypatch.delenv("Q4HIP_KV8_JOINT_SAVES")
    rng = np.random.default_rng(15)
    t, lens = grown(rng, H, KVH, hd, [(positions, seqs)], "f16", max_rows=2000)
    for _ in range(2):
        t.grow(rng, lens, [1] * seqs, "f16")
        t.attend(rng, "f16")
        lens = [n + 1 for n in lens]
