"""Forked sequences of the paged 8-bit cache on the GPU against kv8_fork_ref.py: tables, free pages, codes and scales to the bit,
attention within the bound of kv8_ref.py."""
import ctypes

import numpy as np
import pytest
import torch

import q4hip
from kv8_fork_ref import SharedPool
from test_gpu_kv8 import Both, ints

pytestmark = pytest.mark.gpu


class Forked(Both):
    """Both, with pages that several sequences may hold."""

    def __init__(self, H, KVH, hd, seqs, max_len, pages, max_rows, layers=1):
        super().__init__(H, KVH, hd, seqs, max_len, pages, max_rows, layers)
        self.pool = SharedPool(seqs, max_len, pages)

    def fork(self, source, keep, stream=0):
        f, k = ints(source), ints(keep)
        tables = ints(np.full((self.B, self.pool.W), -7))
        torch.cuda.synchronize()
        self.kv.fork(f.data_ptr(), k.data_ptr(), tables.data_ptr(), stream)
        torch.cuda.synchronize()
        copies = self.pool.fork(source, keep)
        assert copies is not None
        self.copied(copies)
        assert np.array_equal(tables.cpu(), self.pool.table())
        assert self.kv.status() == (0, len(self.pool.stack))
        self.have, self.add, self.slots = list(keep), [0] * self.B, []
        return copies

    def copied(self, copies):
        for layer in self.ref:
            for cache in layer:
                for p, to in copies:
                    cache.codes[to], cache.scales[to] = cache.codes[p], cache.scales[p]

    def grow(self, rng, have, add, dtype="f32"):
        self.plan(have, add)
        for layer in range(self.layers):
            if sum(add):
                self.fill(rng, dtype, layer)

    def refused(self, call, code):
        """A call that changes nothing."""
        before = self.pool.table()
        stack, lens = list(self.pool.stack), list(self.pool.lens)
        with pytest.raises(q4hip.Q4Error) as e:
            call()
        assert e.value.code == code
        assert np.array_equal(before, self.pool.table()) and stack == self.pool.stack and lens == self.pool.lens
        self.have, self.add, self.slots = lens, [0] * self.B, []
        self.check_values()


@pytest.mark.parametrize("hd,KVH,layers,dtype", [(64, 2, 3, "f32"), (128, 1, 1, "bf16"), (128, 3, 2, "f16")])
@pytest.mark.parametrize("keep", [1, 31, 32, 33, 64, 95, 100])
def test_answers_to_one_question(hd, KVH, layers, dtype, keep):
    rng = np.random.default_rng(keep)
    t = Forked(2 * KVH, KVH, hd, 5, 200, 40, 400, layers)
    t.grow(rng, [0] * 5, [100, 0, 40, 0, 0], dtype)
    copies = t.fork([0, 0, 2, 0, 0], [keep, keep, 40, keep, 0])
    assert len(copies) == (2 if keep % 32 else 0)
    for layer in range(layers):
        t.check_values(layer)
    # all go on by themselves
    t.grow(rng, [keep, keep, 40, keep, 0], [3, 50, 1, 1, 2], dtype)
    for layer in range(layers):
        t.check_values(layer)
        t.attend(rng, dtype, layer)
    t.fork([0, 1, 2, 3, 4], [0, 0, 0, keep, 0])
    t.check_values()
    t.plan([0] * 5, [0] * 5, 0)
    assert len(t.pool.stack) == 40


@pytest.mark.parametrize("max_len,pages", [(300, 21), (50000, 21), (300, 5000)])
def test_beams_trade_places(max_len, pages):
    """Every sequence becomes another one, at once, again and again; pages of dropped ones serve the copies."""
    rng = np.random.default_rng(3)
    B = 6
    t = Forked(4, 2, 64, B, max_len, pages, 64, 2)
    t.grow(rng, [0] * B, [50] + [0] * (B - 1))
    lens = t.fork([0] * B, [50] * B) and [50] * B
    for step in range(30):
        t.grow(rng, lens, [1] * B)
        t.attend(rng, "f32", 1)
        lens = [n + 1 for n in lens]
        source = rng.integers(0, B, B).tolist()
        if step % 5 == 0:
            source = [(b + 1) % B for b in range(B)]                 # a cycle
        t.fork(source, [lens[f] for f in source])
        lens = [lens[f] for f in source]
        for layer in range(2):
            t.check_values(layer)


@pytest.mark.parametrize("seqs,max_len", [(3, 64), (70, 200), (700, 90), (1500, 130)])
def test_plans_and_forks_in_turn(seqs, max_len):
    rng = np.random.default_rng(seqs + max_len)
    pages = max(4, seqs * -(-max_len // 32) // 2)
    t = Forked(2, 1, 64, seqs, max_len, pages, seqs * max_len)
    lens = np.zeros(seqs, int)
    plans = forks = failed = 0
    for step in range(14):
        if step % 2:
            source = np.where(rng.random(seqs) < 0.5, np.arange(seqs), rng.integers(0, seqs, seqs))
            keep = np.where(rng.random(seqs) < 0.6, lens[source], rng.integers(0, lens[source] + 1))
            keep[rng.random(seqs) < 0.1] = 0
            saved = t.pool.table(), list(t.pool.stack)
            if t.pool.fork(source.tolist(), keep.tolist()) is None:
                f, k = ints(source), ints(keep)
                torch.cuda.synchronize()
                with pytest.raises(q4hip.Q4Error) as e:
                    t.kv.fork(f.data_ptr(), k.data_ptr())
                assert e.value.code == q4hip.ECONTEXT
                failed += 1
                continue
            t.pool.tables, t.pool.stack, t.pool.lens = [[p for p in r if p >= 0] for r in saved[0].tolist()], saved[1], lens.tolist()
            t.fork(source.tolist(), keep.tolist())
            lens = keep
            forks += 1
        else:
            have = np.where(rng.random(seqs) < 0.1, rng.integers(0, lens + 1), lens)
            have[rng.random(seqs) < 0.15] = 0
            add = np.minimum(rng.integers(0, max_len, seqs) * (rng.random(seqs) < 0.3), max_len - have)
            add[(have < lens) & (have % 32 > 0)] = 0                # not into pages that others may hold
            add[have < lens] *= rng.random(seqs)[have < lens] < 0.2
            free = len(t.pool.stack)
            while (np.maximum(-(-(have + add) // 32) - -(-lens // 32), 0)).sum() > free:
                add = add // 2
                have = np.where(add == 0, np.minimum(have, lens), have)
            rows = int(add.sum())
            held = t.pool.holders()
            blocked = [a and any(held[p] > 1 for p in r[h // 32:]) for r, h, a in zip(t.pool.tables, have, add)]
            add[np.array(blocked, bool)] = 0
            rows = int(add.sum())
            for _ in range(2):                                      # the same plan again
                t.plan(have.tolist(), add.tolist(), rows)
            if rows and rows < 3000:
                t.fill(rng, "f32")
            lens = have + add
            plans += 1
    assert plans == 7 and forks >= 3
    t.plan([0] * seqs, [0] * seqs, 0)
    assert sorted(t.pool.stack) == list(range(pages))


def test_rows_into_a_shared_page():
    """A plan that would write where another sequence reads fails; a fork that cuts back first makes it possible."""
    rng = np.random.default_rng(4)
    t = Forked(2, 1, 64, 3, 300, 30, 300)
    t.grow(rng, [0, 0, 0], [160, 0, 0])
    t.fork([0, 0, 0], [160, 160, 100])
    for have, add in [([160, 50, 100], [1, 1, 1]), ([160, 64, 100], [0, 5, 0]), ([0, 160, 100], [7, 0, 0])]:
        h, a = ints(have), ints(add)
        torch.cuda.synchronize()
        t.refused(lambda: t.kv.plan(h.data_ptr(), a.data_ptr(), 20), q4hip.EINVAL)
        assert t.pool.plan(have, add, 20) is None
    t.plan([160, 50, 100], [0, 0, 0])                  # cut back without rows: fine
    t.check_values()
    t.fork([0, 1, 2], [160, 50, 100])                  # its last page becomes its own
    t.grow(rng, [160, 50, 100], [1, 40, 1])
    t.check_values()
    t.attend(rng, "f32")
    # the last holder may write where others have just gone
    t.plan([0, 90, 101], [0, 0, 0])
    t.grow(rng, [0, 90, 101], [33, 1, 1])
    t.check_values()
    t.attend(rng, "f32")


@pytest.mark.parametrize("max_len", [100, 90000])          # forked by one workgroup, and by many
@pytest.mark.parametrize("source,keep,code", [([0, 3, 2], [5, 5, 5], q4hip.EINVAL), ([0, -1, 2], [5, 5, 0], q4hip.EINVAL),
                                              ([0, 1, 0], [5, 0, 71], q4hip.EINVAL), ([1, 1, 1], [1, 0, 0], q4hip.EINVAL),
                                              ([0, 1, 2], [-1, 0, 0], q4hip.EINVAL), ([0, 0, 2], [70, 70, 40], q4hip.ECONTEXT)])
def test_forks_that_do_not_fit_change_nothing(source, keep, code, max_len):
    rng = np.random.default_rng(5)
    t = Forked(2, 1, 64, 3, max_len, 5, 110)
    t.grow(rng, [0, 0, 0], [70, 0, 40])
    t.pool.plan([70, 0, 40], [0, 0, 0], 0)
    assert t.pool.fork(source, keep) is None
    f, k, out = ints(source), ints(keep), ints(np.full((3, t.pool.W), -7))
    torch.cuda.synchronize()
    t.refused(lambda: t.kv.fork(f.data_ptr(), k.data_ptr(), out.data_ptr()), code)
    assert np.array_equal(out.cpu(), t.pool.table())
    with pytest.raises(q4hip.Q4Error) as e:
        t.kv.status()
    assert e.value.code == code
    t.fork([2, 2, 9], [40, 33, 0])                     # and nothing is left of it
    t.check_values()
    t.grow(rng, [40, 33, 0], [1, 1, 1])
    t.check_values()


def test_the_step_is_over():
    """append and attend do nothing between a fork and the next plan; what a captured step holds, too."""
    rng = np.random.default_rng(6)
    t = Forked(2, 1, 64, 2, 100, 8, 100)
    t.grow(rng, [0, 0], [40, 0])
    x, out = torch.randn(40, 256, device="cuda"), torch.full((40, 128), 7.0, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        s = torch.cuda.current_stream().cuda_stream
        t.kv.append(0, x[:, 128:].data_ptr(), x[:, 192:].data_ptr(), q4hip.F32, 256, 256, s)
        t.kv.attend(0, x.data_ptr(), out.data_ptr(), q4hip.F32, 256, 128, s)
        out.add_(0)
    t.fork([0, 0], [40, 40])
    for _ in range(2):
        g.replay()
        t.kv.append(0, x[:, 128:].data_ptr(), x[:, 192:].data_ptr(), q4hip.F32, 256, 256)
        t.kv.attend(0, x.data_ptr(), out.data_ptr(), q4hip.F32, 256, 128)
        torch.cuda.synchronize()
        assert (out == 7).all()
        t.check_values()


def test_captured_fork_and_plan():
    """A step with a fork in front, captured before the first fork and replayed with other arguments."""
    rng = np.random.default_rng(7)
    H, KVH, hd, B, w = 4, 2, 64, 4, 8 * 64
    t = Forked(H, KVH, hd, B, 400, 40, 400, 2)
    t.grow(rng, [0] * B, [90, 10, 0, 0])
    source, keep, have, add = (ints([0] * B) for _ in range(4))
    tables = ints(np.zeros((B, t.pool.W)))
    x, out = torch.randn(8, w, device="cuda"), torch.full((8, H * hd), 7.0, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        s = torch.cuda.current_stream().cuda_stream
        t.kv.fork(source.data_ptr(), keep.data_ptr(), tables.data_ptr(), s)
        t.kv.plan(have.data_ptr(), add.data_ptr(), 8, stream=s)
        for layer in range(2):
            t.kv.append(layer, x[:, H * hd:].data_ptr(), x[:, (H + KVH) * hd:].data_ptr(), q4hip.F32, w, w, s)
            t.kv.attend(layer, x.data_ptr(), out.data_ptr(), q4hip.F32, w, H * hd, s)
    lens = [90, 10, 0, 0]
    for f, more in [([0, 0, 0, 1], [1, 1, 2, 3]), ([1, 2, 3, 0], [2, 2, 2, 2]), ([3, 3, 3, 3], [1, 0, 0, 1]), ([0, 0, 1, 1], [1, 2, 3, 2])]:
        k = [lens[b] for b in f]
        for buf, a in ((source, f), (keep, k), (have, k), (add, more)):
            buf.copy_(ints(a))
        out.fill_(7.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        t.copied(t.pool.fork(f, k))
        assert np.array_equal(tables.cpu(), t.pool.table())
        n = sum(more)
        t.have, t.add = k, more
        _, _, t.slots, _, t.seq = t.pool.plan(k, more, 8)
        y = x[:n].cpu().numpy()
        for layer in range(2):
            for c, at in ((0, H), (1, H + KVH)):
                t.ref[layer][c].append(y[:, at * hd:(at + KVH) * hd].reshape(n, KVH, hd), t.slots)
            t.check_values(layer)
        assert t.kv.status() == (n, len(t.pool.stack)) and (out[n:] == 7).all()
        t.compare(out[:n].double().cpu().numpy().reshape(n, H, hd), y[:, :H * hd].reshape(n, H, hd), "f32", 1)
        lens = [a + b for a, b in zip(k, more)]


def test_refusals():
    t = Forked(2, 1, 64, 3, 100, 8, 10)
    a, host = ints([0] * 40), np.zeros(40, np.int32)
    torch.cuda.synchronize()
    p = a.data_ptr()
    for args in [(0, p), (p, 0), (host.ctypes.data, p), (p, host.ctypes.data), (p, p, host.ctypes.data), (p + 2, p), (p, p + 1),
                 (p, p + 4 * 38), (p, p, p), (p, p, p + 4), (p, p + 4 * 20, p + 4 * 10)]:
        with pytest.raises(q4hip.Q4Error) as e:
            t.kv.fork(*args)
        assert e.value.code == q4hip.EINVAL, args
    t.kv.fork(p, p)
    assert t.kv.status() == (0, 8)
