"""What plan and attention launch on a cache that was forked: more than before only while pages may be shared."""
import ctypes

import numpy as np
import pytest
import torch
from torch.profiler import ProfilerActivity, profile

import q4hip
from test_gpu_kv8 import ints
from test_gpu_kv8_fork import Forked
from test_gpu_kv8_joint import join_all  # noqa: F401  (a fixture for all tests)

pytestmark = pytest.mark.gpu


def launches(call):
    """Kernels of the cache that a call launches."""
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CUDA]) as p:
        call(0)
        torch.cuda.synchronize()
    return sum("k_kv8" in e.name for e in p.events())


def captured(call):
    """The same of a graph that holds the call."""
    hip, s = q4hip.lib(), torch.cuda.Stream()
    stream, graph, n = ctypes.c_void_p(s.cuda_stream), ctypes.c_void_p(), ctypes.c_size_t(0)
    assert hip.hipStreamBeginCapture(stream, 2) == 0
    call(s.cuda_stream)
    assert hip.hipStreamEndCapture(stream, ctypes.byref(graph)) == 0
    assert hip.hipGraphGetNodes(graph, None, ctypes.byref(n)) == 0 and hip.hipGraphDestroy(graph) == 0
    return n.value


class Chats:
    """6 sequences of 290 positions and more, which add one."""

    def __init__(self):
        self.rng, self.B, self.hd = np.random.default_rng(1), 6, 64
        self.t = Forked(4, 2, 64, self.B, 700, 150, 2000)
        self.t.grow(self.rng, [0] * self.B, [290 + b for b in range(self.B)])
        self.lens = [290 + b for b in range(self.B)]
        self.x, self.out = torch.randn(self.B, 256, device="cuda"), torch.empty(self.B, 256, device="cuda")
        self.h, self.a = ints(self.lens), ints([1] * self.B)
        torch.cuda.synchronize()

    def plan(self, stream):
        self.t.kv.plan(self.h.data_ptr(), self.a.data_ptr(), self.B, stream=stream)

    def attend(self, stream):
        self.t.kv.attend(0, self.x.data_ptr(), self.out.data_ptr(), q4hip.F32, 256, 256, stream)

    def grow(self):
        self.t.grow(self.rng, self.lens, [1] * self.B)
        self.lens = [n + 1 for n in self.lens]

    def fork(self, source, keep):
        self.t.fork(source, keep)                   # reads the status, too
        self.lens = list(keep)

    def of(self):
        """Launches of the last plan, again, and of its attention."""
        self.h.copy_(ints(self.t.have))
        return launches(self.plan), launches(self.attend)

    def captured(self):
        return captured(self.plan), captured(self.attend)


def test_until_nothing_is_shared():
    c = Chats()
    c.grow()
    before = c.of()
    assert before[1] == 1
    assert c.captured() == before
    c.fork(list(range(c.B)), [280] * c.B)            # cut back: nothing is shared
    c.grow()
    assert c.of() == before and c.captured() == (before[0] + 1, 2)      # a graph may be replayed after other forks
    c.fork([0] * 6, [281] * 6)
    c.grow()
    assert c.of() == (before[0] + 1, 2) and c.t.kv.shared() == (True, 1)
    c.t.attend(c.rng, "f32")
    c.t.plan([282, 0, 0, 0, 0, 0], [0] * 6)         # the others end
    c.t.grow(c.rng, [282, 0, 0, 0, 0, 0], [1, 300, 300, 300, 300, 300])
    c.lens = [283] + [300] * 5
    c.grow()
    assert c.of() == before
    c.t.attend(c.rng, "f32")
    c.fork([0, 0, 2, 3, 4, 5], [270, 284] + [301] * 4)      # and again
    c.grow()
    assert c.of() == (before[0] + 1, 2) and c.t.kv.shared() == (True, 1)
    c.t.attend(c.rng, "f32")


def test_a_fork_that_failed():
    c = Chats()
    c.grow()
    before = c.of()
    f, k = ints([0] * 6), ints([10000] * 6)
    torch.cuda.synchronize()
    with pytest.raises(q4hip.Q4Error):
        c.t.kv.fork(f.data_ptr(), k.data_ptr())
    c.grow()
    assert c.of() == before
    c.t.attend(c.rng, "f32")


def test_without_a_call_that_waits():
    """Fork, plan and attention on a stream: shared pages are attended to together, whatever nobody has asked for."""
    c = Chats()
    c.grow()
    before = c.of()
    s = torch.cuda.Stream()
    f, k = ints([0] * 6), ints([280] * 6)
    torch.cuda.synchronize()
    c.t.kv.fork(f.data_ptr(), k.data_ptr(), 0, s.cuda_stream)
    assert launches(c.attend) == 0                   # no step, nothing to attend to
    c.h.copy_(k)
    assert launches(lambda _: c.plan(s.cuda_stream)) == before[0] + 1
    assert launches(lambda _: c.attend(s.cuda_stream)) == 2
    assert c.t.kv.shared(s.cuda_stream) == (True, 1)


def test_a_captured_fork():
    """The graph may be replayed at any time."""
    c = Chats()
    c.grow()
    before = c.of()
    f, k = ints([0] * 6), ints([280] * 6)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        c.t.kv.fork(f.data_ptr(), k.data_ptr(), 0, torch.cuda.current_stream().cuda_stream)
    assert c.t.kv.shared() == (False, 0)
    assert c.of() == (before[0] + 1, 2)
    c.t.attend(c.rng, "f32")                         # and without a joint
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        c.t.copied(c.t.pool.fork([0] * 6, [280] * 6))
        c.lens = [280] * 6
        for joints in (1, 1):
            c.grow()
            assert c.t.kv.shared() == (True, joints)
            c.t.attend(c.rng, "f32")
