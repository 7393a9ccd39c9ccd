"""The paged 8-bit cache on rows whose 16 bytes can be loaded and stored at once, as callers' rows of q|k|v have them (test_gpu_kv8.py's
lie at odd columns): the same references and bounds."""
import numpy as np
import pytest
import torch

from test_gpu_kv8 import LAYOUTS, TYPES, Both

pytestmark = pytest.mark.gpu


class Aligned(Both):
    """Rows of q|k|v, one after the other; `out` likewise."""

    def append(self, k, v, dtype, layer=0):
        typ, t = TYPES[dtype]
        n, w, q = len(self.slots), self.KVH * self.hd, self.H * self.hd
        buf = torch.full((n, q + 2 * w), float("nan"), dtype=t, device="cuda")
        buf[:, q:q + w] = torch.tensor(k.reshape(n, w)).to(t).cuda()
        buf[:, q + w:] = torch.tensor(v.reshape(n, w)).to(t).cuda()
        torch.cuda.synchronize()
        kp, vp = buf[:, q:], buf[:, q + w:]
        assert kp.data_ptr() % 16 == vp.data_ptr() % 16 == buf.stride(0) * buf.element_size() % 16 == 0
        self.kv.append(layer, kp.data_ptr(), vp.data_ptr(), typ, buf.stride(0), buf.stride(0))
        host = buf.float().cpu().numpy()
        self.ref[layer][0].append(host[:, q:q + w].reshape(n, self.KVH, self.hd), self.slots)
        self.ref[layer][1].append(host[:, q + w:].reshape(n, self.KVH, self.hd), self.slots)

    def attend(self, rng, dtype, layer=0, scale=0.0, size=1.0, stream=0):
        typ, t = TYPES[dtype]
        n, w = len(self.slots), self.H * self.hd
        q = torch.tensor(rng.standard_normal((n, w + 16)).astype(np.float32) * size).to(t).cuda()
        out = torch.full((n + 2, w + 8), 7.0, dtype=t, device="cuda")
        torch.cuda.synchronize()
        assert q.data_ptr() % 16 == out.data_ptr() % 16 == q.stride(0) * q.element_size() % 16 == out.stride(0) * out.element_size() % 16 == 0
        self.kv.attend(layer, q.data_ptr(), out.data_ptr(), typ, q.stride(0), out.stride(0), stream, scale)
        torch.cuda.synchronize()
        got = out.double().cpu().numpy()
        assert (got[n:] == 7).all() and (got[:, w:] == 7).all()
        self.compare(got[:n, :w].reshape(n, self.H, self.hd), q[:, :w].float().cpu().numpy().reshape(n, self.H, self.hd),
                     dtype, layer, scale)


@pytest.mark.parametrize("KVH,hd", [(1, 64), (2, 128), (5, 64), (3, 128)])
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_append_runs_of_every_kind(KVH, hd, dtype):
    rng = np.random.default_rng(KVH * hd + 1)
    t = Aligned(KVH, KVH, hd, 4, 300, 40, 700, layers=2)
    lens = [0, 0, 0, 0]
    for add in ([1, 31, 32, 33], [1, 1, 1, 1], [30, 0, 40, 2], [5, 97, 1, 31], [1, 1, 1, 1]):
        t.plan(lens, add)
        for layer in range(2):
            t.fill(rng, dtype, layer, size=float(rng.choice([0.1, 1.0, 30.0])))
        lens = [a + b for a, b in zip(lens, add)]
        for layer in range(2):
            t.check_values(layer)
    t.plan([3, 64, 0, 33], [2, 1, 1, 0])           # cut back: into a page, to its end, to nothing
    t.fill(rng, dtype)
    t.check_values()


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_append_odd_values(dtype):
    """NaN and infinities among rows of a whole page, of a part of one and of one row; the largest numbers of the type."""
    rng = np.random.default_rng(8)
    t = Aligned(2, 2, 128, 3, 100, 12, 200)
    t.plan([0, 0, 0], [64, 40, 1])
    k, v = rng.standard_normal((2, 105, 2, 128)).astype(np.float32)
    k[3, 0, 5], k[70, 1, 0], k[104, 0, 9] = np.nan, np.inf, -np.inf
    v[40, 1, 64], v[103, 0, 127], v[104, 1, 0] = -np.inf, np.nan, np.inf
    v[0, 0, 0] = float(torch.finfo(TYPES[dtype][1]).max) / 2
    t.append(k, v, dtype)
    t.check_values()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("H,KVH,hd", LAYOUTS)
def test_attend_tokens(H, KVH, hd, dtype):
    rng = np.random.default_rng(H * hd + 1)
    have = [0, 31, 32, 33, 0, 250, 1, 700, 95]
    t = Aligned(H, KVH, hd, 9, 800, 60, 1200)
    t.plan([0] * 9, have)
    t.fill(rng, dtype)
    t.plan(have, [1, 1, 1, 1, 0, 1, 0, 1, 1])
    t.fill(rng, dtype)
    t.attend(rng, dtype)
    t.attend(rng, dtype, scale=0.31, size=0.3)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("H,KVH,hd", LAYOUTS)
def test_attend_prompts(H, KVH, hd, dtype):
    rng = np.random.default_rng(H + hd + 1)
    have = [0, 40, 0, 64, 3, 0, 130, 20]
    t = Aligned(H, KVH, hd, 8, 400, 60, 700)
    t.plan([0] * 8, have)
    t.fill(rng, dtype)
    t.plan(have, [2, 17, 65, 64, 130, 1, 33, 5])
    t.fill(rng, dtype)
    t.attend(rng, dtype)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (8, 1, 128)])
def test_attend_long(H, KVH, hd, dtype):
    rng = np.random.default_rng(H + hd + 1)
    have = [9000, 2500]
    t = Aligned(H, KVH, hd, 2, 9100, 400, 12000)
    t.plan([0, 0], have)
    t.fill(rng, dtype)
    t.plan(have, [1, 3])
    t.fill(rng, dtype)
    t.attend(rng, dtype)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("H,KVH,hd,add", [(32, 32, 64, [300, 1, 129, 65, 700, 0, 1500, 2]), (20, 10, 128, [1, 900, 1800, 2, 1200])])
def test_attend_tiles(H, KVH, hd, add, dtype):
    rng = np.random.default_rng(H + 1)
    G = H // KVH
    assert KVH * sum(-(-a * G // 128) if a > max(1, 16 // G) else a > 0 for a in add) >= 640
    have = [int(h) for h in rng.integers(0, 100, len(add))]
    t = Aligned(H, KVH, hd, len(add), 2000, 250, sum(add))
    t.plan([0] * len(add), have)
    t.fill(rng, dtype)
    t.plan(have, add)
    t.fill(rng, dtype)
    t.attend(rng, dtype)
