"""Penalties, biases and masks on logits (q4hip_logits_*) on the GPU.

The header states the operations in fp32 and their order, so results are compared to the bit with numpy's fp32, and with 64 bits
within the bound of those roundings: the penalty's quotient or product, the product with the frequency and its sum, the difference
and the bias' sum round once each, relative to what they give.
"""
import numpy as np
import pytest
import torch

import q4hip

pytestmark = pytest.mark.gpu

TYPES = {"f32": (q4hip.F32, torch.float32), "f16": (q4hip.F16, torch.float16), "bf16": (q4hip.BF16, torch.bfloat16)}


def device(a):
    return torch.from_numpy(np.ascontiguousarray(a).view(np.uint8).reshape(-1).copy()).cuda()


def rules(rng, rows, vocab, history=0, biases=0, masks=0, share=0.5):
    """Random rules of `rows` rows: (params, history, biases, mask words, allowed)."""
    p = np.zeros(rows, q4hip.LOGITS_ROW)
    p["repetition"], p["presence"], p["frequency"] = rng.uniform(0.7, 1.6, rows), rng.uniform(-1, 1, rows), rng.uniform(0, 1, rows)
    n = rng.integers(0, history + 1, rows)
    p["history_end"] = np.cumsum(n)
    p["history_begin"] = p["history_end"] - n
    h = np.minimum(vocab * rng.random(int(n.sum())) ** 3, vocab - 1).astype(np.int32)
    n = rng.integers(0, biases + 1, rows)
    p["bias_end"] = np.cumsum(n)
    p["bias_begin"] = p["bias_end"] - n
    b = np.zeros(int(n.sum()), q4hip.LOGITS_BIAS)
    b["token"], b["value"] = rng.integers(0, vocab, len(b)), 3 * rng.standard_normal(len(b))
    allowed = rng.random((masks, vocab)) < share
    words = -(-vocab // 32)
    padded = np.zeros((masks, words * 32), bool)
    padded[:, :vocab] = allowed
    padded[:, vocab:] = rng.random((masks, words * 32 - vocab)) < 0.5       # bits behind the vocabulary
    mask = np.packbits(padded, axis=1, bitorder="little").view(np.uint32) if masks else np.zeros((0, words), np.uint32)
    p["mask"] = rng.integers(-1, masks, rows) if masks else -1
    return p, h, b, mask, allowed


def plain(x, p, h, b, allowed, wide=np.float32):
    """(values, size of what was rounded, best) of rows x in `wide`."""
    y, size = x.astype(wide), np.abs(x.astype(np.float64))
    with np.errstate(all="ignore"):
        for r, q in enumerate(p):
            tokens = h[max(q["history_begin"], 0):max(q["history_end"], 0)]
            tokens, c = np.unique(tokens[(tokens >= 0) & (tokens < x.shape[1])], return_counts=True)
            v = y[r, tokens]
            rep, fre, pre = wide(q["repetition"]), wide(q["frequency"]), wide(q["presence"])
            v = np.where(v > 0, v / rep, v * rep)
            t = fre * c.astype(wide)
            y[r, tokens] = v - (t + pre)
            size[r, tokens] = 3 * np.abs(v) + 3 * np.abs(t) + 2 * abs(pre)
            for token, value in b[max(q["bias_begin"], 0):max(q["bias_end"], 0)].tolist() and dict(
                    b[max(q["bias_begin"], 0):max(q["bias_end"], 0)].tolist()).items():
                if 0 <= token < x.shape[1]:
                    y[r, token] += wide(value)
                    size[r, token] += abs(float(y[r, token])) + abs(value)
            if 0 <= q["mask"] < len(allowed):
                y[r, ~allowed[q["mask"]]] = -np.inf
    z = np.where(np.isnan(y), -np.inf, y)
    best = np.where(z.max(1) > -np.inf, z.argmax(1), -1)
    return y, size, best


class Case:
    def __init__(self, rng, dtype, rows, vocab, pad=0, **kw):
        self.typ, self.t = TYPES[dtype]
        self.rows, self.vocab, self.dtype = rows, vocab, dtype
        self.lg = q4hip.Logits(vocab, rows)
        x = torch.tensor(4 * rng.standard_normal((rows, vocab + pad)).astype(np.float32)).to(self.t)
        self.x = x.cuda()
        self.set(*rules(rng, rows, vocab, **kw))

    def set(self, p, h, b, mask, allowed):
        self.rules = p, h, b, allowed
        self.sizes = len(h), len(b), len(mask)
        self.p, self.h, self.b, self.mask = (device(a) for a in (p, h, b, mask))

    def run(self, y=None, best=True, stream=0, x=None):
        x = self.x if x is None else x
        y = torch.full_like(x, 7.0) if y is None else y
        self.best = torch.full((self.rows,), -7, dtype=torch.int32, device="cuda")
        torch.cuda.synchronize()
        self.lg.run(x.data_ptr(), y.data_ptr(), self.typ, x.stride(0), y.stride(0), self.rows, self.p.data_ptr(), self.h.data_ptr(),
                    self.sizes[0], self.b.data_ptr(), self.sizes[1], self.mask.data_ptr(), self.sizes[2],
                    self.best.data_ptr() if best else 0, stream)
        torch.cuda.synchronize()
        return y

    def check(self, y, best=True, x=None):
        x = (self.x if x is None else x)[:, :self.vocab].float().cpu().numpy()
        want, _, top = plain(x, *self.rules)
        got = y[:, :self.vocab]
        rounded = torch.from_numpy(want).to(self.t)
        same = (got.cpu() == rounded) | (got.cpu().isnan() & rounded.isnan())
        assert same.all(), torch.nonzero(~same)[:5]
        if best:
            assert np.array_equal(self.best.cpu().numpy(), top)
        exact, size, _ = plain(x, *self.rules, wide=np.float64)
        fine = np.isfinite(exact) & np.isfinite(size) & (np.abs(exact) < torch.finfo(self.t).max)
        err = np.abs(got.double().cpu().numpy()[fine] - exact[fine])
        bound = size[fine] * 2.0 ** -23
        bound = bound + (np.abs(exact[fine]) + bound) * torch.finfo(self.t).eps / 2 + 2.0 ** -25
        assert (err <= bound).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("rows,vocab,pad,history,biases,masks", [
    (1, 1, 0, 3, 2, 1), (1, 31, 0, 40, 5, 2), (3, 33, 0, 0, 0, 0), (5, 1000, 0, 300, 20, 3), (2, 2048, 0, 64, 0, 1), (2, 2049, 7, 64, 9, 2),
    (4, 16383, 0, 5000, 100, 2), (1, 151936, 0, 300, 8, 0), (7, 151936, 0, 4000, 40, 4), (40, 32768, 8, 700, 33, 3), (300, 16390, 2, 90, 5, 3),
    (64, 65537, 0, 200, 3, 2), (600, 77, 3, 10, 4, 5)])
def test_rows(dtype, rows, vocab, pad, history, biases, masks):
    rng = np.random.default_rng(rows + vocab)
    c = Case(rng, dtype, rows, vocab, pad, history=history, biases=biases, masks=masks)
    for _ in range(2):                         # the workspace is as it was
        y = c.run()
        c.check(y)
        assert (y[:, vocab:] == 7).all()
    before = c.x.clone()
    z = c.run(y=c.x)                           # in place
    assert torch.equal(z[:, :vocab].nan_to_num(9.0), y[:, :vocab].nan_to_num(9.0)) and torch.equal(z[:, vocab:], before[:, vocab:])
    c.x = before
    assert torch.equal(c.run(best=False)[:, :vocab].nan_to_num(9.0), y[:, :vocab].nan_to_num(9.0))
    assert (c.best == -7).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("vocab", [5, 5000, 70000])
def test_rows_without_a_choice(dtype, vocab):
    """Masks that allow nothing, one token, the last one; rows of -inf, NaN, ties, both zeros."""
    rng = np.random.default_rng(vocab)
    c = Case(rng, dtype, 8, vocab)
    p, h, b, _, _ = rules(rng, 8, vocab)
    allowed = np.zeros((3, vocab), bool)
    allowed[1, vocab // 2] = allowed[2, vocab - 1] = True
    padded = np.zeros((3, -(-vocab // 32) * 32), bool)
    padded[:, :vocab] = allowed
    p["mask"] = [0, 1, 2, -1, -1, -1, -1, 3]                       # 3: there is none, as -1
    c.set(p, h, b, np.packbits(padded, axis=1, bitorder="little").view(np.uint32), allowed)
    c.x[3] = -float("inf")
    c.x[4] = float("nan")
    c.x[4, vocab - 2] = -3.0
    c.x[5] = 1.5
    c.x[6] = -0.0
    c.x[6, vocab // 3 + 1] = 0.0
    c.x[7, vocab - 1] = float("inf")
    c.check(c.run())
    assert c.best.tolist() == [-1, vocab // 2, vocab - 1, -1, vocab - 2, 0, 0, vocab - 1]


def test_lists_of_every_kind():
    """Entries beyond the vocabulary, lists out of order or beyond their end, the same token many times, shared lists."""
    rng = np.random.default_rng(5)
    vocab = 3000
    c = Case(rng, "f32", 7, vocab)
    p = np.zeros(7, q4hip.LOGITS_ROW)
    p["repetition"], p["presence"], p["frequency"], p["mask"] = 1.25, 0.5, 0.125, -1
    h = rng.integers(0, vocab, 500).astype(np.int32)
    h[:100] = 17
    h[100:110] = [-1, vocab, 2 ** 31 - 1, -2 ** 31, vocab - 1, 0, 0, -5, 17, 17]
    b = np.zeros(60, q4hip.LOGITS_BIAS)
    b["token"], b["value"] = rng.integers(0, 10, 60), rng.standard_normal(60)
    b["token"][:4] = [-1, vocab, -2 ** 31, 2 ** 31 - 1]
    p["history_begin"], p["history_end"] = [0, 0, 500, 300, -5, 499, 7], [500, 110, 0, 2 ** 31 - 1, 400, 500, 7]
    p["bias_begin"], p["bias_end"] = [0, 0, 60, 50, -2 ** 31, 59, 5], [60, 10, 0, 2 ** 31 - 1, 30, 60, 5]
    words = np.zeros((0, -(-vocab // 32)), np.uint32)
    c.set(p, h, b, words, np.zeros((0, vocab), bool))
    c.check(c.run())


def test_infinities():
    """+inf and -inf through penalties and biases; a bias of -inf forbids, one of NaN is passed on."""
    rng = np.random.default_rng(6)
    c = Case(rng, "f32", 2, 2500)
    p = np.zeros(2, q4hip.LOGITS_ROW)
    p["repetition"], p["frequency"], p["mask"] = 2.0, 1.0, -1
    p["history_end"], p["bias_end"] = 6, 5
    c.x[:, :3] = torch.tensor([float("inf"), -float("inf"), float("nan")])
    b = np.zeros(5, q4hip.LOGITS_BIAS)
    b["token"], b["value"] = [1, 5, 6, 0, 7], [np.inf, -np.inf, np.nan, -np.inf, 1e38]
    c.set(p, np.array([0, 1, 2, 3, 5, 6], np.int32), b, np.zeros((0, 79), np.uint32), np.zeros((0, 2500), bool))
    y = c.run()
    c.check(y)
    assert y[0, :3].isnan().all() and y[0, 5] == -float("inf") and y[0, 6].isnan() and c.best[0] == 7


def test_captured():
    """A graph replayed while logits, lists and rules change in place."""
    rng = np.random.default_rng(8)
    c = Case(rng, "bf16", 5, 20000, history=400, biases=10, masks=2)
    y, best = torch.empty_like(c.x), torch.empty(5, dtype=torch.int32, device="cuda")
    room = torch.zeros(4096 * 4, dtype=torch.uint8, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        c.lg.run(c.x.data_ptr(), y.data_ptr(), c.typ, 20000, 20000, 5, c.p.data_ptr(), room.data_ptr(), 4096, c.b.data_ptr(), len(c.rules[2]),
                 c.mask.data_ptr(), 2, best.data_ptr(), torch.cuda.current_stream().cuda_stream)
    for i in range(4):
        p, h, _, _, _ = rules(rng, 5, 20000, 300 + 200 * i)
        p["bias_begin"], p["bias_end"], p["mask"] = c.rules[0]["bias_begin"], c.rules[0]["bias_end"], rng.integers(-1, 2, 5)
        c.rules = p, h, c.rules[2], c.rules[3]
        c.p.copy_(device(p))
        room[:len(h) * 4] = device(h)
        c.x.copy_(4 * torch.randn(5, 20000, device="cuda"))
        y.fill_(7.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        c.best = best
        c.check(y)


def test_refusals():
    rng = np.random.default_rng(9)
    c = Case(rng, "f32", 4, 1000, history=30, biases=5, masks=2)
    y, host = torch.empty_like(c.x), np.zeros(5000, np.float32)
    c.lg.run(c.x.data_ptr(), y.data_ptr(), 0, 1000, 1000, 4, c.p.data_ptr())
    good = dict(x=c.x.data_ptr(), y=y.data_ptr(), dtype=q4hip.F32, x_stride=1000, y_stride=1000, rows=4, params=c.p.data_ptr(),
                history=c.h.data_ptr(), history_n=c.sizes[0], biases=c.b.data_ptr(), biases_n=c.sizes[1], mask=c.mask.data_ptr(), mask_rows=2)
    for change, code in [(dict(x=0), q4hip.EINVAL), (dict(params=0), q4hip.EINVAL), (dict(x=host.ctypes.data), q4hip.EINVAL),
                         (dict(params=host.ctypes.data), q4hip.EINVAL), (dict(history=host.ctypes.data), q4hip.EINVAL),
                         (dict(best=host.ctypes.data), q4hip.EINVAL), (dict(rows=5), q4hip.EINVAL), (dict(rows=-1), q4hip.EINVAL),
                         (dict(dtype=2), q4hip.ETYPE), (dict(x_stride=999), q4hip.EINVAL), (dict(y=c.x.data_ptr() + 4), q4hip.EINVAL),
                         (dict(history_n=-1), q4hip.EINVAL), (dict(history_n=10 ** 7), q4hip.EINVAL), (dict(history=0), q4hip.EINVAL),
                         (dict(mask_rows=10 ** 7), q4hip.EINVAL), (dict(mask=0), q4hip.EINVAL), (dict(biases_n=2 ** 31), q4hip.EINVAL),
                         (dict(params=c.p.data_ptr() + 2), q4hip.EINVAL), (dict(best=y.data_ptr()), q4hip.EINVAL),
                         (dict(best=c.x.data_ptr() + 64), q4hip.EINVAL), (dict(best=c.p.data_ptr()), q4hip.EINVAL),
                         (dict(history=y.data_ptr(), history_n=10), q4hip.EINVAL)]:
        with pytest.raises(q4hip.Q4Error) as e:
            c.lg.run(**{**good, **change})
        assert e.value.code == code, change
    c.lg.run(**{**good, "rows": 0})
