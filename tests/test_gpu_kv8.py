"""The paged 8-bit K/V cache (q4hip_kv8_*) on the GPU against kv8_ref.py: whole numbers, codes and scales to the bit,
attention within the bound that kv8_ref.py derives."""
import numpy as np
import pytest
import torch

import kv8_ref
import q4hip

pytestmark = pytest.mark.gpu

TYPES = {"f32": (q4hip.F32, torch.float32), "f16": (q4hip.F16, torch.float16), "bf16": (q4hip.BF16, torch.bfloat16)}
HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def ints(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


class Both:
    """The library's cache and the plain one, fed the same calls."""

    def __init__(self, H, KVH, hd, seqs, max_len, pages, max_rows, layers=1):
        self.H, self.KVH, self.hd, self.B, self.layers = H, KVH, hd, seqs, layers
        self.kv = q4hip.Kv8(layers, H, KVH, hd, seqs, max_len, pages, max_rows)
        self.pool = kv8_ref.Pool(seqs, max_len, pages)
        self.ref = [[kv8_ref.Cache(pages, KVH, hd) for _ in range(2)] for _ in range(layers)]
        self.max_rows = max_rows

    def plan(self, have, add, rows=None, stream=0):
        rows = sum(add) if rows is None else rows
        h, a = ints(have), ints(add)
        W = self.pool.W
        got = {"starts": ints(np.full(self.B + 1, -7)), "positions": ints(np.full(rows + 3, -7)), "slots": ints(np.full(rows + 3, -7)),
               "tables": ints(np.full((self.B, W), -7))}
        torch.cuda.synchronize()
        self.kv.plan(h.data_ptr(), a.data_ptr(), rows, got["starts"].data_ptr(), got["positions"].data_ptr(),
                     got["slots"].data_ptr(), got["tables"].data_ptr(), stream)
        torch.cuda.synchronize()
        self.have, self.add = list(have), list(add)
        starts, pos, slots, tables, self.seq = want = self.pool.plan(have, add, rows)
        n = len(pos)
        assert np.array_equal(got["starts"].cpu(), starts)
        assert np.array_equal(got["tables"].cpu(), tables)
        for name, w in (("positions", pos), ("slots", slots)):
            g = got[name].cpu().numpy()
            assert np.array_equal(g[:n], w) and (g[n:] == -7).all(), name
        self.slots = slots
        assert self.kv.status() == (n, len(self.pool.stack))
        return want

    def append(self, k, v, dtype, layer=0):
        """k, v: [n][KVH][hd] float arrays; rows lie in a wider buffer."""
        typ, t = TYPES[dtype]
        n, w = len(self.slots), self.KVH * self.hd
        buf = torch.full((n, 2 * w + 5), float("nan"), dtype=t, device="cuda")
        buf[:, 2:2 + w] = torch.tensor(k.reshape(n, w)).to(t).cuda()
        buf[:, 3 + w:3 + 2 * w] = torch.tensor(v.reshape(n, w)).to(t).cuda()
        torch.cuda.synchronize()
        kp, vp = buf[:, 2:], buf[:, 3 + w:]
        self.kv.append(layer, kp.data_ptr(), vp.data_ptr(), typ, buf.stride(0), buf.stride(0))
        host = buf.float().cpu().numpy()
        self.ref[layer][0].append(host[:, 2:2 + w].reshape(n, self.KVH, self.hd), self.slots)
        self.ref[layer][1].append(host[:, 3 + w:3 + 2 * w].reshape(n, self.KVH, self.hd), self.slots)

    def fill(self, rng, dtype, layer=0, size=1.0):
        shape = (len(self.slots), self.KVH, self.hd)
        self.append(rng.standard_normal(shape).astype(np.float32) * size, rng.standard_normal(shape).astype(np.float32), dtype, layer)

    def check_values(self, layer=0):
        """Every position of every sequence, to the bit."""
        lens = [h + a for h, a in zip(self.have, self.add)]
        seq = np.repeat(np.arange(self.B), lens)
        pos = np.concatenate([np.arange(n) for n in lens]).astype(int)
        n = len(seq)
        if not n:
            return
        s, p = ints(seq), ints(pos)
        k, v = (torch.full((n, self.KVH, self.hd), 7.0, device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        self.kv.read(layer, s.data_ptr(), p.data_ptr(), n, k.data_ptr(), v.data_ptr())
        for got, cache in ((k, self.ref[layer][0]), (v, self.ref[layer][1])):
            want = np.concatenate([cache.values(self.pool.tables[b], n) for b, n in enumerate(lens) if n])
            assert np.array_equal(got.cpu().numpy(), want)

    def attend(self, rng, dtype, layer=0, scale=0.0, size=1.0, stream=0):
        typ, t = TYPES[dtype]
        n, w = len(self.slots), self.H * self.hd
        q = torch.tensor(rng.standard_normal((n, w + 3)).astype(np.float32) * size).to(t).cuda()
        out = torch.full((n + 2, w + 1), 7.0, dtype=t, device="cuda")
        torch.cuda.synchronize()
        self.kv.attend(layer, q[:, 1:].data_ptr(), out.data_ptr(), typ, q.stride(0), out.stride(0), stream, scale)
        torch.cuda.synchronize()
        got = out.double().cpu().numpy()
        assert (got[n:] == 7).all() and (got[:, w] == 7).all()          # rows and columns behind are as they were
        self.compare(got[:n, :w].reshape(n, self.H, self.hd), q[:, 1:1 + w].float().cpu().numpy().reshape(n, self.H, self.hd),
                     dtype, layer, scale)
        return out[:n, :w].clone()

    def compare(self, got, q, dtype, layer=0, scale=0.0):
        at = 0
        for b, (h, a) in enumerate(zip(self.have, self.add)):
            if a:
                K, V = (c.values(self.pool.tables[b], h + a) for c in self.ref[layer])
                ks, vs = (c.scale_of(self.pool.tables[b], h + a) for c in self.ref[layer])
                want, bound = kv8_ref.attend(q[at:at + a], K, V, ks, vs, h, scale or self.hd ** -0.5, HALF[dtype])
                err = np.abs(got[at:at + a] - want)
                assert (err <= bound).all(), (b, h, a, float((err / np.maximum(bound, 1e-300)).max()))
            at += a


# ---------------------------------------------------------------------------- plan

@pytest.mark.parametrize("seqs,max_len", [(1, 1), (1, 500), (3, 64), (70, 200), (700, 90), (1024, 40), (1500, 130)])
def test_plan_follows_the_stack(seqs, max_len):
    rng = np.random.default_rng(seqs + max_len)
    W = -(-max_len // 32)
    pages = max(1, seqs * W * 2 // 3)
    t = Both(2, 1, 64, seqs, max_len, pages, seqs * max_len)
    lens = np.zeros(seqs, int)
    done = 0
    while done < 6:
        have = np.where(rng.random(seqs) < 0.2, rng.integers(0, lens + 1), lens)         # some are cut back
        have[rng.random(seqs) < 0.15] = 0
        add = np.minimum(rng.integers(0, max_len, seqs) * (rng.random(seqs) < 0.6), max_len - have)
        if sum(-(-(have + add) // 32)) > pages:
            add[:] = 0
        for _ in range(2):                                                              # the same plan again
            t.plan(have.tolist(), add.tolist(), int(add.sum()) + int(rng.integers(0, 1 + seqs * max_len - add.sum())))
        lens = have + add
        done += 1
    t.plan([0] * seqs, [0] * seqs, 0)
    assert len(t.pool.stack) == pages


@pytest.mark.parametrize("have,add,rows,code", [([3, -1], [1, 1], 2, q4hip.EINVAL), ([3, 1], [1, -1], 2, q4hip.EINVAL),
                                                ([100, 1], [1, 1], 2, q4hip.ECONTEXT), ([0, 2 ** 31 - 1], [1, 2 ** 31 - 1], 2, q4hip.ECONTEXT),
                                                ([0, 0], [4, 5], 8, q4hip.EINVAL), ([90, 60], [1, 1], 2, q4hip.ECONTEXT)])
def test_plan_that_does_not_fit_changes_nothing(have, add, rows, code):
    rng = np.random.default_rng(1)
    t = Both(2, 2, 64, 2, 100, 4, 50)
    t.plan([0, 0], [40, 10])
    t.fill(rng, "f32")
    before = t.kv.status()[1]
    h, a = ints(have), ints(add)
    starts, pos = ints([7] * 3), ints([7] * 50)
    torch.cuda.synchronize()
    for stream in (0, torch.cuda.Stream()):
        if stream:
            t.kv.plan(h.data_ptr(), a.data_ptr(), rows, starts.data_ptr(), pos.data_ptr(), stream=stream.cuda_stream)
            with pytest.raises(q4hip.Q4Error) as e:
                t.kv.status(stream.cuda_stream)
        else:
            with pytest.raises(q4hip.Q4Error) as e:
                t.kv.plan(h.data_ptr(), a.data_ptr(), rows, starts.data_ptr(), pos.data_ptr())
        assert e.value.code == code
        assert starts.tolist() == [0, 0, 0] and set(pos.tolist()) == {7}
        x = torch.full((rows, 128), 9.0, device="cuda")
        out = torch.full((rows, 128), 7.0, device="cuda")
        torch.cuda.synchronize()
        t.kv.append(0, x.data_ptr(), x.data_ptr(), q4hip.F32, 128, 128)
        t.kv.attend(0, x.data_ptr(), out.data_ptr(), q4hip.F32, 128, 128)
        assert (out == 7).all()
    t.plan([40, 10], [0, 0])                       # the next plan starts from what there was
    assert t.kv.status()[1] == before
    t.check_values()


# ---------------------------------------------------------------------------- append

@pytest.mark.parametrize("KVH,hd", [(1, 64), (2, 128), (5, 64), (3, 128)])
@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_append_runs_of_every_kind(KVH, hd, dtype):
    rng = np.random.default_rng(KVH * hd)
    t = Both(KVH, KVH, hd, 4, 300, 40, 700, layers=2)
    lens = [0, 0, 0, 0]
    for add in ([1, 31, 32, 33], [1, 1, 1, 1], [30, 0, 40, 2], [5, 97, 1, 31], [1, 1, 1, 1]):
        t.plan(lens, add)
        for layer in range(2):
            t.fill(rng, dtype, layer, size=float(rng.choice([0.1, 1.0, 30.0])))
        lens = [a + b for a, b in zip(lens, add)]
        for layer in range(2):
            t.check_values(layer)
    lens = [3, 64, 0, 33]                          # cut back: into a page, to its end, to nothing
    t.plan(lens, [2, 1, 1, 0])
    t.fill(rng, dtype)
    t.check_values()


def test_append_scales_at_their_limits():
    """Zeros, the smallest and largest numbers, growth by many doublings, ties of the halving, NaN and infinities."""
    t = Both(1, 1, 64, 1, 200, 8, 200)
    rng = np.random.default_rng(5)
    rows = []
    for size in (0.0, 0.0, 1e-45, 1e-42, 1e-38, 1e-30, 1.0, 1.0, 127.0, 127.0 * 2, 127.0 * 2 + 1, 1e10, 3.0e38, 1.0):
        x = rng.uniform(-1, 1, 64).astype(np.float32) * np.float32(size)
        x[3] = size
        rows.append(x)
    odd = rows[6].copy()
    odd[:4] = [np.nan, np.inf, -np.inf, 0.5]
    rows += [odd, np.full(64, np.nan, np.float32), np.full(64, np.inf, np.float32)]
    one = np.arange(-63, 1).astype(np.float32)      # codes 127 / 63 * n, later halved: ties among them
    rows += [one, one * 2, one * 4]
    at = 0
    for x in rows:
        t.plan([at], [1])
        t.append(x.reshape(1, 1, 64), -x.reshape(1, 1, 64)[..., ::-1].copy(), "f32")
        t.check_values()
        at += 1
    for first in (np.full(64, np.nan, np.float32), np.zeros(64, np.float32), np.full(64, -np.inf, np.float32), odd):
        t.plan([0], [0])
        t.plan([0], [1])
        t.append(first.reshape(1, 1, 64), first.reshape(1, 1, 64), "f32")
        t.check_values()
        t.plan([1], [1])
        t.append(one.reshape(1, 1, 64), one.reshape(1, 1, 64), "f32")
        t.check_values()


def test_read_of_what_is_not_there():
    t = Both(2, 2, 64, 2, 100, 8, 64)
    t.plan([0, 0], [40, 0])
    t.fill(np.random.default_rng(0), "f32")
    seq, pos = ints([0, 0, 1, -1, 2, 0, 0]), ints([39, 40, 0, 0, 0, -1, 2 ** 31 - 1])
    k, v = (torch.full((7, 2, 64), 7.0, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    t.kv.read(0, seq.data_ptr(), pos.data_ptr(), 7, k.data_ptr(), v.data_ptr())
    assert (k[1:] == 0).all() and (v[1:] == 0).all()
    assert np.array_equal(k[0].cpu().numpy(), t.ref[0][0].values(t.pool.tables[0], 40)[39])


# ---------------------------------------------------------------------------- attend

LAYOUTS = [(14, 2, 64), (12, 2, 128), (5, 5, 64), (8, 1, 128), (33, 1, 64), (32, 8, 128), (3, 3, 128)]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("H,KVH,hd", LAYOUTS)
def test_attend_tokens(H, KVH, hd, dtype):
    """One row of each of 9 sequences, from one position on; two hold none and add none."""
    rng = np.random.default_rng(H * hd)
    have = [0, 31, 32, 33, 0, 250, 1, 700, 95]
    t = Both(H, KVH, hd, 9, 800, 60, 1200)
    t.plan([0] * 9, have)
    t.fill(rng, dtype)
    add = [1, 1, 1, 1, 0, 1, 0, 1, 1]
    t.plan(have, add)
    t.fill(rng, dtype)
    t.attend(rng, dtype)
    t.attend(rng, dtype, scale=0.31, size=0.3)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("H,KVH,hd", LAYOUTS)
def test_attend_prompts(H, KVH, hd, dtype):
    """Prompts of many lengths beside tokens, from the start and behind other positions."""
    rng = np.random.default_rng(H + hd)
    have = [0, 40, 0, 64, 3, 0, 130, 20]
    t = Both(H, KVH, hd, 8, 400, 60, 700)
    t.plan([0] * 8, have)
    t.fill(rng, dtype)
    t.plan(have, [2, 17, 65, 64, 130, 1, 33, 5])
    t.fill(rng, dtype)
    t.attend(rng, dtype)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (8, 1, 128)])
def test_attend_long(H, KVH, hd, dtype):
    """Positions enough that the work on one row is shared."""
    rng = np.random.default_rng(H + hd)
    have = [9000, 2500]
    t = Both(H, KVH, hd, 2, 9100, 400, 12000)
    t.plan([0, 0], have)
    t.fill(rng, dtype)
    t.plan(have, [1, 3])
    t.fill(rng, dtype)
    t.attend(rng, dtype)
    t.attend(rng, dtype, size=4.0)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("H,KVH,hd,add", [(32, 32, 64, [300, 1, 129, 65, 700, 0, 1500, 2]), (44, 11, 64, [200, 33, 1000, 1, 700]),
                                          (20, 10, 128, [1, 900, 1800, 2, 1200]), (99, 3, 64, [500, 1, 330, 40])])
def test_attend_tiles(H, KVH, hd, add, dtype):
    """Rows enough for tiles (kKv8MinTiles workgroups), of prompts behind other positions and beside tokens."""
    rng = np.random.default_rng(H)
    G = H // KVH
    assert KVH * sum(-(-a * G // 128) if a > max(1, 16 // G) else a > 0 for a in add) >= 640
    have = [int(h) for h in rng.integers(0, 100, len(add))]
    t = Both(H, KVH, hd, len(add), 2000, 250, sum(add))
    t.plan([0] * len(add), have)
    t.fill(rng, dtype)
    t.plan(have, add)
    t.fill(rng, dtype)
    t.attend(rng, dtype)


def test_attend_many_sequences_and_rows():
    """More sequences than the plan's shared memory holds; lists that are filled by a second launch."""
    rng = np.random.default_rng(3)
    t = Both(4, 2, 64, 1300, 100, 4000, 40000)
    have = rng.integers(0, 60, 1300)
    have[::7] = 0
    t.plan([0] * 1300, have.tolist())
    t.fill(rng, "f32")
    add = np.where(rng.random(1300) < 0.2, 0, 1)
    add[5], add[1111] = 40, 33
    t.plan(have.tolist(), add.tolist())
    t.fill(rng, "f32")
    t.check_values()
    t.attend(rng, "f32")
    t = Both(2, 1, 64, 2, 9000, 400, 9000)
    t.plan([0, 0], [8600, 100])
    t.fill(rng, "bf16")
    t.check_values()
    t.plan([300, 100], [50, 7])
    t.fill(rng, "bf16")
    t.attend(rng, "bf16")


def test_attend_is_the_same_every_time():
    rng = np.random.default_rng(2)
    t = Both(14, 2, 64, 3, 5000, 400, 9000)
    t.plan([0] * 3, [4000, 100, 3000])
    t.fill(rng, "f32")
    t.plan([4000, 100, 3000], [1, 90, 1])
    t.fill(rng, "f32")
    got = [t.attend(np.random.default_rng(9), "f32") for _ in range(4)]
    assert all(torch.equal(g, got[0]) for g in got)


@pytest.mark.parametrize("H,KVH,hd", [(14, 2, 64), (32, 8, 128), (20, 20, 64)])
def test_fp16_tokens_are_as_good_as_their_rounding(H, KVH, hd):
    """Weights in one fp16 number add an error of the size of the output's own rounding where many positions count alike, which makes
    the root of the mean square 1.4 times that of the rounding alone.  Two numbers add 2^-22 relative to the weights, and the
    scores' fp32 rounding less than 2^-18: nothing of 2^-12.  1.1 leaves room for the 2,000 values' chance."""
    rng = np.random.default_rng(15)
    t = Both(H, KVH, hd, 2, 3100, 200, 4000)
    t.plan([0, 0], [3000, 700])
    t.fill(rng, "f16")
    t.plan([3000, 700], [1, 1])
    t.fill(rng, "f16")
    w = H * hd
    q = (0.1 * torch.randn(2, w, generator=torch.Generator().manual_seed(3))).half().cuda()
    out = torch.zeros(2, w, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    t.kv.attend(0, q.data_ptr(), out.data_ptr(), q4hip.F16, w, w)
    got, err, rounding = out.double().cpu().numpy().reshape(2, H, hd), 0.0, 0.0
    for b, n in enumerate((3001, 701)):
        K, V = (c.values(t.pool.tables[b], n) for c in t.ref[0])
        ks, vs = (c.scale_of(t.pool.tables[b], n) for c in t.ref[0])
        want = kv8_ref.attend(q[b:b + 1].float().cpu().numpy().reshape(1, H, hd), K, V, ks, vs, n - 1, hd ** -0.5, HALF["f16"])[0][0]
        err += np.square(got[b] - want).sum()
        rounding += np.square(want.astype(np.float16).astype(np.float64) - want).sum()
    assert err < 1.1 ** 2 * rounding


@pytest.mark.parametrize("H,KVH,hd,have,add", [(20, 20, 64, 12000, 4100), (1, 1, 64, 16000, 40)])
def test_prompts_behind_a_long_text_are_nearly_as_good_as_their_rounding(H, KVH, hd, have, add):
    """fp16 rows whose positions all count alike, on columns of different size, where codes cancel most.  Weights in one fp16
    number add an error of at most 2^-11 / sqrt(3) of a weight in the root of the mean square (all of them just above a power of
    two), as the outputs' own rounding has it: with random signs sqrt(2) to sqrt(1 + 2) of the rounding alone, whose values lie
    anywhere between two powers (ln 2 * 3 / 2 of that square).  The fp32 sums of code + 128 over 2,048 positions add
    sqrt(64) 2^-25 * 128 * 2048 / (sqrt(2048) * 12) of a sum of codes of 12: 1.2e-4, half of the rounding.  So below
    sqrt(3 + 1 / 4) = 1.8; the sums over all 16,000 would be 7 to 8 times the 1.2e-4."""
    rng = np.random.default_rng(16)
    t = Both(H, KVH, hd, 1, have + add, 520, have + add)
    cols = np.exp(0.5 * rng.standard_normal((1, KVH, hd))).astype(np.float32)
    for plan in (([0], [have]), ([have], [add])):
        t.plan(*plan)
        shape = (len(t.slots), KVH, hd)
        t.append(rng.standard_normal(shape).astype(np.float32), rng.standard_normal(shape).astype(np.float32) * cols, "f16")
    w = H * hd
    q = (0.03 * torch.randn(add, w, generator=torch.Generator().manual_seed(3))).half().cuda()
    out = torch.zeros(add, w, dtype=torch.float16, device="cuda")
    torch.cuda.synchronize()
    t.kv.attend(0, q.data_ptr(), out.data_ptr(), q4hip.F16, w, w)
    K, V = (c.values(t.pool.tables[0], have + add) for c in t.ref[0])
    ks, vs = (c.scale_of(t.pool.tables[0], have + add) for c in t.ref[0])
    rows, err, rounding = np.linspace(0, add - 1, 40).astype(int), 0.0, 0.0
    y, got = q.float().cpu().numpy().reshape(add, H, hd), out.double().cpu().numpy().reshape(add, H, hd)
    for r in rows:
        n = have + r
        want = kv8_ref.attend(y[r:r + 1], K[:n + 1], V[:n + 1], ks[:n + 1], vs[:n + 1], n, hd ** -0.5, HALF["f16"])[0][0]
        err += np.square(got[r] - want).sum()
        rounding += np.square(want.astype(np.float16).astype(np.float64) - want).sum()
    assert err < 1.8 ** 2 * rounding


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attend_large_and_small_values(dtype):
    """Rows and pages of very different size: scores far apart, V scales from 1e-6 to 1e6."""
    rng = np.random.default_rng(3)
    t = Both(4, 2, 64, 2, 400, 30, 500)
    t.plan([0, 0], [200, 10])
    n = 210
    k = rng.standard_normal((n, 2, 64)).astype(np.float32) * np.float32(10.0) ** (np.arange(n)[:, None, None] // 32 % 3 - 1)
    v = rng.standard_normal((n, 2, 64)).astype(np.float32) * np.float32(10.0) ** ((np.arange(n)[:, None, None] // 32 % 5) * 3 - 6)
    t.append(k, v, dtype)
    t.plan([200, 10], [70, 1])
    t.fill(rng, dtype)
    for size in (1e-4, 1.0, 50.0):
        t.attend(rng, dtype, size=size)


def test_the_largest_queries_of_bf16_on_a_cache_of_zeros():
    """Scores of 0: the mean of V, however large q is."""
    rng = np.random.default_rng(14)
    t = Both(14, 2, 64, 2, 700, 30, 700)
    t.plan([0, 0], [600, 40])
    v = rng.standard_normal((640, 2, 64)).astype(np.float32)
    t.append(np.zeros_like(v), v, "bf16")
    t.plan([600, 40], [1, 1])
    v = rng.standard_normal((2, 2, 64)).astype(np.float32)
    t.append(np.zeros_like(v), v, "bf16")
    t.attend(rng, "bf16", size=1e35)
    t.attend(rng, "bf16", size=2e37)


def test_nan_and_infinite_queries_stay_in_their_rows():
    rng = np.random.default_rng(4)
    t = Both(14, 2, 64, 3, 200, 30, 300)
    t.plan([0] * 3, [100, 5, 0])
    t.fill(rng, "f32")
    t.plan([100, 5, 0], [1, 3, 80])
    t.fill(rng, "f32")
    n, w = 84, 14 * 64
    q = rng.standard_normal((n, w)).astype(np.float32)
    bad = {(0, 0): np.nan, (2, 3): np.inf, (3, 13): -np.inf, (50, 6): np.nan}
    for (r, h), x in bad.items():
        q[r, h * 64 + 5] = x
    d, out = torch.tensor(q).cuda(), torch.empty(n, w, device="cuda")
    torch.cuda.synchronize()
    t.kv.attend(0, d.data_ptr(), out.data_ptr(), q4hip.F32, w, w)
    got = out.double().cpu().numpy().reshape(n, 14, 64)
    for (r, h), x in bad.items():
        if np.isnan(x):
            assert np.isnan(got[r, h]).all()
        got[r, h] = 0
        q[r, h * 64:h * 64 + 64] = 0
    want = Both.compare
    for (r, h) in bad:                             # compare the others: these rows as if q were 0
        b = t.seq[r]
        i = r - [0, 1, 4][b]
        V = t.ref[0][1].values(t.pool.tables[b], t.have[b] + i + 1)[:, h // 7].astype(np.float64)
        got[r, h] = V.mean(0)
    want(t, got, q.reshape(n, 14, 64), "f32")


def test_pages_beyond_32_bits():
    """A pool of more than 4 GiB: another sequence holds the first pages."""
    rng = np.random.default_rng(6)
    H, KVH, hd = 16, 8, 128
    first = 70000                                  # pages of 64 KB
    kv = q4hip.Kv8(1, H, KVH, hd, 2, first * 32, first + 8, 256)
    h, a = ints([first * 32, 0]), ints([0, 200])
    tables = torch.empty(2, first, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    kv.plan(h.data_ptr(), a.data_ptr(), 200, tables=tables.data_ptr())
    assert tables[1, :7].tolist() == list(range(first, first + 7))
    t = Both.__new__(Both)
    t.kv, t.H, t.KVH, t.hd, t.B, t.layers, t.have, t.add = kv, H, KVH, hd, 2, 1, [0, 0], [0, 200]
    t.pool = kv8_ref.Pool(2, 32 * 7, 7)
    t.slots = t.pool.plan([0, 0], [0, 200], 200)[2]
    t.ref = [[kv8_ref.Cache(7, KVH, hd) for _ in range(2)]]
    t.fill(rng, "bf16")
    t.check_values()
    t.attend(rng, "bf16")


# ---------------------------------------------------------------------------- streams, graphs, refusals

def test_a_step_of_a_server_captured_and_replayed():
    """plan, append and attend of two layers in a graph: lengths and rows change between the replays, with
    eager work on the same handle in between."""
    rng = np.random.default_rng(8)
    H, KVH, hd, B = 14, 2, 64, 5
    t = Both(H, KVH, hd, B, 600, 60, 1000, layers=2)
    lens = [40, 0, 300, 31, 7]
    t.plan([0] * B, lens)
    for layer in range(2):
        t.fill(rng, "f32", layer)
    R, w = 8, (H + 2 * KVH) * hd
    have, add = ints([0] * B), ints([0] * B)
    x = [torch.zeros(R, w, device="cuda") for _ in range(2)]
    out = [torch.zeros(R, H * hd, device="cuda") for _ in range(2)]
    s = torch.cuda.Stream()

    def step(stream):
        t.kv.plan(have.data_ptr(), add.data_ptr(), R, stream=stream)
        for layer in range(2):
            y = x[layer]
            t.kv.append(layer, y[:, H * hd:].data_ptr(), y[:, (H + KVH) * hd:].data_ptr(), q4hip.F32, w, w, stream)
            t.kv.attend(layer, y.data_ptr(), out[layer].data_ptr(), q4hip.F32, w, H * hd, stream)

    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        step(torch.cuda.current_stream().cuda_stream)
    for i, more in enumerate(([1, 1, 1, 1, 1], [1, 4, 0, 2, 1], [0, 0, 0, 0, 0], [8, 0, 0, 0, 0], [1, 1, 1, 1, 1])):
        if i == 3:
            lens[2] = 33                           # a chat cut back
        have.copy_(ints(lens))
        add.copy_(ints(more))
        data = [rng.standard_normal((R, w)).astype(np.float32) for _ in range(2)]
        for layer in range(2):
            x[layer].copy_(torch.tensor(data[layer]))
            out[layer].fill_(7.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        n = sum(more)
        starts, pos, t.slots, tables, t.seq = t.pool.plan(lens, more, R)
        t.have, t.add = list(lens), list(more)
        assert t.kv.status() == (n, len(t.pool.stack))
        for layer in range(2):
            y = data[layer][:n]
            for c, at in ((0, H), (1, H + KVH)):
                t.ref[layer][c].append(y[:, at * hd:(at + KVH) * hd].reshape(n, KVH, hd), t.slots)
            t.check_values(layer)
            assert (out[layer][n:] == 7).all()
            t.compare(out[layer][:n].double().cpu().numpy().reshape(n, H, hd), y[:, :H * hd].reshape(n, H, hd), "f32", layer)
        once = [o.clone() for o in out]
        torch.cuda.synchronize()
        step(0)                                    # the same step, eagerly: the same results
        assert all(torch.equal(a, b) for a, b in zip(once, out))
        lens = [a + b for a, b in zip(lens, more)]


def test_a_graph_on_a_plan_that_is_too_large():
    """append and attend captured for 8 rows do nothing on a plan of 20, and the status says so."""
    rng = np.random.default_rng(10)
    t = Both(4, 2, 64, 2, 300, 20, 300)
    t.plan([0, 0], [30, 0])
    t.fill(rng, "f32")
    t.plan([30, 0], [4, 4])
    w = 8 * 64
    x, out = torch.randn(20, w, device="cuda"), torch.full((20, 256), 7.0, device="cuda")
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        st = torch.cuda.current_stream().cuda_stream
        t.kv.append(0, x[:, 256:].data_ptr(), x[:, 384:].data_ptr(), q4hip.F32, w, w, st)
        t.kv.attend(0, x.data_ptr(), out.data_ptr(), q4hip.F32, w, 256, st)
    t.plan([30, 0], [10, 10])
    t.fill(rng, "f32")
    g.replay()
    torch.cuda.synchronize()
    assert (out == 7).all()
    with pytest.raises(q4hip.Q4Error) as e:
        t.kv.status()
    assert e.value.code == q4hip.ESTATE
    t.check_values()
    t.plan([30, 0], [4, 4])
    g.replay()
    torch.cuda.synchronize()
    y = x[:8].cpu().numpy()
    for c, at in ((0, 4), (1, 6)):
        t.ref[0][c].append(y[:, at * 64:(at + 2) * 64].reshape(8, 2, 64), t.slots)
    assert (out[8:] == 7).all()
    t.compare(out[:8].double().cpu().numpy().reshape(8, 4, 64), y[:, :256].reshape(8, 4, 64), "f32")
    assert t.kv.status()[0] == 8


def test_two_handles_on_two_streams():
    rng = np.random.default_rng(12)
    ts = [Both(14, 2, 64, 2, 3000, 200, 4000) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in ts]
    for t in ts:
        t.plan([0, 0], [2500, 300])
        t.fill(rng, "f32")
        t.plan([2500, 300], [1, 1])
        t.fill(rng, "f32")
    w = 14 * 64
    q = [torch.randn(2, w, device="cuda") for _ in ts]
    out = [[torch.zeros(2, w, device="cuda") for _ in range(8)] for _ in ts]
    torch.cuda.synchronize()
    for i in range(8):
        for t, s, y, o in zip(ts, streams, q, out):
            t.kv.attend(0, y.data_ptr(), o[i].data_ptr(), q4hip.F32, w, w, s.cuda_stream)
    torch.cuda.synchronize()
    for t, y, o in zip(ts, q, out):
        assert all(torch.equal(a, o[0]) for a in o)
        t.compare(o[0].double().cpu().numpy().reshape(2, 14, 64), y.cpu().numpy().reshape(2, 14, 64), "f32")


def test_refusals():
    kv = q4hip.Kv8(2, 4, 2, 64, 2, 100, 8, 16)
    d = torch.zeros(16 * 256 + 1, device="cuda")
    i = ints([0, 0, 0])
    host = torch.zeros(4096)
    one, four = ints([1, 0]), ints([4, 0])
    both = torch.zeros(16 * 1024, device="cuda")
    torch.cuda.synchronize()
    p, ip, hp = d.data_ptr(), i.data_ptr(), host.data_ptr()

    def refused(code, call, *args):
        with pytest.raises(q4hip.Q4Error) as e:
            call(*args)
        assert e.value.code == code, e.value

    refused(q4hip.EINVAL, kv.plan, 0, ip, 1)
    refused(q4hip.EINVAL, kv.plan, ip, 0, 1)
    refused(q4hip.EINVAL, kv.plan, ip, ip, 17)
    refused(q4hip.EINVAL, kv.plan, ip, ip, -1)
    refused(q4hip.EINVAL, kv.plan, hp, ip, 1)
    refused(q4hip.EINVAL, kv.plan, ip, ip, 1, hp)
    kv.append(0, p, p, q4hip.F32, 128, 128)        # a step without rows: nothing to do
    kv.attend(0, p, p, q4hip.F32, 256, 256)
    kv.plan(ip, one.data_ptr(), 1)
    for layer in (-1, 2):
        refused(q4hip.EINVAL, kv.append, layer, p, p, q4hip.F32, 128, 128)
        refused(q4hip.EINVAL, kv.attend, layer, p, p, q4hip.F32, 256, 256)
        refused(q4hip.EINVAL, kv.read, layer, ip, ip, 1, p, p)
    for typ in (2, 8, 31, -1):
        refused(q4hip.ETYPE, kv.append, 0, p, p, typ, 128, 128)
        refused(q4hip.ETYPE, kv.attend, 0, p, p, typ, 256, 256)
    refused(q4hip.EINVAL, kv.append, 0, p, p, q4hip.F32, 127, 128)
    refused(q4hip.EINVAL, kv.append, 0, p, p, q4hip.F32, 128, -128)
    refused(q4hip.EINVAL, kv.append, 0, p, p, q4hip.F32, 128, 1 << 40)
    refused(q4hip.EINVAL, kv.append, 0, p + 2, p, q4hip.F32, 128, 128)
    refused(q4hip.EINVAL, kv.append, 0, p, p + 1, q4hip.BF16, 128, 128)
    refused(q4hip.EINVAL, kv.append, 0, hp, p, q4hip.F32, 128, 128)
    refused(q4hip.EINVAL, kv.append, 0, 0, p, q4hip.F32, 128, 128)
    refused(q4hip.EINVAL, kv.attend, 0, p, 0, q4hip.F32, 256, 256)
    refused(q4hip.EINVAL, kv.attend, 0, p, hp, q4hip.F32, 256, 256)
    refused(q4hip.EINVAL, kv.attend, 0, p, p, q4hip.F32, 255, 256)
    refused(q4hip.EINVAL, kv.attend, 0, p, p, q4hip.F32, 256, 255)
    a, wide = both.data_ptr(), 1024
    kv.plan(ip, four.data_ptr(), 4)
    refused(q4hip.EINVAL, kv.attend, 0, a, a, q4hip.F32, 256, 256)
    refused(q4hip.EINVAL, kv.attend, 0, a, a + 4, q4hip.F32, wide, wide)
    refused(q4hip.EINVAL, kv.attend, 0, a + 4 * 255, a, q4hip.F32, wide, wide)
    refused(q4hip.EINVAL, kv.attend, 0, a, a + 4 * (wide + 255), q4hip.F32, wide, wide)
    refused(q4hip.EINVAL, kv.attend, 0, a, a + 4 * 256, q4hip.F32, wide, 256)
    kv.attend(0, a, a + 4 * 256, q4hip.F32, wide, wide)
    kv.attend(0, a + 4 * 256, a, q4hip.F32, wide, wide)
    kv.attend(0, a, a + 4 * 1024, q4hip.F32, 256, 256)
    kv.plan(ip, one.data_ptr(), 1)
    refused(q4hip.EINVAL, kv.plan, ip + 2, ip, 1)
    refused(q4hip.EINVAL, kv.plan, ip, ip, 1, 0, ip + 1)
    refused(q4hip.EINVAL, kv.read, 0, ip, ip + 2, 1, p, p)
    for scale in (float("nan"), float("inf"), -1.0):
        refused(q4hip.EINVAL, kv.attend, 0, p, p, q4hip.F32, 256, 256, 0, scale)
    refused(q4hip.EINVAL, kv.read, 0, ip, ip, -1, p, p)
    refused(q4hip.EINVAL, kv.read, 0, ip, hp, 1, p, p)
    kv.read(0, ip, ip, 0, p, p)
    assert kv.status() == (1, 7)
    kv.close()
