"""Rotary positions (q4hip_rope_*) on the GPU against 64 bits.

The bound of a turned value a = A (x cos t - y sin t): the angle's part of a turn is cut to 2^-32 (2^-29 rad), and as an fp32
number within pi / 4 it has three roundings (pi / 4 * 3 * 2^-24); the series' own rounding is under 2 * 2^-24 and what they leave out under
2e-9; so cosine and sine are off by 5 * 2^-24 at most.  The amplitude's product, the product with y and the fused sum round once
each: (|x| + |y|) A * 8 * 2^-24 in all, then the rounding to the type.
"""
import numpy as np
import pytest
import torch

import q4hip

pytestmark = pytest.mark.gpu

TYPES = {"f32": (q4hip.F32, torch.float32), "f16": (q4hip.F16, torch.float16), "bf16": (q4hip.BF16, torch.bfloat16)}
LEAST = {"f32": 2.0 ** -150, "f16": 2.0 ** -25, "bf16": 2.0 ** -134}      # half of the smallest step


def want_of(x, pos, freq, amplitude, heads, head_dim, rot, order, half_eps, least):
    """(values, bound) in 64 bits; the angles' full turns are taken off in 80 bits."""
    n = x.shape[0]
    x = x.reshape(n, heads, head_dim)
    turns = np.asarray(pos, np.longdouble)[:, None] * (np.asarray(freq, np.longdouble) / (2 * np.longdouble("3.14159265358979323846264338")))
    t = (2 * np.pi * (turns - np.floor(turns)).astype(np.float64))[:, None, :]
    first, second = (np.s_[:, :, :rot // 2], np.s_[:, :, rot // 2:rot]) if order == "halves" else (np.s_[:, :, :rot:2], np.s_[:, :, 1:rot:2])
    a, b = x[first], x[second]
    y, bound = x.copy(), np.zeros_like(x)
    y[first] = amplitude * (a * np.cos(t) - b * np.sin(t))
    y[second] = amplitude * (b * np.cos(t) + a * np.sin(t))
    err = (np.abs(a) + np.abs(b)) * abs(amplitude) * 8 * 2.0 ** -24
    for at in (first, second):
        bound[at] = err + (np.abs(y[at]) + err) * half_eps + least
    return y.reshape(n, heads * head_dim), bound.reshape(n, heads * head_dim)


def check(got, x, dtype, *args):
    half = torch.finfo(TYPES[dtype][1]).eps / 2
    want, bound = want_of(x.double().cpu().numpy(), *args, half, LEAST[dtype])
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= bound).all(), float((err / np.maximum(bound, 1e-300)).max())


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("order", ["halves", "pairs"])
@pytest.mark.parametrize("rows,heads,head_dim,rot,offset", [
    (1, 16, 64, 64, 0), (1, 1, 2, 2, 0), (7, 3, 128, 64, 0), (65, 40, 128, 128, 0), (5, 5, 80, 20, 0), (9, 2, 64, 6, 0),
    (33, 4, 64, 32, 1), (3, 7, 12, 12, 3), (2100, 2, 64, 64, 0), (4100, 3, 96, 48, 0), (2, 1, 512, 512, 0), (130, 9, 50, 50, 0)])
def test_rows(dtype, order, rows, heads, head_dim, rot, offset):
    """Rows within wider ones, `offset` columns in; what lies around them stays as it is."""
    rng = np.random.default_rng(rows + heads + rot)
    typ, t = TYPES[dtype]
    freq, amplitude = q4hip.rope_frequencies(rot, 1e4)
    r = q4hip.Rope(head_dim, rot, order, freq)
    w = heads * head_dim
    x = torch.tensor(rng.standard_normal((rows, w + offset + 5 * (offset > 0)))).to(t).cuda()
    pos = rng.integers(0, 200000, rows)
    p = torch.tensor(pos, dtype=torch.int32, device="cuda")
    y = torch.full((rows + 1, w + 2 * offset), 7.0, dtype=t, device="cuda")
    torch.cuda.synchronize()
    r.run(x[:, offset:].data_ptr(), y[:, offset:].data_ptr(), heads, typ, x.stride(0), y.stride(0), p.data_ptr(), rows)
    assert (y[rows:] == 7).all() and (y[:, :offset] == 7).all() and (y[:, w + offset:] == 7).all()
    check(y[:rows, offset:offset + w], x[:, offset:offset + w], dtype, pos, freq, amplitude, heads, head_dim, rot, order)
    before = x.clone()
    out = y[:rows, offset:offset + w].clone()
    r.run(x[:, offset:].data_ptr(), x[:, offset:].data_ptr(), heads, typ, x.stride(0), x.stride(0), p.data_ptr(), rows)
    assert torch.equal(x[:, offset:offset + w], out)                  # in place: the same bits
    x[:, offset:offset + w] = before[:, offset:offset + w]
    assert torch.equal(x, before)


@pytest.mark.parametrize("order", ["halves", "pairs"])
@pytest.mark.parametrize("scaling,p", [("plain", {}), ("linear", dict(factor=8)), ("bands", dict(factor=8, original=8192, low=1, high=4)),
                                       ("yarn", dict(factor=16, original=4096, low=1, high=32))])
def test_far_positions(order, scaling, p):
    """Every position of 32 bits, negative ones, too."""
    freq, amplitude = q4hip.rope_frequencies(128, 1e6, scaling, **p)
    r = q4hip.Rope(128, 128, order, freq, amplitude)
    pos = np.concatenate([np.arange(-3, 70), [2 ** k + d for k in range(7, 31) for d in (-1, 0, 1)], [2 ** 31 - 1, -2 ** 31, -1000001]])
    x = torch.randn(len(pos), 256, device="cuda")
    ip = torch.tensor(pos, dtype=torch.int32, device="cuda")
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    r.run(x.data_ptr(), y.data_ptr(), 2, q4hip.F32, 256, 256, ip.data_ptr(), len(pos))
    check(y, x, "f32", pos, freq, amplitude, 2, 128, 128, order)


def test_frequencies_of_the_caller():
    """Any finite ones: of more than a turn a position, negative, zero."""
    freq = np.array([0.0, -0.3, 7.5, 1e6, -2 * np.pi, 1e-30])
    r = q4hip.Rope(12, 12, "halves", freq, -0.5)
    pos = np.arange(500)
    x, p = torch.randn(500, 12, device="cuda"), torch.arange(500, dtype=torch.int32, device="cuda")
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    r.run(x.data_ptr(), y.data_ptr(), 1, q4hip.F32, 12, 12, p.data_ptr(), 500)
    check(y, x, "f32", pos, freq, -0.5, 1, 12, 12, "halves")


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_columns_that_are_not_turned(dtype):
    """They keep their bits: NaN, infinities, zeros of either sign; turned ones follow the arithmetic."""
    typ, t = TYPES[dtype]
    freq, _ = q4hip.rope_frequencies(16, 1e4)
    r = q4hip.Rope(64, 16, "halves", freq)
    x = torch.randn(4, 128, device="cuda").to(t)
    x[:, 20], x[:, 21], x[:, 90], x[:, 91] = float("nan"), float("inf"), -0.0, -float("inf")
    x[1, 3], x[2, 70] = float("nan"), float("inf")
    p = torch.tensor([0, 5, 9, 100], dtype=torch.int32, device="cuda")
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    r.run(x.data_ptr(), y.data_ptr(), 2, typ, 128, 128, p.data_ptr(), 4)
    bits = torch.int32 if dtype == "f32" else torch.int16
    for h in (0, 64):
        assert torch.equal(x.view(bits)[:, h + 16:h + 64], y.view(bits)[:, h + 16:h + 64])
    assert y[1, 3].isnan() and y[1, 11].isnan() and not y[2, 70].isfinite() and not y[2, 78].isfinite()
    assert int((~y[:, :16].isfinite()).sum()) == 2 and int((~y[:, 64:80].isfinite()).sum()) == 2


@pytest.mark.parametrize("rows,count", [(5, 3), (5, 0), (5, 9), (5, -1), (3000, 2049)])
def test_count(rows, count):
    freq, amplitude = q4hip.rope_frequencies(64, 1e4)
    r = q4hip.Rope(64, 64, "halves", freq)
    x, p = torch.randn(rows, 64, device="cuda"), torch.arange(rows, dtype=torch.int32, device="cuda")
    c = torch.tensor([count], dtype=torch.int32, device="cuda")
    y = torch.full_like(x, 7.0)
    torch.cuda.synchronize()
    r.run(x.data_ptr(), y.data_ptr(), 1, q4hip.F32, 64, 64, p.data_ptr(), rows, c.data_ptr())
    n = max(0, min(rows, count))
    assert (y[n:] == 7).all()
    check(y[:n], x[:n], "f32", np.arange(n), freq, amplitude, 1, 64, 64, "halves")


def test_captured_and_on_two_streams():
    """A graph replayed with other positions and rows, two streams at once on one handle."""
    freq, amplitude = q4hip.rope_frequencies(128, 1e6)
    r = q4hip.Rope(128, 128, "halves", freq)
    n, heads, w = 100, 10, 1280
    x, y = (torch.randn(n, w, device="cuda").to(torch.bfloat16) for _ in range(2))
    p, c = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=torch.cuda.Stream()):
        r.run(x.data_ptr(), y.data_ptr(), heads, q4hip.BF16, w, w, p.data_ptr(), n, c.data_ptr(), torch.cuda.current_stream().cuda_stream)
    for i, count in enumerate((100, 1, 57)):
        x.copy_(torch.randn(n, w, device="cuda"))
        p.copy_(torch.randint(0, 100000, (n,), device="cuda"))
        c.fill_(count)
        y.fill_(7.0)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert (y[count:] == 7).all()
        check(y[:count], x[:count], "bf16", p.cpu().numpy()[:count], freq, amplitude, heads, 128, 128, "halves")
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.empty_like(x) for _ in streams]
    for s, out in zip(streams, outs):
        r.run(x.data_ptr(), out.data_ptr(), heads, q4hip.BF16, w, w, p.data_ptr(), n, 0, s.cuda_stream)
    torch.cuda.synchronize()
    assert torch.equal(outs[0], outs[1])


def test_refusals():
    freq, _ = q4hip.rope_frequencies(64, 1e4)
    r = q4hip.Rope(64, 64, "halves", freq)
    x, y = torch.zeros(8, 128, device="cuda"), torch.zeros(8, 128, device="cuda")
    p = torch.zeros(8, dtype=torch.int32, device="cuda")
    host = np.zeros((8, 128), np.float32)
    good = dict(x=x.data_ptr(), y=y.data_ptr(), heads=2, dtype=q4hip.F32, x_stride=128, y_stride=128, pos=p.data_ptr(), rows=8)
    r.run(**good)
    for change, code in [(dict(x=host.ctypes.data), q4hip.EINVAL), (dict(y=host.ctypes.data), q4hip.EINVAL), (dict(x=0), q4hip.EINVAL),
                         (dict(pos=0), q4hip.EINVAL), (dict(pos=host.ctypes.data), q4hip.EINVAL), (dict(pos=p.data_ptr() + 2), q4hip.EINVAL),
                         (dict(x=x.data_ptr() + 2), q4hip.EINVAL), (dict(x_stride=127), q4hip.EINVAL), (dict(y_stride=64), q4hip.EINVAL),
                         (dict(x_stride=2 ** 32), q4hip.EINVAL), (dict(heads=0), q4hip.EINVAL), (dict(heads=20000), q4hip.EINVAL),
                         (dict(rows=-1), q4hip.EINVAL), (dict(rows=600000), q4hip.EINVAL), (dict(dtype=7), q4hip.ETYPE),
                         (dict(count=p.data_ptr() + 1), q4hip.EINVAL), (dict(count=host.ctypes.data), q4hip.EINVAL),
                         (dict(y=x.data_ptr() + 4), q4hip.EINVAL), (dict(y=x.data_ptr(), y_stride=129), q4hip.EINVAL),
                         (dict(y=x.data_ptr() + 256, rows=4), q4hip.EINVAL)]:
        with pytest.raises(q4hip.Q4Error) as e:
            r.run(**{**good, **change})
        assert e.value.code == code, change
    with pytest.raises(q4hip.Q4Error):          # positions among the rows that it writes
        r.run(**{**good, "pos": y.view(torch.int32)[3].data_ptr()})
    r.run(**{**good, "rows": 0, "x": p.data_ptr()})
    # q and k's columns of the same rows as x and y share no byte
    r.run(x.data_ptr(), x.data_ptr() + 256, 1, q4hip.F32, 128, 128, p.data_ptr(), 8)
