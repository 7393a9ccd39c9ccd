"""Rotary positions: frequencies and refusals that need no GPU."""
import ctypes
import math

import numpy as np
import pytest

import q4hip


@pytest.mark.parametrize("rot,theta", [(2, 1e4), (32, 1e4), (64, 1e6), (128, 5e5), (80, 1e4)])
def test_plain_and_linear(rot, theta):
    want = [theta ** (-2 * i / rot) for i in range(rot // 2)]
    f, a = q4hip.rope_frequencies(rot, theta)
    assert a == 1.0 and np.allclose(f, want, rtol=4e-15, atol=0)
    f, a = q4hip.rope_frequencies(rot, theta, "linear", factor=2.5)
    assert a == 1.0 and np.allclose(f, np.array(want) / 2.5, rtol=4e-15, atol=0)


def test_bands():
    """By the turns over the original context: whole below `low`, none above `high`, in proportion between."""
    rot, theta, factor, original, low, high = 128, 5e5, 8.0, 8192, 1.0, 4.0
    plain, _ = q4hip.rope_frequencies(rot, theta)
    f, a = q4hip.rope_frequencies(rot, theta, "bands", factor, original, low, high)
    assert a == 1.0
    kinds = set()
    for p, x in zip(plain, f):
        turns = original * p / (2 * math.pi)
        if turns <= low:
            kinds.add("whole")
            assert x == pytest.approx(p / factor, rel=1e-14)
        elif turns >= high:
            kinds.add("none")
            assert x == pytest.approx(p, rel=1e-14)
        else:
            kinds.add("part")
            share = (turns - low) / (high - low)
            assert x == pytest.approx(p / factor * (1 - share) + p * share, rel=1e-13)
    assert kinds == {"whole", "none", "part"}


def test_yarn():
    rot, theta, factor, original, low, high = 64, 1e6, 4.0, 4096, 1.0, 32.0
    plain, _ = q4hip.rope_frequencies(rot, theta)
    f, a = q4hip.rope_frequencies(rot, theta, "yarn", factor, original, low, high)
    assert a == pytest.approx(0.1 * math.log(4.0) + 1, rel=1e-7)
    # the pair that makes t turns: original * theta^(-2 i / rot) = 2 pi t
    at = {t: rot / 2 * math.log(original / (2 * math.pi * t)) / math.log(theta) for t in (low, high)}
    first, last = math.floor(at[high]), math.ceil(at[low])
    for i, (p, x) in enumerate(zip(plain, f)):
        share = min(max((i - first) / (last - first), 0), 1)
        assert x == pytest.approx(p / factor * share + p * (1 - share), rel=1e-13)
    assert f[0] == plain[0] and f[-1] == pytest.approx(plain[-1] / factor, rel=1e-14)
    f, a = q4hip.rope_frequencies(rot, theta, "yarn", 1.0, original, low, high)
    assert a == 1.0 and np.allclose(f, plain, rtol=1e-15, atol=0)


@pytest.mark.parametrize("rot,theta,scaling,p", [
    (0, 1e4, "plain", {}), (3, 1e4, "plain", {}), (514, 1e4, "plain", {}), (64, 1.0, "plain", {}), (64, math.nan, "plain", {}),
    (64, math.inf, "plain", {}), (64, 1e4, "linear", dict(factor=0.5)), (64, 1e4, "linear", dict(factor=math.nan)),
    (64, 1e4, "bands", dict(factor=2, original=0, low=1, high=4)), (64, 1e4, "bands", dict(factor=2, original=100, low=4, high=4)),
    (64, 1e4, "yarn", dict(factor=2, original=100, low=0, high=4)), (64, 1e4, "yarn", dict(factor=math.inf, original=100, low=1, high=4))])
def test_frequencies_refuse(rot, theta, scaling, p):
    with pytest.raises(q4hip.Q4Error) as e:
        q4hip.rope_frequencies(rot, theta, scaling, **p)
    assert e.value.code == q4hip.EINVAL


@pytest.mark.parametrize("head_dim,rot,order,freq,amplitude", [
    (64, 0, 0, [], 1.0), (64, 66, 0, [1.0] * 33, 1.0), (64, 31, 0, [1.0] * 16, 1.0), (1, 2, 0, [1.0], 1.0), (1024, 64, 0, [1.0] * 32, 1.0),
    (64, 4, 2, [1.0, 1.0], 1.0), (64, 4, -1, [1.0, 1.0], 1.0), (64, 4, 0, [1.0, math.nan], 1.0), (64, 4, 0, [math.inf, 1.0], 1.0),
    (64, 4, 0, [1.0, 1.0], math.inf)])
def test_create_refuses(head_dim, rot, order, freq, amplitude):
    h = ctypes.c_void_p()
    f = (ctypes.c_double * max(len(freq), 1))(*freq)
    assert q4hip.lib().q4hip_rope_create(ctypes.byref(h), head_dim, rot, order, f, amplitude, 0) == q4hip.EINVAL
    assert not h.value


def test_null_arguments():
    L = q4hip.lib()
    one = ctypes.c_double(0)
    p = ctypes.addressof(one)
    assert L.q4hip_rope_create(None, 64, 64, 0, p, 1.0, 0) == q4hip.EINVAL
    assert L.q4hip_rope_frequencies(2, 1e4, 0, 1.0, 0.0, 0.0, 0.0, None, None) == q4hip.EINVAL
    assert L.q4hip_rope_run(None, p, p, 1, 0, 64, 64, p, 1, None, None) == q4hip.EINVAL
    L.q4hip_rope_destroy(None)
