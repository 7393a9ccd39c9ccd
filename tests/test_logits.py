"""Logits' rules: refusals that need no GPU, the records' layout."""
import ctypes

import pytest

import q4hip


@pytest.mark.parametrize("vocab,rows", [(0, 1), (-1, 1), (1 << 31 - 1, 1 << 20), (100, 0), (100, -2), (100, (1 << 20) + 1), ((1 << 30) + 1, 1)])
def test_create_refuses(vocab, rows):
    h = ctypes.c_void_p()
    assert q4hip.lib().q4hip_logits_create(ctypes.byref(h), vocab, rows, 0) == q4hip.EINVAL
    assert not h.value


def test_null_arguments():
    L = q4hip.lib()
    one = ctypes.c_int(0)
    p = ctypes.addressof(one)
    assert L.q4hip_logits_create(None, 100, 1, 0) == q4hip.EINVAL
    assert L.q4hip_logits_run(None, p, p, 0, 100, 100, 1, p, None, 0, None, 0, None, 0, None, None) == q4hip.EINVAL
    L.q4hip_logits_destroy(None)


def test_records():
    assert q4hip.LOGITS_ROW.itemsize == 32 and q4hip.LOGITS_BIAS.itemsize == 8
