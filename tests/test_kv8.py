"""The paged 8-bit cache's refusals that need no GPU."""
import ctypes

import pytest

import q4hip

GOOD = dict(layers=2, heads=4, kv_heads=2, head_dim=64, seqs=3, max_len=100, pages=8, max_rows=16)


@pytest.mark.parametrize("change", [dict(layers=0), dict(heads=0), dict(kv_heads=0), dict(heads=5), dict(head_dim=32),
                                    dict(head_dim=96), dict(seqs=0), dict(max_len=0), dict(pages=0), dict(max_rows=0),
                                    dict(pages=1 << 27), dict(max_len=(1 << 31) - 1), dict(heads=65536, kv_heads=1),
                                    dict(layers=65536), dict(seqs=-1), dict(pages=-5)])
def test_create_refuses(change):
    with pytest.raises(q4hip.Q4Error) as e:
        q4hip.Kv8(**{**GOOD, **change})
    assert e.value.code == q4hip.EINVAL


def test_null_arguments():
    L = q4hip.lib()
    one = ctypes.c_int(0)
    p = ctypes.addressof(one)
    assert L.q4hip_kv8_create(None, 1, 1, 1, 64, 1, 1, 1, 1, 0) == q4hip.EINVAL
    assert L.q4hip_kv8_plan(None, p, p, 1, None, None, None, None, None) == q4hip.EINVAL
    assert L.q4hip_kv8_status(None, None, None, None) == q4hip.EINVAL
    assert L.q4hip_kv8_append(None, 0, p, p, 0, 64, 64, None) == q4hip.EINVAL
    assert L.q4hip_kv8_read(None, 0, p, p, 1, p, p, None) == q4hip.EINVAL
    assert L.q4hip_kv8_attend(None, 0, p, p, 0, 64, 64, 0.0, None) == q4hip.EINVAL
    L.q4hip_kv8_destroy(None)
