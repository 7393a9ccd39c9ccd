"""Device memory of the 8-bit cache beside its pages: what forks and shared pages need, only where there can be any."""
import pytest
import torch

import q4hip
import synth

pytestmark = pytest.mark.gpu

B, CTX, PAGES = 256, 4096, 100000
SHAPE = synth.Shape(1024, 1, 256, 16, 16, 512)


def taken(make):
    torch.cuda.synchronize()
    before = torch.cuda.mem_get_info()[0]
    x = make()
    after = torch.cuda.mem_get_info()[0]
    return x, before - after


def test_a_batch_never_forks():
    """A batch's cache against the same one for callers of their own: joints of 256 sequences, 2 * 256 slots of 32 rows for each of 16 kv
    heads, are 67 MB, a second table 0.13 MB, three arrays of pages 1.2 MB."""
    m = q4hip.Model(SHAPE, ctx=CTX, mt=256)
    bt, own = taken(lambda: q4hip.Batch(m, B, kv8_pages=PAGES))
    kv, other = taken(lambda: q4hip.Kv8(1, SHAPE.heads, SHAPE.kv_heads, SHAPE.head_dim, B, CTX, PAGES, CTX))
    kv.close()
    assert own + 60_000_000 < other
    bt.close()
    m.close()
