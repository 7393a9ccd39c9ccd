"""Batches on the paged 8-bit cache: attention in every layer, behind earlier passes of the same prompt, and of a chat cut back.

Attention of one layer at a time is made visible: the other layers' attention output and FFN are zero, so that they pass on
what they get, and behind that layer the matrices are the identity (test_gpu_batch_kv8.py's one-layer models, its references and
bounds).  The layers' K and V differ, as their weights do.
"""
import numpy as np
import pytest

import kv8_ref
import oracle
import q4hip
import synth
from test_gpu_batch_kv8 import carry, model

pytestmark = pytest.mark.gpu

LAYERS = {"three64": synth.Shape(256, 3, 512, 4, 2, 512), "three128": synth.Shape(256, 3, 512, 2, 1, 512)}


def only(shape, layer, seed):
    """Tensors of a model of which one layer does something, and those of that layer as a one-layer model's."""
    t = synth.make_model(shape, seed)

    def put(tensor, m):
        t[tensor].data = synth.quantize_q4_0(m.astype(np.float32)).reshape(t[tensor].data.shape)

    for l in range(shape.layers):
        put(f"blk.{l}.attn_output.weight", np.eye(shape.dim) if l == layer else np.zeros((shape.dim, shape.dim)))
        put(f"blk.{l}.ffn_down.weight", np.zeros((shape.dim, shape.ffn)))
    put("output.weight", np.eye(shape.vocab, shape.dim))
    one = {n.replace(f"blk.{layer}.", "blk.0."): x for n, x in t.items() if not n.startswith("blk.") or n.startswith(f"blk.{layer}.")}
    return t, one


def expected(shape, t, layer, ids, ctx, cuts):
    """[(values, scales)] of K and V of a layer after appends of ids[a:b] for the cuts (a, b), by the oracle's fp32 rows."""
    o = oracle.Model(shape, t, ctx=ctx)
    o.forward(ids, 0)
    n, pages, got = len(ids), -(-len(ids) // 32), []
    for rows in o.kv():
        c = kv8_ref.Cache(pages, shape.kv_heads, shape.head_dim)
        x = rows[layer, :, :n].transpose(1, 0, 2).copy()
        for a, b in cuts:
            c.append(x[a:b], np.arange(a, b))
        got.append((c.values(list(range(pages)), n), c.scale_of(list(range(pages)), n)))
    o.close()
    return got


@pytest.mark.parametrize("mt", [0, 16])
@pytest.mark.parametrize("layer", [0, 1, 2])
@pytest.mark.parametrize("name", sorted(LAYERS))
def test_attention_of_every_layer(name, layer, mt):
    """Prompts in one pass or in passes of 16 rows, then steps."""
    shape, ctx, steps = LAYERS[name], 160, 4
    t, one = only(shape, layer, 50 + layer)
    g = q4hip.Model(shape, ctx=ctx, mt=mt)
    g.load(t)
    rng = np.random.default_rng(layer)
    lens = [5, 40, 100]
    prompts = [rng.integers(0, shape.vocab, n).astype(np.int32) for n in lens]
    bt = q4hip.Batch(g, 3, kv8_pages=9)

    def check(b, fed, cuts, lg):
        n = len(fed)
        kv = expected(shape, t, layer, fed, ctx, cuts)
        for h in range(shape.kv_heads):
            k, v = bt.get_kv(b, layer, h, 0, n)
            assert np.array_equal(k, kv[0][0][:, h]) and np.array_equal(v, kv[1][0][:, h])
        want, E = carry(shape, one, fed[-1], n - 1, kv, ctx)
        assert (lg[shape.dim:] == 0).all()
        assert (np.abs(lg[:shape.dim] - want) <= E).all(), float((np.abs(lg[:shape.dim] - want) / E).max())
        assert E.max() < 0.1 * want.std()          # a bound that another layer's pages break

    try:
        first, cuts = [], []
        for b, ids in enumerate(prompts):
            n, pass_ = len(ids), mt or len(ids)
            first.append(bt.prefill(b, ids, 0))
            cuts.append([(a, min(a + pass_, n)) for a in range(0, n, pass_)])
            check(b, list(ids), cuts[b], g.read_logits())
        out = bt.generate(first, lens, steps)
        lg = bt.read_logits()
        for b, n in enumerate(lens):
            check(b, list(prompts[b]) + [first[b]] + out[:-1, b].tolist(), cuts[b] + [(n + i, n + i + 1) for i in range(steps)], lg[b])
    finally:
        bt.close()
        g.close()


@pytest.mark.parametrize("name,cut", [("one64", 50), ("one128", 50), ("one64x4", 50), ("one64x4", 64), ("one64", 1)])
def test_a_chat_cut_back(name, cut):
    """100 positions in passes of 16, cut back to `cut` and continued by 5 others: every position to the bit (the page cut in its
    middle keeps its scale), and the logits."""
    ctx = 160
    shape, t, g = model(name, 5, ctx, mt=16)
    rng = np.random.default_rng(9)
    ids, more = (rng.integers(0, shape.vocab, n).astype(np.int32) for n in (100, 5))
    fed = np.concatenate([ids[:cut], more])
    n = cut + 5
    bt = q4hip.Batch(g, 1, kv8_pages=4)
    try:
        bt.prefill(0, ids, 0)
        bt.prefill(0, more, cut)
        o = oracle.Model(shape, t, ctx=ctx)
        caches, table = [], [0, 1, 2, 3]
        for ids_, runs in ((ids, [(a, min(a + 16, 100)) for a in range(0, 100, 16)]), (fed, [(cut, n)])):
            o.forward(ids_, 0)
            for i, rows in enumerate(o.kv()):
                if len(caches) <= i:
                    caches.append(kv8_ref.Cache(4, shape.kv_heads, shape.head_dim))
                x = rows[0, :, :len(ids_)].transpose(1, 0, 2).copy()
                for a, b in runs:
                    caches[i].append(x[a:b], np.arange(a, b))
        o.close()
        kv = [(c.values(table, n), c.scale_of(table, n)) for c in caches]
        for h in range(shape.kv_heads):
            k, v = bt.get_kv(0, 0, h, 0, n)
            assert np.array_equal(k, kv[0][0][:, h]) and np.array_equal(v, kv[1][0][:, h])
        want, E = carry(shape, t, int(fed[-1]), n - 1, kv, ctx)
        assert (np.abs(g.read_logits()[:shape.dim] - want) <= E).all()
    finally:
        bt.close()
        g.close()
