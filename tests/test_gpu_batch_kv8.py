"""Batches on the paged 8-bit cache (q4hip_batch_create_kv8).

Layer 0's K and V do not depend on attention, so the cache of layer 0 is checked to the bit: the oracle's fp32 rows,
rounded as kv8_ref.py does.  Of models with one layer attention itself is checked, too, in models whose matrices behind
it pass it on (attention's output and the head are the identity, the FFN adds nothing), so that the first logits are the
normalised sum of embedding and attention: in 64 bits with kv8_ref.py's bound, carried through the roundings to 8 bits
on the way (carry below).
"""
import json
import subprocess

import numpy as np
import pytest

import kv8_ref
import oracle
import q4hip
import synth

pytestmark = pytest.mark.gpu

SHAPES = {"one64": synth.Shape(128, 1, 256, 2, 1, 512), "one128": synth.Shape(256, 1, 512, 2, 1, 512),
          "one64x4": synth.Shape(256, 1, 512, 4, 2, 512)}


def model(name, seed, ctx, mt=0):
    shape = SHAPES.get(name) or synth.SHAPES[name]
    t = synth.make_model(shape, seed)
    if name in SHAPES:
        for tensor, m in (("blk.0.attn_output.weight", np.eye(shape.dim)), ("output.weight", np.eye(shape.vocab, shape.dim)),
                          ("blk.0.ffn_down.weight", np.zeros((shape.dim, shape.ffn)))):
            t[tensor].data = synth.quantize_q4_0(m.astype(np.float32)).reshape(t[tensor].data.shape)
    g = q4hip.Model(shape, ctx=ctx, mt=mt)
    g.load(t)
    return shape, t, g


def expected_kv(shape, t, ids, ctx, cuts):
    """(K, V) kv8_ref values [n][kv_heads][head_dim] and scales of layer 0 after appends of ids[a:b] for the cuts (a, b)."""
    o = oracle.Model(shape, t, ctx=ctx)
    o.forward(ids, 0)
    n, pages = len(ids), -(-len(ids) // 32)
    got = []
    for rows in o.kv():
        c = kv8_ref.Cache(pages, shape.kv_heads, shape.head_dim)
        x = rows[0, :, :n].transpose(1, 0, 2).copy()
        for a, b in cuts:
            c.append(x[a:b], np.arange(a, b))
        got.append((c.values(list(range(pages)), n), c.scale_of(list(range(pages)), n)))
    o.close()
    return got


def check_layer0(bt, seq, shape, kv):
    n = kv[0][0].shape[0]
    for g in range(shape.kv_heads):
        k, v = bt.get_kv(seq, 0, g, 0, n)
        assert np.array_equal(k, kv[0][0][:, g]) and np.array_equal(v, kv[1][0][:, g]), (seq, g)


def carry(shape, t, token, pos, kv, ctx):
    """(first logits, bound) of the token at `pos` of a one-layer model whose cache is `kv`, in 64 bits.  E is how far the
    engine's value may be from the one here.  A quantization whose argument is nearer to a tie than E may be to the next
    integer, else its error is that of the scale.  Each elementwise step adds a few roundings of 2^-24."""
    D, hd, H = shape.dim, shape.head_dim, shape.heads
    u = 2.0 ** -23

    def quantize(v, E):
        b, e = v.reshape(-1, 32), E.reshape(-1, 32)
        amax = np.abs(b).max(1, keepdims=True)
        d, ed = amax / 127, e.max(1, keepdims=True) / 127 + amax / 127 * u
        c = b / d
        ec = (e + np.abs(c) * ed) / d + 1e-5
        steps = np.where(np.abs(np.abs(c - np.trunc(c)) - 0.5) <= ec, np.ceil(ec), 0)
        return (np.rint(c) * d).reshape(-1), (np.abs(np.rint(c)) * ed + steps * (d + ed)).reshape(-1)

    def norm(x, E, w):
        ms = (x * x).mean() + shape.eps
        r = ms ** -0.5
        er = (np.abs(x) * E).mean() / ms + x.size * u
        return x * r * w, np.abs(w) * r * (E + np.abs(x) * er) + 4 * u * np.abs(x * r * w)

    raw = t["token_embd.weight"].data.reshape(shape.vocab, -1, 18)[token]
    x = oracle.embed_row(*synth.q4_0_blocks(raw)).astype(np.float64)
    # q exactly as the engine has it
    y = oracle.rmsnorm(x.astype(np.float32), t["blk.0.attn_norm.weight"].data, shape.eps)
    q = oracle.matvec_q4(t["blk.0.attn_q.weight"].data, D, D, y) + t["blk.0.attn_q.bias"].data
    cs = oracle.rope_table(ctx, hd, shape.rope_theta).reshape(ctx, hd)[pos]
    q = np.stack([oracle.rope_head(h, cs) for h in q.astype(np.float32).reshape(H, hd)])[None]
    n = pos + 1
    (K, ks), (V, vs) = kv
    att, E = kv8_ref.attend(q, K[:n], V[:n], ks[:n], vs[:n], pos, hd ** -0.5, 2.0 ** -24)
    o, E = quantize(att.reshape(-1), E.reshape(-1))
    x, E = x + o, E + u * np.abs(x + o)
    z, ez = norm(x, E, np.asarray(t["output_norm.weight"].data, np.float64))
    return quantize(z, ez)


@pytest.mark.parametrize("name", sorted(SHAPES))
def test_prompts_and_steps_of_one_layer(name):
    ctx, B, steps, seed = 200, 4, 5, 71
    shape, t, g = model(name, seed, ctx)
    rng = np.random.default_rng(seed)
    lens = [1, 40, 97, 150]
    prompts = [rng.integers(0, shape.vocab, n).astype(np.int32) for n in lens]
    bt = q4hip.Batch(g, B, kv8_pages=4 * 7)
    try:
        first = []
        for b, ids in enumerate(prompts):
            first.append(bt.prefill(b, ids, 0))
            kv = expected_kv(shape, t, ids, ctx, [(0, len(ids))])
            check_layer0(bt, b, shape, kv)
            lg = g.read_logits()
            assert first[b] == int(lg.argmax())
            want, E = carry(shape, t, ids[-1], len(ids) - 1, kv, ctx)
            assert (lg[shape.dim:] == 0).all()
            assert (np.abs(lg[:shape.dim] - want) <= E).all(), float((np.abs(lg[:shape.dim] - want) / E).max())
            assert E.max() < 0.1 * want.std()          # a bound that a wrong row or page breaks
        out = bt.generate(first, lens, steps)
        lg = bt.read_logits()
        for b, ids in enumerate(prompts):
            fed = list(ids) + [first[b]] + out[:-1, b].tolist()
            n = lens[b]
            kv = expected_kv(shape, t, fed, ctx, [(0, n)] + [(n + i, n + i + 1) for i in range(steps)])
            check_layer0(bt, b, shape, kv)
            assert out[-1, b] == int(lg[b].argmax())
            want, E = carry(shape, t, fed[-1], n + steps - 1, kv, ctx)
            assert (np.abs(lg[b, :shape.dim] - want) <= E).all(), (b, float((np.abs(lg[b, :shape.dim] - want) / E).max()))
    finally:
        bt.close()
        g.close()


@pytest.mark.parametrize("name", ["tiny", "small", "small128"])
def test_a_pool_shared_released_and_cut_back(name):
    """A prompt in passes of 16 tokens, a chat cut back and continued, a sequence that ends and one that takes its
    pages, and a pool that is too small: nothing changes then."""
    ctx = 160
    shape, t, g = model(name, 5, ctx, mt=16)
    rng = np.random.default_rng(9)
    ids = [rng.integers(0, shape.vocab, n).astype(np.int32) for n in (100, 33, 150)]
    bt = q4hip.Batch(g, 3, kv8_pages=6)
    try:
        bt.prefill(0, ids[0], 0)
        cuts = [(a, min(a + 16, 100)) for a in range(0, 100, 16)]
        check_layer0(bt, 0, shape, expected_kv(shape, t, ids[0], ctx, cuts))
        bt.prefill(1, ids[1], 0)
        assert bt.free_pages() == 0
        before = [bt.get_kv(b, 0, 0, 0, n) for b, n in ((0, 100), (1, 33))]
        for call in (lambda: bt.prefill(2, ids[2][:1], 0), lambda: bt.prefill(0, ids[0][:30], 100),
                     lambda: bt.generate([1, 2, 3], [100, 33, 0], 2)):
            with pytest.raises(q4hip.Q4Error) as e:
                call()
            assert e.value.code == q4hip.ECONTEXT
        after = [bt.get_kv(b, 0, 0, 0, n) for b, n in ((0, 100), (1, 33))]
        for x, y in zip(before, after):
            assert np.array_equal(x[0], y[0]) and np.array_equal(x[1], y[1])
        bt.prefill(0, ids[2][:5], 50)                   # cut back to 50 positions and continued
        assert bt.free_pages() == 2
        fed = np.concatenate([ids[0][:50], ids[2][:5]])
        # position 50 lies in the page of 48..63 of the old run: its scale and the codes before stay
        o = expected_kv(shape, t, np.concatenate([ids[0][:64]]), ctx, cuts[:4])
        k, _ = bt.get_kv(0, 0, 0, 0, 55)
        assert np.array_equal(k[:32], o[0][0][:32, 0])
        bt.release(1)
        assert bt.free_pages() == 4
        bt.prefill(2, ids[2][:120], 0)
        assert bt.free_pages() == 0
        check_layer0(bt, 2, shape, expected_kv(shape, t, ids[2][:120], ctx, [(a, min(a + 16, 120)) for a in range(0, 120, 16)]))
        k2, _ = bt.get_kv(0, 0, 0, 0, 55)
        assert np.array_equal(k, k2) and len(fed) == 55
        bt.release(0)
        bt.release(2)
        assert bt.free_pages() == 6
        x = bt.prefill(1, ids[1], 0)
        y = q4hip.Batch(g, 1, kv8_pages=2)
        assert y.prefill(0, ids[1], 0) == x              # which pages a sequence has makes no difference
        y.close()
    finally:
        bt.close()
        g.close()


def test_rows_from_the_host():
    """set_kv in pieces, every layer and head, read back to the bit; and what is refused."""
    shape, t, g = model("one64x4", 3, 150, mt=40)
    rng = np.random.default_rng(4)
    K, V = rng.standard_normal((2, 2, 110, 64), dtype=np.float32)
    bt = q4hip.Batch(g, 2, kv8_pages=6)
    try:
        ref = [kv8_ref.Cache(4, 2, 64) for _ in range(2)]
        for a, b in ((0, 70), (70, 110)):
            for h in range(2):
                bt.set_kv(1, 0, h, a, K[h, a:b], V[h, a:b])
        for c, x in zip(ref, (K, V)):
            for a, b in ((0, 70), (70, 110)):
                c.append(x[:, a:b].transpose(1, 0, 2), np.arange(a, b))
        for h in range(2):
            k, v = bt.get_kv(1, 0, h, 0, 110)
            assert np.array_equal(k, ref[0].values([0, 1, 2, 3], 110)[:, h])
            assert np.array_equal(v, ref[1].values([0, 1, 2, 3], 110)[:, h])
        k, v = bt.get_kv(1, 0, 1, 33, 7)
        assert np.array_equal(k, ref[0].values([0, 1, 2, 3], 110)[33:40, 1])

        def refused(code, call, *args):
            with pytest.raises(q4hip.Q4Error) as e:
                call(*args)
            assert e.value.code == code

        refused(q4hip.EINVAL, bt.set_kv, 1, 0, 0, 111, K[0, :2], V[0, :2])      # a gap
        refused(q4hip.EINVAL, bt.set_kv, 1, 0, 0, 10, K[0, :2], V[0, :2])       # before the end
        refused(q4hip.ECONTEXT, bt.set_kv, 0, 0, 0, 0, K[0, :70], V[0, :70])    # two pages are left
        refused(q4hip.ECONTEXT, bt.get_kv, 1, 0, 0, 100, 11)
        refused(q4hip.ECONTEXT, bt.get_kv, 0, 0, 0, 0, 1)
        refused(q4hip.EINVAL, bt.get_kv, 2, 0, 0, 0, 1)
        refused(q4hip.EINVAL, bt.get_kv, 1, 1, 0, 0, 1)
        refused(q4hip.EINVAL, bt.get_kv, 1, 0, 2, 0, 1)
        refused(q4hip.EINVAL, bt.release, 2)
        refused(q4hip.EINVAL, bt.prefill, 0, [1], 1)
        refused(q4hip.EINVAL, bt.generate, [1, 1], [1, 5], 1)
        refused(q4hip.EINVAL, q4hip.Batch, g, 2, -3)
        plain = q4hip.Batch(g, 1)
        refused(q4hip.EINVAL, plain.release, 0)
        refused(q4hip.EINVAL, plain.free_pages)
        refused(q4hip.EINVAL, plain.get_kv, 0, 0, 0, 0, 1)
        plain.close()
    finally:
        bt.close()
        g.close()


def test_other_batches_are_as_they_were():
    """A batch on the fp32 cache beside one on the 8-bit cache of the same context gives the oracle's tokens."""
    shape, t, g = model("small", 42, 96)
    rng = np.random.default_rng(6)
    prompts = [rng.integers(0, shape.vocab, n).astype(np.int32) for n in (12, 30)]
    o = oracle.Model(shape, t, ctx=96)
    a, b = q4hip.Batch(g, 2), q4hip.Batch(g, 2, kv8_pages=8)
    try:
        fa = [a.prefill(i, p, 0) for i, p in enumerate(prompts)]
        fb = [b.prefill(i, p, 0) for i, p in enumerate(prompts)]
        b.generate(fb, [12, 30], 3)
        out = a.generate(fa, [12, 30], 6)
        b.generate(fb, [12, 30], 3)
        for i, p in enumerate(prompts):
            assert [fa[i]] + out[:, i].tolist() == o.generate(p, 7)
    finally:
        a.close()
        b.close()
        g.close()
        o.close()


def test_through_napi(tmp_path):
    """createBatch(B, {kv8Pages}) through the addon: the tokens of the Python binding, pages given back, errors."""
    import os
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    shape = synth.SHAPES["tiny"]
    t = synth.make_model(shape, 8)
    path = str(tmp_path / "m.gguf")
    synth.write_gguf(path, shape, t)
    prompts = [synth.prompt_ids(90 + b, n, shape.vocab) for b, n in enumerate([9, 23, 40])]
    js = """
    const { LLM } = require(process.argv[1]);
    (async () => {
      const prompts = JSON.parse(process.argv[3]);
      const llm = await LLM.load({ path: process.argv[2], ctx: 128 });
      const bt = llm.be.createBatch(3, { kv8Pages: 6 });
      const first = [];
      for (let b = 0; b < 3; b++) first.push(await bt.prefill(b, prompts[b], 0));
      const free = [bt.freePages()];
      const tokens = await bt.generate(first, prompts.map((p) => p.length), 8);
      free.push(bt.freePages());
      let full = null, bad = null;
      try { await bt.generate(first, [9 + 8, 23 + 8, 40 + 8], 40); } catch (e) { full = e.message; }
      try { llm.be.createBatch(3, { kv8Pages: 0 }); } catch (e) { bad = e.message; }
      bt.release(2);
      free.push(bt.freePages());
      llm.destroy();
      process.stdout.write(JSON.stringify({ first, tokens, free, full, bad }));
    })().catch((e) => { process.stderr.write(String(e.stack)); process.exit(1); });
    """
    run = subprocess.run(["node", "-e", js, os.path.join(repo, "e2e-browser-voice-agent_amd", "engine", "llm.js"), path,
                          json.dumps([list(map(int, p)) for p in prompts])], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stderr
    out = json.loads(run.stdout)
    g = q4hip.Model(shape, ctx=128)
    g.load(t)
    bt = q4hip.Batch(g, 3, kv8_pages=6)
    first = [bt.prefill(b, p, 0) for b, p in enumerate(prompts)]
    tokens = bt.generate(first, [len(p) for p in prompts], 8)
    assert out["first"] == first and out["tokens"] == tokens.T.tolist()
    assert out["free"] == [2, 2, 4] and "cache full" in out["full"] and "0 pages" in out["bad"]
    bt.close()
    g.close()
