"""Batches on the paged 8-bit cache: sequences that sit a call out.  Models and references are those of test_gpu_batch_kv8.py."""
import numpy as np
import pytest

import q4hip
import synth
from test_gpu_batch_kv8 import carry, check_layer0, expected_kv, model

pytestmark = pytest.mark.gpu


def all_kv(bt, seq, shape, n):
    return [bt.get_kv(seq, l, g, 0, n) for l in range(shape.layers) for g in range(shape.kv_heads)]


def same(x, y):
    return all(np.array_equal(a, b) for p, q in zip(x, y) for a, b in zip(p, q))


@pytest.mark.parametrize("name", ["one64", "one128", "one64x4"])
def test_ended_and_paused_sequences_sit_out(name):
    """A full pool: sequence 1 has ended, 2 is paused, 4 was never used.  The others step, as the references have it; then 2
    goes on from where it was."""
    ctx, steps, seed = 200, 6, 23
    shape, t, g = model(name, seed, ctx)
    rng = np.random.default_rng(seed)
    lens = [40, 60, 33, 62]
    prompts = [rng.integers(0, shape.vocab, n).astype(np.int32) for n in lens]
    bt = q4hip.Batch(g, 5, kv8_pages=8)                # 2 + 2 + 2 + 2
    try:
        first = [bt.prefill(b, ids, 0) for b, ids in enumerate(prompts)] + [0]
        assert bt.free_pages() == 0
        bt.release(1)
        paused = all_kv(bt, 2, shape, 33)
        out = bt.generate([first[0], -5, shape.vocab, first[3], 0], [40, -1, -1, 62, -1], steps)
        assert bt.free_pages() == 1                    # 62 + 6 positions take a third page
        assert (out[:, [1, 2, 4]] == -1).all() and (out[:, [0, 3]] >= 0).all()
        assert same(paused, all_kv(bt, 2, shape, 33))
        for b in (1, 4):
            with pytest.raises(q4hip.Q4Error):
                bt.get_kv(b, 0, 0, 0, 1)
        lg = bt.read_logits()

        def check(b, fed, cuts, logits):
            kv = expected_kv(shape, t, fed, ctx, cuts)
            check_layer0(bt, b, shape, kv)
            want, E = carry(shape, t, fed[-1], len(fed) - 1, kv, ctx)
            assert (np.abs(logits[:shape.dim] - want) <= E).all(), b

        fed = {}
        for b in (0, 3):
            n = lens[b]
            fed[b] = list(prompts[b]) + [first[b]] + out[:-1, b].tolist()
            check(b, fed[b], [(0, n)] + [(n + i, n + i + 1) for i in range(steps)], lg[b])
            assert out[-1, b] == int(lg[b].argmax())
        # 2 goes on, the others sit out: their logits stay
        more = bt.generate([0, 0, first[2], 0, 0], [-1, -1, 33, -1, -1], 2)
        lg2 = bt.read_logits()
        check(2, list(prompts[2]) + [first[2], more[0, 2]], [(0, 33), (33, 34), (34, 35)], lg2[2])
        assert np.array_equal(lg2[[0, 3]], lg[[0, 3]]) and (more[:, [0, 1, 3, 4]] == -1).all()
        # and all that are there together, from where each is
        last = bt.generate([int(out[-1, 0]), 0, int(more[-1, 2]), int(out[-1, 3]), 7], [46, -1, 35, 68, -1], 1)
        lg3 = bt.read_logits()
        n = 40
        check(0, fed[0] + [int(out[-1, 0])], [(0, n)] + [(n + i, n + i + 1) for i in range(steps + 1)], lg3[0])
        assert last[0, 1] == -1 and last[0, 0] == int(lg3[0].argmax())
        for pos in ([-1] * 5, [46, -1, 36, 70, -1], [-2, -1, 36, 69, -1], [47, -1, 36, 69, 1]):
            with pytest.raises(q4hip.Q4Error):
                bt.generate([1] * 5, pos, 1)
        assert bt.time_generate([1] * 5, [47, -1, -1, -1, -1], 2)[0].shape == (2, 5)
    finally:
        bt.close()
        g.close()


@pytest.mark.parametrize("seq", [0, 1, 2])
def test_one_of_three(seq):
    """Two of three sit out; the third gives what it gives in a batch of its own."""
    shape, t, g = model("small", 4, 96)
    ids = np.random.default_rng(1).integers(0, shape.vocab, 20).astype(np.int32)
    a, b = q4hip.Batch(g, 3, kv8_pages=6), q4hip.Batch(g, 1, kv8_pages=2)
    try:
        x, y = a.prefill(seq, ids, 0), b.prefill(0, ids, 0)
        pos = [-1] * 3
        pos[seq] = 20
        p, q = a.generate([x] * 3, pos, 9), b.generate([y], [20], 9)
        assert x == y and np.array_equal(p[:, seq], q[:, 0])
        assert np.array_equal(a.read_logits()[seq], b.read_logits()[0])
        assert same(all_kv(a, seq, shape, 29), all_kv(b, 0, shape, 29))
    finally:
        a.close()
        b.close()
        g.close()


def test_other_caches_have_no_idle_sequences():
    shape, t, g = model("tiny", 4, 96)
    bt = q4hip.Batch(g, 2)
    try:
        with pytest.raises(q4hip.Q4Error) as e:
            bt.generate([1, 1], [0, -1], 1)
        assert e.value.code == q4hip.ECONTEXT
    finally:
        bt.close()
        g.close()


def test_through_napi(tmp_path):
    """generate with pos -1 through createBatch: an empty array of the one that sits out, the other's tokens as in Python."""
    import json
    import os
    import subprocess
    repo = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    shape = synth.SHAPES["tiny"]
    t = synth.make_model(shape, 8)
    path = str(tmp_path / "m.gguf")
    synth.write_gguf(path, shape, t)
    ids = [int(i) for i in synth.prompt_ids(90, 9, shape.vocab)]
    js = """
    const { LLM } = require(process.argv[1]);
    (async () => {
      const ids = JSON.parse(process.argv[3]);
      const llm = await LLM.load({ path: process.argv[2], ctx: 128 });
      const bt = llm.be.createBatch(2, { kv8Pages: 4 });
      await bt.prefill(0, ids, 0);
      const first = await bt.prefill(1, ids, 0);
      bt.release(0);
      const tokens = await bt.generate([0, first], [-1, ids.length], 8);
      process.stdout.write(JSON.stringify({ first, tokens, free: bt.freePages() }));
      llm.destroy();
    })().catch((e) => { process.stderr.write(String(e.stack)); process.exit(1); });
    """
    run = subprocess.run(["node", "-e", js, os.path.join(repo, "e2e-browser-voice-agent_amd", "engine", "llm.js"), path,
                          json.dumps(ids)], capture_output=True, text=True, timeout=120)
    assert run.returncode == 0, run.stderr
    out = json.loads(run.stdout)
    g = q4hip.Model(shape, ctx=128)
    g.load(t)
    bt = q4hip.Batch(g, 1, kv8_pages=4)
    first = bt.prefill(0, ids, 0)
    assert out == {"first": first, "tokens": [[], bt.generate([first], [9], 8)[:, 0].tolist()], "free": 3}
    bt.close()
    g.close()


@pytest.mark.parametrize("first,then", [(70, 40), (64, 3), (5, 1)])
def test_positions_that_no_row_has_reached_are_zeros(first, then):
    """set_kv of one layer and head on pages that another sequence has held: zeros in all others, until they are set; what the
    head itself holds is as without them."""
    import kv8_ref
    shape, t, g = model("small", 3, 150)
    rng = np.random.default_rng(4)
    n = first + then
    K, V = rng.standard_normal((2, n, shape.head_dim), dtype=np.float32)
    bt = q4hip.Batch(g, 2, kv8_pages=-(-n // 32))
    try:
        bt.prefill(0, rng.integers(0, shape.vocab, n).astype(np.int32), 0)
        bt.release(0)
        last, head = shape.layers - 1, shape.kv_heads - 1
        ref = [kv8_ref.Cache(-(-n // 32), 1, shape.head_dim) for _ in range(2)]
        table = list(range(-(-n // 32)))
        for a, b in ((0, first), (first, n)):
            bt.set_kv(1, last, head, a, K[a:b], V[a:b])
            for l in range(shape.layers):
                for h in range(shape.kv_heads):
                    k, v = bt.get_kv(1, l, h, 0, b)
                    if (l, h) != (last, head):
                        assert (k == 0).all() and (v == 0).all(), (l, h)
            for c, x in zip(ref, (K, V)):
                c.append(x[a:b, None], np.arange(a, b))
            k, v = bt.get_kv(1, last, head, 0, b)
            assert np.array_equal(k, ref[0].values(table, b)[:, 0]) and np.array_equal(v, ref[1].values(table, b)[:, 0])
        # the others afterwards, up to the end
        bt.set_kv(1, 0, 0, first, K[first:], V[first:])
        k, _ = bt.get_kv(1, 0, 0, 0, n)
        assert (k[:first] == 0).all()
        step = np.abs(K[first:]).max() / 127
        assert (np.abs(k[first:] - K[first:]) <= step).all()
        k, _ = bt.get_kv(1, last, head, 0, n)
        assert np.array_equal(k, ref[0].values(table, n)[:, 0])
    finally:
        bt.close()
        g.close()


def test_a_pool_of_no_pages_is_refused():
    shape, t, g = model("tiny", 4, 96)
    try:
        with pytest.raises(q4hip.Q4Error) as e:
            q4hip.Batch(g, 1, kv8_pages=0)
        assert e.value.code == q4hip.EINVAL
        bt = q4hip.Batch(g, 1, kv8_pages=None)
        with pytest.raises(q4hip.Q4Error):
            bt.free_pages()
        bt.close()
    finally:
        g.close()
