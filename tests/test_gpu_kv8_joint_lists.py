"""The lists of a step whose sequences begin with the same pages."""
import numpy as np
import pytest
import torch

import q4hip
from test_gpu_kv8 import ints
from test_gpu_kv8_joint import grown, join_all  # noqa: F401  (a fixture for all tests)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seqs", [20, 1100])       # the plan's sums in shared memory, and in global
def test_lengths_in_the_plans_own_results(seqs):
    """The caller's lengths lie where the plan writes its results to: all launches count with what the first one has read."""
    rng = np.random.default_rng(seqs)
    t, lens = grown(rng, 4, 1, 64, [(300, seqs)], "f32", own=20, max_rows=30000)
    t.grow(rng, lens, [1] * seqs)
    t.attend(rng, "f32")
    lens = [n + 1 for n in lens]
    first, second = ints(lens + [0]), ints([1] * seqs)
    torch.cuda.synchronize()
    t.kv.plan(first.data_ptr(), second.data_ptr(), seqs, starts=first.data_ptr(), positions=second.data_ptr())
    t.have, t.add = lens, [1] * seqs
    starts, positions, t.slots, _, t.seq = t.pool.plan(lens, [1] * seqs, seqs)
    assert np.array_equal(first.cpu(), starts) and np.array_equal(second.cpu(), positions)
    t.fill(rng, "f32")
    t.check_values()
    t.attend(rng, "f32")


def joints_of(t, room=256):
    """Joints that a step has: 32 rows of attention each, of the sequences with the same first page that add up to 16 heads' rows and
    have 8 pages and more in common before these.  A group that there is no room for has none, nor have those behind it; nor has a cache
    of more than 16 heads to a kv head."""
    G = t.H // t.KVH
    if G > 16:
        return 0
    unit = max(1, 16 // G)
    room = min(room, (t.B * unit * G + 31) // 32 + t.B // 2)
    groups = {}
    for b, (h, a) in enumerate(zip(t.have, t.add)):
        if 0 < a <= unit and h // 32 >= 8:
            groups.setdefault(t.pool.tables[b][0], []).append(b)
    joints = at = 0
    for g in groups.values():                       # in the order of their first sequences
        first = t.pool.tables[g[0]]
        common = min(t.have[b] // 32 for b in g)
        for b in g:
            own = t.pool.tables[b]
            while own[:common] != first[:common]:
                common -= 1
        if len(g) > 1 and common >= 8:
            n = -(-sum(t.add[b] for b in g) * G // 32)
            at += n
            joints += n if at <= room else 0
    return joints


def step(t, rng, have, add, dtype, joints=None):
    t.grow(rng, have, add, dtype)
    want = joints_of(t)
    assert joints is None or want == joints
    shared, got = t.kv.shared()
    assert shared == any(n > 1 for n in t.pool.holders()) and got == (want if shared and sum(add) > 1 else 0)
    t.attend(rng, dtype)
    return got


@pytest.mark.parametrize("H,KVH,hd,prefixes,joints", [
    (14, 2, 64, [(300, 2)], 1), (16, 1, 64, [(256, 5), (999, 3)], 5), (4, 1, 128, [(289, 33)], 5), (3, 3, 64, [(480, 70), (257, 30)], 4),
    (4, 1, 64, [(300, 1100)], 138), (16, 1, 64, [(256, 40)], 20), (2, 1, 64, [(255, 20)], 0), (8, 1, 64, [(300, 1)], 0)])
def test_joints_of_a_token_each(H, KVH, hd, prefixes, joints):
    rng = np.random.default_rng(H + hd)
    t, lens = grown(rng, H, KVH, hd, prefixes, "bf16", own=3)
    step(t, rng, lens, [1] * t.B, "bf16", joints)
    t.check_values()


@pytest.mark.parametrize("H,prefixes,joints", [
    (16, [(256, 300), (288, 300)], 150),            # the second does not fit behind the first
    (16, [(256, 600), (288, 20)], 0),               # nor does what is behind one that does not
    (16, [(256, 512)], 256), (16, [(256, 514)], 0),     # as many as there are, and one more
    (16, [(256, 700), (288, 400)], 0), (16, [(256, 400), (288, 700)], 200)])       # of more than 1,024 sequences
def test_groups_without_room(H, prefixes, joints):
    """They are attended to one by one beside those that fit."""
    rng = np.random.default_rng(sum(n for _, n in prefixes))
    t, lens = grown(rng, H, 1, 64, prefixes, "bf16", own=3)
    step(t, rng, lens, [1] * t.B, "bf16", joints)


@pytest.mark.parametrize("seqs", [15, 1050])
@pytest.mark.parametrize("H,KVH", [(2, 2), (10, 2), (20, 1)])
def test_joints_of_rows_of_every_kind(H, KVH, seqs):
    """Sequences that add no row, one, up to a unit's and more."""
    rng = np.random.default_rng(H + seqs)
    t, lens = grown(rng, H, KVH, 64, [(480, seqs * 3 // 5), (257, seqs * 2 // 5)], "bf16", own=20, spare=2, max_rows=20 * seqs + 4000)
    unit = max(1, 16 * KVH // H)
    found = 0
    for _ in range(3):
        add = rng.choice([0, 1, 1, min(2, unit), unit, unit + 1, 40], t.B, p=[0.2, 0.3, 0.2, 0.1, 0.14, 0.04, 0.02])
        found += step(t, rng, lens, add.tolist(), "bf16")
        lens = [n + int(a) for n, a in zip(lens, add)]
    assert found or H > 16


def test_joints_of_forks_of_forks():
    """What all sequences with one first page have in common counts, and where that is too little there are none."""
    rng = np.random.default_rng(17)
    B = 12
    t = grown(rng, 4, 2, 64, [(700, 1)], "f32", own=0, spare=B - 1)[0]
    t.fork([0] * B, [700] * 6 + [600] * 3 + [330] * 3)
    lens = [700] * 6 + [600] * 3 + [330] * 3
    assert step(t, rng, lens, [1] * B, "f32") == 1
    t.fork(list(range(B)), [701] * 6 + [601] * 3 + [331] * 2 + [100])
    lens = [701] * 6 + [601] * 3 + [331] * 2 + [100]
    assert step(t, rng, lens, [1] * B, "f32") == 1        # the last one takes part in none
    t.fork([0, 1, 2, 3, 4, 5, 0, 0, 8, 9, 9, 9], [702] * 6 + [702, 702, 602, 332, 200, 300])
    step(t, rng, [702] * 6 + [702, 702, 602, 332, 200, 300], [1] * B, "f32")


def test_no_joints():
    """None without a page in common, behind a step without rows, after a plan that failed and after a fork."""
    rng = np.random.default_rng(18)
    t, lens = grown(rng, 8, 1, 64, [(300, 8)], "f32", own=5)
    assert step(t, rng, lens, [1] * 8, "f32") == 2
    lens = [n + 1 for n in lens]
    t.plan(lens, [0] * 8)
    assert t.kv.shared() == (True, 0)
    assert step(t, rng, lens, [1] * 8, "f32") == 2
    h, a = ints([-1] * 8), ints([1] * 8)
    torch.cuda.synchronize()
    with pytest.raises(q4hip.Q4Error):
        t.kv.plan(h.data_ptr(), a.data_ptr(), 8)
    assert t.kv.shared() == (True, 0)
    lens = [n + 1 for n in lens]
    assert step(t, rng, lens, [1] * 8, "f32") == 2
    t.fork(list(range(8)), [lens[0]] + [0] * 7)
    assert t.kv.shared() == (False, 0)
    t.grow(rng, [0] * 8, [400] * 8)
    assert t.kv.shared() == (False, 0)
    t.grow(rng, [400] * 8, [1] * 8)
    assert t.kv.shared() == (False, 0)
    t.attend(rng, "f32")


@pytest.mark.parametrize("H,KVH,hd,positions,seqs,own,joins", [
    (16, 8, 64, 1200, 64, 40, False),               # 17,760 pages of 64 columns, 8,880, and a round of workgroups more
    (16, 8, 64, 1200, 16, 40, False), (16, 8, 64, 1200, 24, 40, True),      # 2,220 and 3,256, no round more
    (4, 2, 64, 3000, 30, 40, False), (4, 2, 64, 3000, 34, 40, False), (4, 2, 64, 3000, 36, 40, True),     # 2,604, 2,883, 3,069
    (4, 2, 64, 3000, 20, 40, False), (4, 2, 128, 3000, 20, 40, True),       # 1,674, 3,348
    (16, 1, 64, 300, 2, 5, False)])
def test_what_it_has_to_save(monkeypatch, H, KVH, hd, positions, seqs, own, joins):
    """Pages of 128 columns: 3,000, and 8,000 for each further round of 512 items."""
    monkeypatch.delenv("Q4HIP_KV8_JOINT_SAVES")
    rng = np.random.default_rng(positions)
    t, lens = grown(rng, H, KVH, hd, [(positions, seqs)], "bf16", own=own)
    t.grow(rng, lens, [1] * seqs, "bf16")
    want = joints_of(t)
    assert want and t.kv.shared() == (True, want if joins else 0)
    t.attend(rng, "bf16")
