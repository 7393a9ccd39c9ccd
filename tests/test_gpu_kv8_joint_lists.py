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
