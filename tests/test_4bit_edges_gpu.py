"""A cache in 4 bits on the GPU, at its edges: tokens that have no place, scores far from zero, single tokens of every head size from attention to
sums.  The tolerances are those of tests/test_4bit_gpu.py."""


import pytest
import torch

import plain_4bit as p4
import test_4bit_gpu as t4
from test_4bit_gpu import BF16, F32, ops  # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("copies", [1, 400])
@pytest.mark.parametrize("dtype,D", [(F32, 64), (BF16, 80)])
@pytest.mark.parametrize("window", [None, 300])
def test_a_token_without_a_place_is_zero(ops, copies, dtype, D, window):  # noqa: F811
    """A token of no sequence, or whose place lies behind or in front of the table, sees nothing, whether a block goes through its slices
    or a second kernel joins them (few tokens); the others are as ever."""
    H, G, lens = 4, 2, [700, 700, 1100, 700, 900]
    c = p4.Cache(lens, G, D, 16, seed=D)
    n, new = len(lens) * copies, [1] * len(lens) * copies
    q = t4.queries(n, H, D, 3, dtype)
    table = c.table.repeat(copies, 1)
    args = dict(dtype=dtype, table=table, window=window)
    want = t4.attend(ops, c, q, new, lens * copies, H, D ** -0.5, **args)
    step = p4.step_of(new, lens * copies, 16)
    step.token_seq[0], step.token_seq[1] = -1, n
    step.positions[2], step.positions[3] = table.shape[1] * 16, -2
    got = t4.attend(ops, c, q, new, lens * copies, H, D ** -0.5, step=step, **args)
    assert bool((got[:4] == 0).all()) and torch.equal(got[4:], want[4:])
