"""Edges of the paged operators on the GPU: owners of one tile between owners of two.
Tolerances as in test_paged_gpu.py."""

import pytest
import torch

import nanochat_b200 as ncb
from tests import paged_cases as plain
from tests.test_paged_gpu import DTYPES, run_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [0, 100])
@pytest.mark.parametrize("seed", [1, 2, 3])
def test_owners_of_one_tile_between_owners_of_two(dtype, window, seed):
    """A tile without rows in some pieces passes over their pages, and its next border page is in a place that only the other tile has used.
    Short contexts and a long one, so that owners are cut; what no request wrote is NaN."""
    short = [(200 + 13 * i, 20 + i % 7) if i % 3 else (250 + 11 * i, 60 - i % 5) for i in range(24)]
    lens, new = ([n for n, _ in short] + [20000], [k for _, k in short] + [45])
    pool, plan, q, out = run_attention(dtype, 8, 2, lens, new, window=window, seed=seed)
    if window == 0:
        (_, _, _, _, (total, share, whole), owners, _, _, _), = [c for c in plain.schedule(
            plan.work.tolist(), len(lens), plan.rows, plan.max_new, 4, plan.blocks) if c[3] == 8]
        assert not whole and plan.max_new > 32  # cut, and two different tiles
    for _ in range(20):
        assert torch.equal(ncb.paged_attention(q, pool.cache, plan, window=window)[:sum(new)], out[:sum(new)])
