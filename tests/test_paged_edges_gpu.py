"""Edges of the paged operators on the GPU: owners of one tile between owners of two, keys that are not finite, sizes of plans.
Tolerances as in test_paged_gpu.py."""

import subprocess
import sys
from pathlib import Path

import pytest
import torch

import nanochat_b200 as ncb
from tests import paged_cases as plain
from tests.test_paged_gpu import DTYPES, PAGE, Pool, run_attention, words

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


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("new", [3, 20, 150])  # the small kernel; both tiles with the rows; rows of their own
def test_keys_that_are_not_finite_reach_their_rows(dtype, new, value):
    """A key in one of two inner pages with such a value in one dimension, at each position of eight: rows whose score is NaN or infinite are NaN, as
    in 64 bits, others leave the key out (a score of minus infinity) or have another head."""
    if dtype != torch.bfloat16 and value == float("inf"):
        pytest.skip("a code of e4m3 is never infinite")
    n, dim = 400 + new, 5
    pool = Pool(dtype, 8, 2, [n], [new], seed=new)
    page, kept = pool.pages.table[0].tolist(), pool.cache.pages.clone()
    for at in [128 + j for j in range(8)] + [192 + 16 + j for j in range(8)]:
        if dtype == torch.bfloat16:
            pool.cache.pages[page[at // PAGE], 1, 0, at % PAGE, dim] = value
        else:
            j = at % PAGE
            pool.cache.pages[page[at // PAGE], 1, j * 128 + (((dim >> 4) ^ ((j >> 2) & 7)) << 4) + (dim & 15)] = 0x7f
        k = pool.cache.read(words(page), n)[0].double()
        assert k[1, at, dim].isnan() if value != value else k[1, at, dim].isinf()
        out = ncb.paged_attention(pool.q, pool.cache, pool.plan)[:new]
        want, size = plain.attention(pool.q[:new].double(), k, pool.v[0], n - new, 0)
        bad = want.isnan()
        same = torch.equal(out.isnan(), bad)
        assert same and bad[:, 4:].any() and not bad[:, :4].any(), at
        rounding = 2.0 ** -11 if pool.cache.e4m3 else 2.0 ** -8
        off = (out.double() - want).abs() - 2.0 ** -8 * want.abs() - (rounding + 2.0 ** -14) * size
        assert off[~bad].max().item() <= 0, at
        pool.cache.pages.copy_(kept)


def test_plans_of_every_number_of_requests():
    """Around the number whose shared memory passes 48 KB with and without what the kernel has besides, in a process that has made no larger plan."""
    done = subprocess.run([sys.executable, "-c", """
import torch, nanochat_b200 as ncb
for n in (2437, 2438, 2450, 2457, 2458, 2459):
    pages = ncb.PageTable(n, n, 64)
    plan = ncb.page_plan(pages, pages.lens, torch.ones(n, dtype=torch.int32, device="cuda"), n, max_new=1, Hq=4, Hkv=4)
    assert plan.pos.eq(0).all() and plan.place.tolist() == [64 * b for b in range(n)], n
"""], cwd=Path(__file__).parent.parent, capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr[-2000:]
