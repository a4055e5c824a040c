"""Edges of the paged operators on the GPU: owners of one tile between owners of two, keys that are not finite, sizes of plans, lengths that go back, closer bounds.
Tolerances as in test_paged_gpu.py."""

import subprocess
import sys
from pathlib import Path

import numpy as np
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


def give_back(table, free, held, keep):
    """trim (release: keep 0) on lists: the entries behind min(keep, held) positions, a request's last page first."""
    for row, n, k in zip(table, held, keep):
        first, end = -(-min(k, n) // PAGE), min(-(-n // PAGE), len(row))
        free += reversed(row[first:end])
        row[first:end] = [-1] * (end - first)


def check_pages(pages, table, free, lens):
    """The device's table is the lists', and every page is a request's or free, once."""
    assert pages.table.tolist() == table and pages.lens.tolist() == lens
    count = pages.free_count.item()
    assert pages.free[:count].tolist() == free
    held = [p for row in table for p in row if p >= 0]
    assert sorted(held + free) == list(range(pages.n_pages)) and len(held) == sum(-(-n // PAGE) for n in lens)


@pytest.mark.parametrize("in_place", [True, False])
def test_rejected_drafts_lose_no_page(in_place):
    """Steps of up to 70 drafts of which some stay, across borders of pages, with requests that come and go: by default the plan advances the table."""
    n, n_pages, width = 40, 120, 6
    rng = np.random.default_rng(7)
    pages, status = ncb.PageTable(n_pages, n, width * PAGE), words([0])
    table, free, lens = [[-1] * width for _ in range(n)], list(range(n_pages - 1, -1, -1)), [0] * n
    for step in range(60):
        drafts = np.where(rng.random(n) < 0.2, rng.integers(0, 70, n), rng.integers(0, 6, n))
        new = np.minimum(drafts, [width * PAGE - x for x in lens]).tolist()
        want, bits = plain.plan(table, lens, new, free, sum(new), 70)
        plan = ncb.page_plan(pages, pages.lens, words(new), sum(new), max_new=70, Hq=4, Hkv=2, lens=pages.lens if in_place else None, status=status)
        assert status.item() == bits and plan.lens.tolist() == want["lens"] and plan.place.tolist() == want["place"]
        status.zero_()
        table, free, now = want["table"], free[:want["left"]], want["lens"]
        check_pages(pages, table, free, now)
        keep = [int(rng.integers(a, b + 1)) for a, b in zip(lens, now)]
        pages.trim(words(keep), status=status)
        give_back(table, free, now, keep)
        lens = keep
        check_pages(pages, table, free, lens)
        done = [int(rng.random() < 0.1) for _ in range(n)]
        pages.release(words(done), status=status)
        give_back(table, free, lens, [0 if d else x for d, x in zip(done, lens)])
        lens = [0 if d else x for d, x in zip(done, lens)]
        check_pages(pages, table, free, lens)
        assert status.item() == 0
    pages.trim(words([0] * n))
    assert pages.free_count.item() == n_pages and not pages.lens.any() and (pages.table == -1).all()


def test_trim_keeps_no_more_than_there_is():
    pages, status = ncb.PageTable(30, 5, 5 * PAGE), words([0])
    ncb.page_plan(pages, pages.lens, words([300, 64, 65, 0, 128]), 557, max_new=300, Hq=4, Hkv=4)
    before = pages.table.tolist()
    pages.trim(words([301, 2 ** 31 - 1, 300, 9, 128]), status=status)  # nothing goes back
    assert pages.lens.tolist() == [300, 64, 65, 0, 128] and pages.table.tolist() == before and pages.free_count.item() == 30 - 10 and status.item() == 0
    pages.trim(words([-1, 63, 64, 0, -2 ** 31]), status=status)  # negative ones are flagged and keep all
    assert pages.lens.tolist() == [300, 63, 64, 0, 128] and status.item() == 4 and pages.free_count.item() == 30 - 9
    assert pages.table.tolist() == [before[0], before[1], [before[2][0], -1, -1, -1, -1], before[3], before[4]]
    pages.trim(pages.lens)
    assert pages.lens.tolist() == [300, 63, 64, 0, 128] and pages.free_count.item() == 30 - 9
    pages.table[0, 4] = 30  # outside the pool
    status.zero_()
    pages.trim(words([256, 0, 64, 0, 0]), status=status)
    assert status.item() == 16 and pages.lens.tolist() == [256, 0, 64, 0, 0] and pages.free_count.item() == 30 - 5 - 1
    assert sorted(pages.free[:24].tolist()) == sorted(set(range(30)) - set(before[0][:4]) - {before[2][0]} - {before[0][4]})


def test_a_captured_step_of_drafts():
    """Plan, append, attention and trim in one graph, replayed, against the same eager steps."""
    Hq, Hkv, gen = 4, 2, torch.Generator().manual_seed(29)
    cos, sin = ncb.rotary_table(6 * PAGE, 1e4, "cuda")
    gain = torch.ones(128, device="cuda")

    class Side:
        def __init__(self):
            self.pages, self.cache, self.status = ncb.PageTable(30, 4, 6 * PAGE), ncb.PagedKVCache(30, Hkv, torch.bfloat16), words([0])
            self.new, self.rejected = words([0] * 4), words([0] * 4)
            self.qkv, self.plan, self.out = torch.zeros(80, (Hq + 2 * Hkv) * 128, dtype=torch.bfloat16, device="cuda"), None, None

        def step(self):
            self.plan = ncb.page_plan(self.pages, self.pages.lens, self.new, 80, max_new=20, Hq=Hq, Hkv=Hkv, plan=self.plan, status=self.status)
            q = ncb.paged_append(self.qkv, gain, gain, cos, sin, self.plan.pos, self.plan.place, self.cache, Hq, status=self.status)
            self.out = ncb.paged_attention(q, self.cache, self.plan, status=self.status)
            self.pages.trim(self.pages.lens - self.rejected, status=self.status)

    eager, captured = Side(), Side()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        captured.step()  # first-use set-up, all requests idle
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured.step()
    torch.cuda.current_stream().wait_stream(side)
    rng = np.random.default_rng(3)
    for i in range(40):
        new = rng.integers(0, 21, 4)
        back = np.minimum(new, rng.integers(0, 21, 4))
        x = torch.randn(80, (Hq + 2 * Hkv) * 128, generator=gen).bfloat16().cuda()
        for s in (eager, captured):
            s.new.copy_(words(new.tolist()))
            s.rejected.copy_(words(back.tolist()))
            s.qkv.copy_(x)
        eager.step()
        graph.replay()
        assert torch.equal(eager.out[:new.sum()], captured.out[:new.sum()])
        assert torch.equal(eager.pages.table, captured.pages.table) and torch.equal(eager.pages.lens, captured.pages.lens)
        held = sum(-(-n // PAGE) for n in eager.pages.lens.tolist())
        assert eager.pages.free_count.item() == captured.pages.free_count.item() == 30 - held
    assert eager.status.item() == captured.status.item() == 0


@pytest.mark.parametrize("width", [1, 40])
@pytest.mark.parametrize("heads", [(4, 4), (8, 2), (12, 1), (16, 1)])
def test_few_slots_keep_both_terms_of_their_probabilities(heads, width):
    lens, new = [200, 131, 64, 1, 900], [1, 1, 1, 1, 1] if heads[1] == 1 else [1, 2, 4, 1, 3]
    pool, plan, q, out = run_attention(torch.bfloat16, *heads, lens, new, seed=19, width=width)
    at = 0
    for b, (n, k) in enumerate(zip(lens, new)):
        want, size = plain.attention(q[at:at + k].double(), pool.k[b], pool.v[b], n - k, 0)
        assert ((out[at:at + k].double() - want).abs() <= plain.few_slots_bound(want, size)).all()
        at += k


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [(8, 2), (2, 2), (16, 1)])
@pytest.mark.parametrize("new", [1, 4, 20, 33, 150])
def test_rows_beside_what_they_do_not_see(dtype, heads, new):
    """A key and a value that are not finite, behind some rows or left behind by their window: the other rows are right, within the bounds of clean calls."""
    Hq, Hkv = heads
    n = 200 + new
    for window, at, clean in ((0, n - 2, range(0, new - 2)), (50, n - new - 49, range(1, new)), (0, n - 1, range(0, new - 1)), (50, 100, range(0, new)), (64, 3, range(0, new))):
        pool = Pool(dtype, Hq, Hkv, [n], [new], window=window, seed=13)
        if pool.cache.e4m3:
            nan, inf = torch.full((Hkv, 1, 128), 0x7f, dtype=torch.uint8), torch.full((Hkv, 1), float("inf"))
            pool.cache.write(words(pool.table[0]), nan, nan, inf, inf, start=at)
        else:
            v = torch.full((Hkv, 1, 128), float("nan"), dtype=torch.bfloat16)
            v[..., ::2] = float("inf")
            pool.cache.write(words(pool.table[0]), torch.full_like(v, float("inf")), v, start=at)
        out = ncb.paged_attention(pool.q, pool.cache, pool.plan, window=window)
        rounding = 2.0 ** -11 if pool.cache.e4m3 else 2.0 ** -8
        for i in clean:
            want, size = plain.attention(pool.q[i:i + 1].double(), pool.k[0], pool.v[0], n - new + i, window)
            off = (out[i:i + 1].double() - want).abs() - 2.0 ** -8 * want.abs() - (rounding + 2.0 ** -14) * size
            assert off.max().item() <= 0, (window, at, i)
