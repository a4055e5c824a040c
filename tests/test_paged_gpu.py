"""The paged cache on the GPU: page plans against a loop over requests, appends bit for bit against kv_append, attention against 64
bits, and steps of them together.

Tolerances of attention, per output o with A = sum of p |v|: the result's rounding to bf16 is at most 2^-8 |o|; a probability that enters
the product with values as f16 (e4m3 pages) is off by 2^-11 at most, as one bf16 term (bf16 pages) by 2^-8; scores and sums in fp32 over 128
products of values near 1 and exp2 add under 2^-14 of A. So 2^-8 |o| + (2^-11 + 2^-14) A, or 2^-8 in place of 2^-11."""

import numpy as np
import pytest
import torch

import nanochat_b200 as ncb
from nanochat_b200 import native
from tests import paged_cases as plain

pytestmark = pytest.mark.gpu
PAGE = 64


def words(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def make_table(cached, n_pages, width, free=None, seed=0, extra=0):
    """A table whose requests hold `cached` positions in shuffled pages; the rest is free."""
    gen = torch.Generator().manual_seed(seed)
    order = torch.randperm(n_pages, generator=gen).tolist()
    table = [[-1] * width for _ in cached]
    for b, c in enumerate(cached):
        for i in range(min(-(-max(c, 0) // PAGE), width)):
            table[b][i] = order.pop()
    rest = order if free is None else order[:free]
    pages = ncb.PageTable(n_pages, len(cached), width * PAGE, table=words(table), lens=words(cached),
                          free=words(rest + [0] * (n_pages - len(rest))), free_count=words([len(rest)]))
    return pages, table, rest


def check_plan(cached, new, rows, max_new, n_pages, width, free=None, in_place=False, Hq=8, Hkv=2, windows=(0,)):
    pages, table, rest = make_table(cached, n_pages, width, free)
    want, bits = plain.plan(table, cached, new, rest, rows, max_new)
    status = words([0])
    plan = ncb.page_plan(pages, pages.lens if in_place else words(cached), words(new), rows, max_new=max_new, Hq=Hq, Hkv=Hkv, windows=windows,
                         lens=pages.lens if in_place else None, status=status)
    assert status.item() == bits
    for name in ("row_start", "fresh", "lens", "pos", "place", "request"):
        assert getattr(plan, name).tolist() == want[name], name
    assert pages.table.tolist() == want["table"] and pages.free_count.item() == want["left"] and pages.ticket.item() == 0
    if in_place:
        assert pages.lens.tolist() == want["lens"]
    check_schedule(plan, want, cached, new, rows, Hq // Hkv, Hkv, max_new)
    return pages, plan


def check_schedule(plan, want, cached, new, rows, group, Hkv, max_new):
    """Every row in reach in one owner; owners see their pages; pieces cover every page once; no two pieces have the same part."""
    each = len(plan.work) // len(plan.windows)
    for w, window in enumerate(plan.windows):
        cover = []
        for per, blocks, overhead, least, (total, share, whole), owners, starts, joins, listed in plain.schedule(
                plan.work[w * each:(w + 1) * each].tolist(), plan.pages.requests, rows, max_new, group, plan.blocks):
            before = 0
            for b, row, count, pos, page0, pages, at, _ in owners.tolist():
                row0 = row - want["row_start"][b]
                assert 0 < count <= per and row0 % per == 0
                if group <= 16 and max_new > 16 // group:  # both classes
                    assert (want["row_start"][b + 1] - want["row_start"][b] > 16 // group) == (overhead == 4) or want["row_start"][b + 1] > rows
                cover += range(row, row + count)
                if want["fresh"][b]:
                    first, last = cached[b] + row0, cached[b] + row0 + count - 1
                    assert pos == first and page0 == (max(0, first + 1 - window) // PAGE if window else 0) and page0 + pages == last // PAGE + 1
                else:
                    assert pages == 0
                assert at == before
                before += max(pages, 1) + overhead
            assert total == before and share == max(-(-total * Hkv // blocks), least)
            tile = overhead == 4
            slack = 6 if not tile else 8 if max_new <= per // 2 else 20
            fit = len(owners) == 0 or (tile or len(owners) * Hkv <= blocks) and plain.last_whole(owners[:, 5].clip(1) + overhead, Hkv, blocks) <= share + slack
            assert whole == (fit or (len(owners) * Hkv >= 8 * blocks if tile else plan.pages.width <= 16))
            if whole or len(owners) == 0:
                assert not joins[:, 1].any()
            if whole or len(owners) == 0 or len(owners) * Hkv > 100000:
                continue
            done, joined = plain.pieces(owners, Hkv, blocks, overhead, total, share)
            parts = sorted(p[5] for p in done if p[5] >= 0)
            assert parts == sorted(set(parts)) == sorted(x for j in joined.values() for x in j)
            want_joins = {j[0] // 2: [owners[i, 1], owners[i, 2] * group, head, j[0] // 2, j[-1] // 2] for (head, i), j in joined.items()}
            assert {b: j[:5] for b, j in enumerate(joins.tolist()) if j[1]} == want_joins
            assert sum(p[4] - p[3] for p in done) == Hkv * int(owners[:, 5].sum())
            ends = owners[:, 6] + np.maximum(owners[:, 5], 1) + overhead
            for blk, (o, head, local, _) in enumerate(starts.tolist()):
                if blk * share < total * Hkv:
                    assert head * total + owners[o, 6] + local == blk * share and 0 <= local and owners[o, 6] + local < ends[o]
            if tile:
                done.sort(key=lambda p: (p[0], p[1], p[2], p[3]))
                want_pieces = [[*owners[i, :4].tolist(), int(owners[i, 4]) + a, z - a, head, part] for _, head, i, a, z, part in done]
                assert listed[:len(done)].tolist() == want_pieces
                count = np.bincount([p[0] for p in done], minlength=blocks)
                assert starts[:, 3].tolist() == [0, *np.cumsum(count).tolist()]
        assert sorted(cover) == [r for r in range(rows) if want["request"][r] >= 0]


@pytest.mark.parametrize("cached, new, rows", [
    ([0], [1], 1), ([63], [1], 1), ([64], [1], 1), ([127], [130], 140), ([5, 0, 64, 63], [0, 0, 0, 0], 3), ([5, 0, 64, 63], [1, 0, 1, 2], 4),
    ([300, 0, 64, 63, 1], [1, 200, 1, 2, 65], 300)])
def test_plan_small(cached, new, rows):
    check_plan(cached, new, rows, 256, 64, 9, windows=(0, 100))


@pytest.mark.parametrize("n, seed", [(33, 0), (1000, 1), (1025, 2), (8192, 3)])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_many(n, seed, in_place):
    rng = np.random.default_rng(seed)
    cached, new = rng.integers(0, 400, n).tolist(), np.where(rng.random(n) < 0.1, rng.integers(0, 90, n), rng.integers(0, 2, n)).tolist()
    need = sum(-(-(c + k) // PAGE) for c, k in zip(cached, new))
    check_plan(cached, new, sum(new) + 17, 90, need + 3, 8, in_place=in_place, windows=(0, 64, 200))


def test_plan_long_requests_are_cut():
    check_plan([131071 - 64 * 3, 9000, 20], [1, 1, 64], 70, 64, 2300, 2048, Hq=32, Hkv=8, windows=(0, 5000))


def test_plan_many_rows_of_one_request():
    check_plan([100], [20000], 20000, 20000, 400, 330, Hq=12, Hkv=1)
    check_plan([0], [70000], 70001, 70000, 1200, 1100, Hq=4, Hkv=4, windows=(0, 333))


@pytest.mark.parametrize("free", [0, 1, 2, 3, 7])
def test_plan_when_pages_run_out(free):
    """In order; a request that needs none is served all the same."""
    check_plan([64, 10, 64, 64, 10, 0], [1, 1, 129, 1, 3, 1], 136, 200, 30, 8, free=free)


def test_plan_refuses_requests():
    check_plan([10, -1, 10, 500, 10, 10], [1, 1, -3, 20, 31, 4], 70, 30, 30, 8)   # negative, over the table, over max_new
    check_plan([10, 10, 10], [3, 5, 1], 7, 30, 30, 8)                            # rows that the step does not have
    check_plan([10, 10], [2 ** 31 - 1, 1], 7, 30, 30, 8)
    check_plan([2 ** 31 - 1, 10], [1, 1], 7, 30, 30, 8)


def test_plan_flags_pages_outside_the_pool():
    pages, table, rest = make_table([10, 64], 8, 4)
    pages.table[0, 0] = 8
    pages.free[pages.free_count.item() - 1] = -5
    status = words([0])
    plan = ncb.page_plan(pages, pages.lens, words([1, 1]), 2, max_new=1, Hq=4, Hkv=4, status=status)
    assert status.item() == 16 and plan.place.tolist() == [-1, -1] and pages.table[1, 1].item() == -1


def test_release_and_reuse():
    pages = ncb.PageTable(20, 5, 4 * PAGE)
    status = words([0])
    new = words([100, 64, 0, 200, 1])
    ncb.page_plan(pages, pages.lens, new, 365, max_new=200, Hq=4, Hkv=4, lens=pages.lens, status=status)
    assert pages.lens.tolist() == [100, 64, 0, 200, 1] and pages.free_count.item() == 20 - 8
    assert pages.table.tolist() == [[0, 1, -1, -1], [2, -1, -1, -1], [-1] * 4, [3, 4, 5, 6], [7, -1, -1, -1]]
    pages.release(words([1, 0, 1, 1, 0]), status=status)
    assert pages.lens.tolist() == [0, 64, 0, 0, 1] and pages.free_count.item() == 18
    assert pages.table.tolist() == [[-1] * 4, [2, -1, -1, -1], [-1] * 4, [-1] * 4, [7, -1, -1, -1]]
    pages.release(words([1, 0, 0, 1, 0]), status=status)  # twice: nothing is held any more
    assert pages.free_count.item() == 18 and sorted(pages.free[:18].tolist()) == [p for p in range(20) if p not in (2, 7)]
    ncb.page_plan(pages, pages.lens, words([0, 0, 250, 0, 0]), 250, max_new=250, Hq=4, Hkv=4, lens=pages.lens, status=status)
    assert pages.table[2].tolist() == [3, 4, 5, 6] and status.item() == 0  # the last ones given back, in their order


def test_release_of_many():
    n = 1500
    rng = np.random.default_rng(5)
    lens = rng.integers(0, 64 * 40, n).tolist()
    held = [-(-x // PAGE) for x in lens]
    pages, table, rest = make_table(lens, sum(held) + 9, 40)
    which = (rng.random(n) < 0.5).astype(int).tolist()
    pages.release(words(which))
    back = [p for b in range(n) if which[b] for p in table[b][:held[b]]]
    assert pages.free_count.item() == len(rest) + len(back)
    assert sorted(pages.free[len(rest):len(rest) + len(back)].tolist()) == sorted(back)
    assert pages.lens.tolist() == [0 if w else x for w, x in zip(which, lens)]
    assert pages.table.tolist() == [[-1] * 40 if which[b] else table[b] for b in range(n)]


# ---- append -------------------------------------------------------------------------------------------------------------------


@pytest.mark.parametrize("heads", [(4, 4), (8, 2), (10, 10), (12, 1)])
@pytest.mark.parametrize("new, cached", [([1, 0, 1], [0, 7, 63]), ([16, 1, 50], [16, 64, 0]), ([130, 17, 3], [1, 60, 15]), ([300, 256, 1], [0, 64, 127])])
def test_append_has_the_slot_caches_bits(heads, new, cached):
    Hq, Hkv = heads
    gen = torch.Generator().manual_seed(hash((heads, tuple(new))) % 1000)
    rows = sum(new)
    pages, *_ = make_table(cached, 40, 8)
    status = words([0])
    plan = ncb.page_plan(pages, pages.lens, words(new), rows + 5, max_new=300, Hq=Hq, Hkv=Hkv, status=status)
    wide = torch.randn(rows + 5, (Hq + 2 * Hkv + 1) * 128, generator=gen).bfloat16().cuda()
    qkv = wide[:, 128:]  # a row stride of its own
    gains = [(1 + 0.1 * torch.randn(128, generator=gen)).cuda() for _ in "qk"]
    cos, sin = ncb.rotary_table(600, 1e4, "cuda")
    cache = ncb.PagedKVCache(40, Hkv)
    marked = torch.full((rows + 5, Hq, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    q = ncb.paged_append(qkv, *gains, cos, sin, plan.pos, plan.place, cache, Hq, q_out=marked, status=status)
    slots = ncb.Fp8KVCache(len(new), Hkv, 8 * PAGE)
    slot_map = plan.request.clamp(min=0)
    want = ncb.kv_append(qkv, *gains, cos, sin, plan.pos, slots, Hq, slot_map=slot_map, status=status)
    assert status.item() == 0
    assert torch.equal(q[:rows], want[:rows]) and (q[rows:] == 7).all()  # rows behind the last request
    mapped = torch.zeros(40, dtype=torch.bool)
    for b in range(len(new)):
        for i in range(-(-(cached[b] + new[b]) // PAGE)):
            page = pages.table[b, i].item()
            mapped[page] = True
            assert torch.equal(cache.pages[page], slots.pages[b, :, i])
    assert not cache.pages[~mapped.cuda()].any()
    # bf16 pages: keys have the bits that q gets from the same row and gain, values are the rows
    as_q = torch.cat([qkv[:, Hq * 128:(Hq + Hkv) * 128], qkv[:, Hq * 128:]], 1).contiguous()
    k = ncb.kv_append(as_q, gains[1], gains[1], cos, sin, plan.pos, ncb.Fp8KVCache(len(new), Hkv, 8 * PAGE), Hkv, slot_map=slot_map)
    wide_cache = ncb.PagedKVCache(40, Hkv, torch.bfloat16)
    q = ncb.paged_append(qkv, *gains, cos, sin, plan.pos, plan.place, wide_cache, Hq)
    assert torch.equal(q[:rows], want[:rows])
    page, j = plan.place[:rows].long() // PAGE, plan.place[:rows].long() % PAGE
    assert torch.equal(wide_cache.pages[page, :, 0, j], k[:rows])
    assert torch.equal(wide_cache.pages[page, :, 1, j], qkv[:rows, (Hq + Hkv) * 128:].reshape(rows, Hkv, 128))
    assert wide_cache.pages.count_nonzero() <= 2 * rows * Hkv * 128


def test_append_skips_what_is_outside():
    qkv = torch.randn(6, 3 * 128, device="cuda").bfloat16()
    one = torch.ones(128, device="cuda")
    cos, sin = ncb.rotary_table(64, 1e4, "cuda")
    for dtype in (torch.float8_e4m3fn, torch.bfloat16):
        cache, status = ncb.PagedKVCache(2, 1, dtype), words([0])
        q = torch.full((6, 1, 128), 7.0, dtype=torch.bfloat16, device="cuda")
        ncb.paged_append(qkv, one, one, cos, sin, words([-1, 3, 64, 5, 6, 7]), words([4, -1, 4, 128, 2 ** 31 - 1, 127]), cache, 1, q_out=q, status=status)
        assert status.item() == 1 and (q[:5] == 7).all() and not (q[5] == 7).any()
        assert cache.pages[1].any() and not cache.pages[0].any()


# ---- attention ------------------------------------------------------------------------------------------------------------------


class Pool:
    """A pool whose every byte that no request wrote is NaN (codes and scales too), with requests of lens positions, of which a plan
    (`plan`, with spare rows behind the last) has just added the last new."""

    def __init__(self, dtype, Hq, Hkv, lens, new, window=0, seed=0, tail=3, free=None, width=1, bound=1):
        gen = torch.Generator().manual_seed(seed)
        held = [-(-n // PAGE) for n in lens]
        self.n_pages, self.rows = sum(held) + 3, sum(new)
        cached, status = [n - k for n, k in zip(lens, new)], words([0])
        self.pages, *_ = make_table(cached, self.n_pages, max(held + [1, width - 1]) + 1, free=free, seed=seed)
        self.plan = ncb.page_plan(self.pages, words(cached), words(new), self.rows + tail, max_new=max(new + [bound]), Hq=Hq, Hkv=Hkv, windows=(window,),
                                  status=status)
        self.status = status.item()
        self.table = table = self.pages.table.tolist()
        served = self.plan.fresh.tolist()
        self.lens = lens = [c + k for c, k in zip(cached, served)]
        self.q = torch.randn(self.rows + tail, Hq, 128, generator=torch.Generator().manual_seed(seed + 1)).bfloat16().cuda()
        if dtype == torch.bfloat16:
            full = torch.full((self.n_pages, Hkv, 2, PAGE, 128), float("nan"), dtype=dtype, device="cuda")
        else:
            full = torch.full((self.n_pages, Hkv, 16896), 255, dtype=torch.uint8, device="cuda")
        self.cache = ncb.PagedKVCache(self.n_pages, Hkv, dtype, pages=full)
        self.k, self.v = [], []
        for b, n in enumerate(lens):
            k, v = (torch.randn(Hkv, n, 128, generator=gen).bfloat16() for _ in range(2))
            row = words(table[b])
            if n:
                self.store(row, k, v, 0)
            got = self.cache.read(row, n) if n else (torch.zeros(Hkv, 0, 128, device="cuda"),) * 2
            self.k.append(got[0].double())
            self.v.append(got[1].double())

    def store(self, row, k, v, start):
        if not self.cache.e4m3:
            self.cache.write(row, k, v, start=start)
            return
        args = []
        for x in (k, v):
            scale = x.float().abs().amax(-1) / 448
            args.append(((x.float() / scale[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), scale))
        self.cache.write(row, args[0][0], args[1][0], args[0][1], args[1][1], start=start)


def run_attention(dtype, Hq, Hkv, lens, new, window=0, seed=0, tail=3, scale_q=1.0, width=1, bound=1):
    """The last new[b] of request b's lens[b] positions attend. Checks every row against 64 bits; returns the pieces."""
    pool = Pool(dtype, Hq, Hkv, lens, new, window, seed, tail, width=width, bound=bound)
    rows, plan, status = pool.rows, pool.plan, words([0])
    q = (pool.q.float() * scale_q).bfloat16()
    out = torch.full((rows + tail, Hq, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    got = ncb.paged_attention(q, pool.cache, plan, window=window, out=out, status=status)
    assert got is out and status.item() == 0
    assert (out[rows:] == 7).all()
    check_rows(pool, q, out, lens, new, window)
    return pool, plan, q, out


def check_rows(pool, q, out, lens, new, window):
    rounding = 2.0 ** -11 if pool.cache.e4m3 else 2.0 ** -8
    at = 0
    for b, (n, k) in enumerate(zip(lens, new)):
        if k:
            want, size = plain.attention(q[at:at + k].double(), pool.k[b], pool.v[b], n - k, window)
            off = (out[at:at + k].double() - want).abs() - 2.0 ** -8 * want.abs() - (rounding + 2.0 ** -14) * size
            assert not off.isnan().any() and off.max().item() <= 0, (b, n, k, off.max().item())
        at += k


DTYPES = [torch.float8_e4m3fn, torch.bfloat16]


@pytest.mark.parametrize("width", [1, 40])  # tables of few pages: no owner is cut
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [(1, 1), (4, 1), (8, 2), (9, 3), (5, 5), (12, 1), (16, 2), (32, 1), (40, 1), (64, 1)])
@pytest.mark.parametrize("lens, new", [([1], [1]), ([64, 1, 65, 63], [1, 1, 1, 1]), ([200, 130, 64, 700], [1, 0, 3, 17]), ([513, 40], [70, 40])])
def test_attention_shapes(dtype, heads, lens, new, width):
    run_attention(dtype, *heads, lens, new, seed=len(lens), width=width)


@pytest.mark.parametrize("width", [1, 40])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 100, 1000])
@pytest.mark.parametrize("lens, new", [([300, 64, 129], [1, 1, 1]), ([300, 500, 20], [5, 130, 20])])
def test_attention_windows(dtype, window, lens, new, width):
    run_attention(dtype, 8, 2, lens, new, window=window, seed=7, width=width)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens, new", [([20000], [1]), ([9000, 100, 3000], [1, 1, 1]), ([6000, 1], [100, 1]), ([5000, 4000], [33, 5])])
def test_attention_long_contexts_are_split(dtype, lens, new):
    run_attention(dtype, 8, 2, lens, new, seed=9)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window", [0, 64, 700])
@pytest.mark.parametrize("heads, lens, new", [
    ((8, 2), [9000, 64, 700, 20, 65, 129], [20, 20, 7, 18, 17, 1]),   # 16 < slots <= 128: both tiles have them
    ((8, 2), [3000, 40, 1500], [32, 32, 31]), ((16, 1), [900, 128, 5000, 66], [8, 3, 5, 2]), ((2, 2), [4000, 127, 128, 129], [128, 127, 60, 65])])
def test_attention_of_few_rows(dtype, window, heads, lens, new):
    pool, plan, q, out = run_attention(dtype, *heads, lens, new, window=window, seed=15)
    for _ in range(3):
        assert torch.equal(ncb.paged_attention(q, pool.cache, plan, window=window)[:sum(new)], out[:sum(new)])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bound", [32, 33, 1000, 2 ** 30, 2 ** 31 - 1])
def test_attention_under_bounds_that_nobody_reaches(dtype, bound):
    run_attention(dtype, 8, 2, [300, 64, 1000, 129], [1, 0, 30, 5], seed=17, bound=bound)
    run_attention(dtype, 8, 2, [300, 64], [1, 1], seed=17, bound=bound)
    if bound >= 1000:
        run_attention(dtype, 8, 2, [300, 900], [1, 700], seed=17, bound=bound)


@pytest.mark.parametrize("width", [1, 40])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_of_many_small_requests(dtype, width):
    rng = np.random.default_rng(3)
    lens = rng.integers(1, 150, 600).tolist()
    new = [min(n, int(k)) for n, k in zip(lens, rng.integers(0, 4, 600))]
    run_attention(dtype, 4, 2, lens, new, seed=11, width=width)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale_q", [1e-20, 30.0, 1e4])
def test_attention_of_extreme_queries(dtype, scale_q):
    """Flat and one-hot softmaxes. Score errors grow with the scores: at 30 a score of 1,000 is off by 2^-24 128 1000 / 11, under 2^-14
    of A times e^x; at 1e4 only the finite-ness is looked at."""
    if scale_q < 1:
        run_attention(dtype, 8, 2, [300, 70], [1, 10], seed=5, scale_q=scale_q)
        return
    pool = Pool(dtype, 8, 2, [300, 70], [1, 10], seed=5, tail=0)
    q = (pool.q.float() * scale_q).bfloat16()
    out = ncb.paged_attention(q, pool.cache, pool.plan)
    assert out.isfinite().all()
    if scale_q == 30.0:
        at = 0
        for b, (n, k) in enumerate(((300, 1), (70, 10))):
            want, size = plain.attention(q[at:at + k].double(), pool.k[b], pool.v[b], n - k, 0)
            assert ((out[at:at + k].double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -7 * size).all()
            at += k


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [(8, 2), (2, 2)])
@pytest.mark.parametrize("new", [4, 20, 150])
def test_what_a_row_does_not_see_does_not_reach_it(dtype, heads, new):
    """A later row's key and value are infinite and NaN: the rows before it keep their results bit for bit. So do rows whose window
    has left such a position behind."""
    Hq, Hkv = heads
    n = 200 + new
    for window, at, clean in ((0, n - 2, slice(0, new - 2)), (50, n - new - 49, slice(1, new)), (0, n - 1, slice(0, new - 1))):
        pool, plan, q, out = run_attention(dtype, Hq, Hkv, [n], [new], window=window, seed=13)
        k = torch.full((Hkv, 1, 128), float("inf"), dtype=torch.bfloat16)
        v = torch.full((Hkv, 1, 128), float("nan"), dtype=torch.bfloat16)
        v[..., ::2] = float("inf")
        if pool.cache.e4m3:
            nan = torch.full((Hkv, 1, 128), 0x7f, dtype=torch.uint8)
            inf = torch.full((Hkv, 1), float("inf"))
            pool.cache.write(words(pool.table[0]), nan, nan, inf, inf, start=at)
        else:
            pool.cache.write(words(pool.table[0]), k, v, start=at)
        again = ncb.paged_attention(q, pool.cache, plan, window=window)
        assert torch.allclose(again[clean].float(), out[clean].float(), rtol=2 ** -6, atol=2 ** -6) and again[clean].isfinite().all()
        seen = again[new - 1] if window == 0 else again[0]
        assert seen.isnan().any() or seen.isinf().any()


@pytest.mark.parametrize("dtype", DTYPES)
def test_nan_queries_stay_nan(dtype):
    pool, plan, q, out = run_attention(dtype, 8, 2, [2000, 70], [1, 10], seed=5)
    q = q.clone()
    q[0, 3], q[4, 1] = float("nan"), float("nan")
    again = ncb.paged_attention(q, pool.cache, plan)
    bad = torch.zeros(11, 8, dtype=torch.bool)
    bad[0, 3] = bad[4, 1] = True
    assert again[:11][bad.cuda()].isnan().all() and torch.equal(again[:11][~bad.cuda()], out[:11][~bad.cuda()])


@pytest.mark.parametrize("dtype", DTYPES)
def test_attention_of_strided_rows(dtype):
    pool, plan, q, out = run_attention(dtype, 8, 2, [300, 70], [1, 10], seed=5)
    wide = torch.zeros(len(q), 12, 128, dtype=torch.bfloat16, device="cuda")
    wide[:, 2:10] = q
    into = torch.full((len(q), 10, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    ncb.paged_attention(wide[:, 2:10], pool.cache, plan, out=into[:, 1:9])
    assert torch.equal(into[:11, 1:9], out[:11]) and (into[:, 0] == 7).all() and (into[:, 9] == 7).all() and (into[11:] == 7).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_that_were_not_served_are_zero(dtype):
    pool = Pool(dtype, 8, 2, [100, 144, 90], [5, 80, 1], seed=3, tail=4, free=1)
    plan, q = pool.plan, pool.q
    assert pool.status == 8 and plan.fresh.tolist() == [5, 0, 1]
    out = torch.full((90, 8, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    ncb.paged_attention(q, pool.cache, plan, out=out)
    assert (out[5:85] == 0).all() and (out[86:] == 7).all()
    check_rows(pool, torch.cat([q[:5], q[85:86]]), torch.cat([out[:5], out[85:86]]), [100, 64, 90], [5, 0, 1], 0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_pages_outside_the_pool_are_flagged_and_left_out(dtype):
    pool = Pool(dtype, 8, 2, [200, 100], [1, 1], seed=3, tail=0)
    plan, q = pool.plan, pool.q
    want = ncb.paged_attention(q, pool.cache, plan)
    for bad in (-1, pool.n_pages, 2 ** 31 - 1, -2 ** 31):
        pool.pages.table[0, 1] = bad
        status = words([0])
        out = ncb.paged_attention(q, pool.cache, plan, status=status)
        assert status.item() == 16 and torch.equal(out[1], want[1]) and out[0].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bound", [1, 20, 100])
def test_requests_past_the_bound_get_zeros(dtype, bound):
    gen = torch.Generator().manual_seed(33)
    wide, Hq, Hkv = torch.randn(301, 12 * 128, generator=gen).bfloat16().cuda(), 8, 2
    gain, (cos, sin) = torch.ones(128, device="cuda"), ncb.rotary_table(512, 1e4, "cuda")
    found = []
    for new, take in (([bound, 200, 1], slice(0, bound + 201)), ([bound, 0, 1], [*range(bound), bound + 200])):
        pages, status = ncb.PageTable(20, 3, 512), words([0])
        cache, qkv = ncb.PagedKVCache(20, Hkv, dtype), wide[take].contiguous()
        plan = ncb.page_plan(pages, pages.lens, words(new), len(qkv), max_new=bound, Hq=Hq, Hkv=Hkv, lens=pages.lens, status=status)
        q = ncb.paged_append(qkv, gain, gain, cos, sin, plan.pos, plan.place, cache, Hq)
        found.append(ncb.paged_attention(q, cache, plan, out=torch.full_like(q, 7.0)))
        assert status.item() == (4 if new[1] else 0) and plan.fresh.tolist() == [bound, 0, 1]
    assert not found[0][bound:bound + 200].any()
    got = torch.cat([found[0][:bound], found[0][bound + 200:]]).float()
    assert torch.allclose(got, found[1].float(), rtol=2 ** -7, atol=2 ** -10)


@pytest.mark.parametrize("dtype, many", [(torch.float8_e4m3fn, 300_000), (torch.bfloat16, 150_000)])
def test_pages_behind_4_gib(dtype, many):
    """The same step in the last pages of a pool of 5 GB and in a small one: the same bits."""
    gen = torch.Generator().manual_seed(31)
    new, rows, Hq, Hkv = words([1, 300, 20]), 321, 4, 1
    qkv = torch.randn(rows, (Hq + 2 * Hkv) * 128, generator=gen).bfloat16().cuda()
    gain = torch.ones(128, device="cuda")
    cos, sin = ncb.rotary_table(512, 1e4, "cuda")
    found = []
    for n_pages in (12, many):
        pages = ncb.PageTable(n_pages, 3, 512)
        pages.free.copy_(torch.arange(n_pages, dtype=torch.int32))  # the last ones first
        cache = ncb.PagedKVCache(n_pages, Hkv, dtype)
        plan = ncb.page_plan(pages, pages.lens, new, rows, max_new=300, Hq=Hq, Hkv=Hkv, lens=pages.lens)
        q = ncb.paged_append(qkv, gain, gain, cos, sin, plan.pos, plan.place, cache, Hq)
        found.append(ncb.paged_attention(q, cache, plan))
        assert pages.table[0, 0].item() == n_pages - 1
        del cache
    assert torch.equal(*found) and found[0].isfinite().all()


def test_operands_of_another_device_are_refused():
    pages = ncb.PageTable(4, 2, 2 * PAGE)
    new, other = words([1, 1]), torch.tensor([1, 1], dtype=torch.int32)
    with pytest.raises(AssertionError):
        ncb.page_plan(pages, pages.lens, other, 2, max_new=1, Hq=4, Hkv=2)
    with pytest.raises(AssertionError):
        pages.release(other)
    plan = ncb.page_plan(pages, pages.lens, new, 2, max_new=1, Hq=4, Hkv=2)
    cos, sin = ncb.rotary_table(2 * PAGE, 1e4, "cuda")
    cache, gain = ncb.PagedKVCache(4, 2), torch.ones(128, device="cuda")
    operands = [torch.zeros(2, 8 * 128, dtype=torch.bfloat16, device="cuda"), gain, gain, cos, sin, plan.pos, plan.place]
    for i in range(len(operands)):
        with pytest.raises(AssertionError):
            ncb.paged_append(*operands[:i], operands[i].cpu(), *operands[i + 1:], cache, 4)
    q = ncb.paged_append(*operands, cache, 4)
    for bad in (dict(q=q.cpu()), dict(out=q.cpu()), dict(workspace=torch.empty(64, dtype=torch.uint8)),
                dict(cache=ncb.PagedKVCache(4, 2, device="cpu"))):
        with pytest.raises(AssertionError):
            ncb.paged_attention(**(dict(q=q, cache=cache, plan=plan) | bad))



def test_calls_on_two_streams():
    """Two plans and their calls at once: each has its own workspace."""
    pool, plan, q, out = run_attention(torch.bfloat16, 8, 2, [20000, 70], [1, 10], seed=5)
    other, plan2, q2, out2 = run_attention(torch.float8_e4m3fn, 8, 2, [9000, 300], [2, 30], seed=6)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    found = []
    for _ in range(10):
        for s, args in zip(streams, ((q, pool.cache, plan), (q2, other.cache, plan2))):
            with torch.cuda.stream(s):
                found.append(ncb.paged_attention(*args))
    torch.cuda.synchronize()
    for i, x in enumerate(found):
        assert torch.equal(x[:11], out[:11]) if i % 2 == 0 else torch.equal(x[:32], out2[:32])


# ---- steps ------------------------------------------------------------------------------------------------------------------------


def step_inputs(gen, rows, Hq, Hkv):
    return torch.randn(rows, (Hq + 2 * Hkv) * 128, generator=gen).bfloat16().cuda()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Hq, Hkv", [(8, 2), (5, 5)])
def test_a_server_s_steps(dtype, Hq, Hkv):
    """Requests come in chunks, decode, finish, and others take their pages: plan, append and attention step by step, against keys and values
    kept apart in 64 bits."""
    gen = torch.Generator().manual_seed(17)
    pages, status = ncb.PageTable(14, 4, 6 * PAGE), words([0])
    cache = ncb.PagedKVCache(14, Hkv, dtype)
    cos, sin = ncb.rotary_table(6 * PAGE, 1e4, "cuda")
    gains = [(1 + 0.1 * torch.randn(128, generator=gen)).cuda() for _ in "qk"]
    lens = [0, 0, 0, 0]
    plan = None
    for new, done in (([100, 3, 0, 0], []), ([120, 1, 64, 0], []), ([1, 1, 1, 200], [1]), ([1, 33, 1, 1], [0]), ([90, 1, 1, 1], []), ([1, 1, 1, 1], [2, 3]),
                      ([200, 1, 5, 0], [])):
        qkv = step_inputs(gen, 330, Hq, Hkv)
        plan = ncb.page_plan(pages, pages.lens, words(new), 330, max_new=200, Hq=Hq, Hkv=Hkv, windows=(0, 70), lens=pages.lens, plan=plan, status=status)
        q = ncb.paged_append(qkv, *gains, cos, sin, plan.pos, plan.place, cache, Hq, status=status)
        for window in (0, 70):
            out = ncb.paged_attention(q, cache, plan, window=window, status=status)
            pool = type("Seen", (), {"cache": cache})
            both = [cache.read(pages.table[b], lens[b] + new[b]) if lens[b] + new[b] else (torch.zeros(Hkv, 0, 128, device="cuda"),) * 2 for b in range(4)]
            pool.k, pool.v = [x[0].double() for x in both], [x[1].double() for x in both]
            check_rows(pool, q, out, [a + b for a, b in zip(lens, new)], new, window)
        lens = [a + b for a, b in zip(lens, new)]
        assert pages.lens.tolist() == lens and status.item() == 0
        pages.release(words([int(b in done) for b in range(4)]), status=status)
        lens = [0 if b in done else x for b, x in enumerate(lens)]
    assert pages.free_count.item() == 14 - sum(-(-x // PAGE) for x in lens)


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_captured_step_serves_lengths_that_change(dtype):
    """One graph, replayed as the requests grow, against eager steps on a second table and pool."""
    Hq, Hkv, gen = 8, 2, torch.Generator().manual_seed(23)
    cos, sin = ncb.rotary_table(10 * PAGE, 1e4, "cuda")
    gains = [(1 + 0.1 * torch.randn(128, generator=gen)).cuda() for _ in "qk"]

    class Side:
        def __init__(self):
            self.pages, self.cache, self.status = ncb.PageTable(40, 5, 10 * PAGE), ncb.PagedKVCache(40, Hkv, dtype), words([0])
            self.new, self.qkv, self.plan = words([0] * 5), torch.zeros(64, (Hq + 2 * Hkv) * 128, dtype=torch.bfloat16, device="cuda"), None
            self.out = torch.zeros(64, Hq, 128, dtype=torch.bfloat16, device="cuda")

        def step(self):
            self.plan = ncb.page_plan(self.pages, self.pages.lens, self.new, 64, max_new=40, Hq=Hq, Hkv=Hkv, lens=self.pages.lens, plan=self.plan, status=self.status)
            q = ncb.paged_append(self.qkv, *gains, cos, sin, self.plan.pos, self.plan.place, self.cache, Hq, status=self.status)
            ncb.paged_attention(q, self.cache, self.plan, out=self.out, status=self.status)

    eager, captured = Side(), Side()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        captured.step()  # first-use set-up, all requests idle
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            captured.step()
    torch.cuda.current_stream().wait_stream(side)
    for i in range(60):
        new = [40, 1, 0, 1, 22] if i % 7 == 0 else [1, 1, i % 2, 3, 0] if i % 7 else [0] * 5
        if i >= 40:
            new = [1, 1, 1, 0, 1]
        x = step_inputs(gen, 64, Hq, Hkv)
        for s in (eager, captured):
            s.new.copy_(words(new))
            s.qkv.copy_(x)
        eager.step()
        graph.replay()
        rows = sum(new)
        assert torch.equal(eager.out[:rows], captured.out[:rows])
    assert eager.status.item() == captured.status.item() == 0
    assert torch.equal(eager.pages.table, captured.pages.table) and torch.equal(eager.pages.lens, captured.pages.lens)
