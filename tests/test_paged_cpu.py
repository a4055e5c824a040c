"""The paged operators without a GPU: refusals of the C entry points and of their Python faces, sizes of schedules, the pools' layout."""

import ctypes

import pytest
import torch

import nanochat_b200 as ncb
from nanochat_b200 import native, paged
from oracle import kv_append as okv

P, NUL = 4096, None  # a non-NULL, aligned stand-in: validation fails before any use


def plan_args(**changes):
    names = [f for f, _ in native.Plan._fields_ if f not in ("windows",)]
    args = native.Plan(**{n: P for n in names if dict(native.Plan._fields_)[n] is native.c_ptr})
    for n, x in dict(rows=64, requests=4, width=8, n_pages=32, max_fresh=16, group=4, kv_heads=2, blocks=296, n_windows=1).items():
        setattr(args, n, x)
    for n, x in changes.items():
        if n == "window":
            args.windows[0] = x
        else:
            setattr(args, n, x)
    return ctypes.byref(args)


@pytest.mark.parametrize("changes, status", [
    (dict(requests=0), 1), (dict(requests=8193), 1), (dict(rows=-1), 1), (dict(rows=1 << 27), 1), (dict(width=0), 1), (dict(n_pages=0), 1),
    (dict(n_pages=1 << 26), 1), (dict(max_fresh=0), 1), (dict(group=0), 1), (dict(group=65), 1), (dict(kv_heads=0), 1), (dict(blocks=0), 1),
    (dict(n_windows=-1), 1), (dict(n_windows=9), 1), (dict(window=-1), 1), (dict(work=P + 4), 2),
    *[(dict([(n, NUL)]), 1) for n in ("table", "cached", "fresh", "free_pages", "free_count", "free_left", "row_start", "served", "lens", "pos", "place", "request", "work", "ticket")]])
def test_page_plan_refuses(changes, status):
    assert native.cuda_library("page_plan").page_plan(plan_args(**changes), NUL) == status


def test_page_release_refuses():
    lib = native.cuda_library("page_plan")
    assert lib.page_release(P, P, P, P, P, 0, 8, 32, NUL, NUL) == 1
    assert lib.page_release(P, P, P, P, P, 8193, 8, 32, NUL, NUL) == 1
    assert lib.page_release(P, NUL, P, P, P, 4, 8, 32, NUL, NUL) == 1


def test_append_refuses():
    f = native.cuda_library("paged_append").paged_append
    good = [P] * 9 + [4, 8, 2, 12 * 128, 64, 32, 1, NUL, NUL]

    def at(i, x):
        return good[:i] + [x] + good[i + 1:]
    assert f(*at(9, -1)) == 1 and f(*at(9, 0)) == 0
    assert f(*at(11, 3)) == 1          # 8 heads over 3
    assert f(*at(12, 12 * 128 - 8)) == 1
    assert f(*at(12, 12 * 128 + 4)) == 2
    assert f(*at(13, 0)) == 1 and f(*at(14, 0)) == 1 and f(*at(14, 1 << 26)) == 1
    for i in range(9):
        assert f(*at(i, NUL)) == 1
        if i not in (5, 6):  # positions and places are words
            assert f(*at(i, P + 8)) == 2


def attn_args(**changes):
    args = native.Paged(*[P] * 6, None, 64, 8 * 128, 8 * 128, 1 << 40, 4, 8, 32, 16, 8, 2, 1, 0, 296, 0.1)
    for n, x in changes.items():
        setattr(args, n, x)
    return ctypes.byref(args)


@pytest.mark.parametrize("changes, status", [
    (dict(Hq=7), 1), (dict(Hkv=0), 1), (dict(Hq=130, Hkv=2), 1), (dict(requests=0), 1), (dict(rows=-1), 1), (dict(width=0), 1), (dict(n_pages=0), 1),
    (dict(max_fresh=0), 1), (dict(window=-1), 1), (dict(scale=0.0), 1), (dict(scale=-1.0), 1), (dict(scale=float("nan")), 1), (dict(ldq=8 * 128 - 8), 1),
    (dict(ldo=8), 1), (dict(ldq=8 * 128 + 4), 2), (dict(q=P + 8), 2), (dict(out=P + 8), 2), (dict(workspace_bytes=16), 3), (dict(rows=0), 0),
    (dict(n_pages=1 << 24, e4m3=0, Hkv=2), 5),
    *[(dict([(n, NUL)]), 1) for n in ("q", "pool", "out", "workspace", "table", "work")]])
def test_attention_refuses(changes, status):
    assert native.cuda_library("paged_attn").paged_attn(attn_args(**changes), NUL) == status


def test_schedules_have_a_size_for_every_head_group():
    words, size = native.cuda_library("page_plan").page_plan_words, native.cuda_library("paged_attn").paged_attn_workspace_bytes
    for group in (1, 3, 4, 12, 64):
        assert words(64, 64, 1, group, 8, 296) > 64 * 8
        assert size(64, 64, 40, 1, group * 8, 8, 296) > 0
        assert (size(64, 64, 16, 1, group * 8, 8, 296) == 0) == (group <= 16)  # few pages, one row each: no owner is cut
    assert words(64, 64, 1, 65, 8, 296) == -1 and size(64, 64, 40, 1, 9, 8, 296) == -1 and size(64, 64, 0, 1, 8, 8, 296) == -1
    assert words(8192, 1 << 26, 1 << 20, 64, 1, 296) > 0


def test_python_faces_refuse():
    with pytest.raises(ValueError):
        ncb.PagedKVCache(4, 2, torch.float16, device="cpu")
    with pytest.raises(AssertionError):
        ncb.PagedKVCache(4, 2, torch.bfloat16, device="cpu", pages=torch.zeros(4, 2, 2, 64, 64, dtype=torch.bfloat16))
    pages = ncb.PageTable(16, 4, 200, device="cpu")
    assert pages.width == 4 and pages.capacity == 256 and pages.free.tolist() == list(range(15, -1, -1))
    with pytest.raises(AssertionError):
        ncb.PageTable(16, 4, 200, device="cpu", table=torch.zeros(4, 3, dtype=torch.int32))
    with pytest.raises(AssertionError):
        ncb.PagePlan(pages, 8, 8, 8, 3)
    with pytest.raises(AssertionError):
        ncb.PagePlan(pages, 8, 8, 8, 2, windows=())
    with pytest.raises(AssertionError):
        ncb.PagePlan(pages, 8, 8, 8, 2, windows=(0, 0))
    with pytest.raises(ValueError):
        ncb.PagePlan(pages, 8, 8, 130, 2)
    words = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(AssertionError):  # not on a GPU
        ncb.page_plan(pages, words, words, 8, max_new=8, Hq=8, Hkv=2)
    with pytest.raises(AssertionError):
        ncb.page_plan(pages, words.long(), words, 8, max_new=8, Hq=8, Hkv=2)
    plan = ncb.PagePlan(pages, 8, 8, 8, 2, windows=(0, 128))
    cache, q = ncb.PagedKVCache(16, 2, device="cpu"), torch.zeros(8, 8, 128, dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        ncb.paged_attention(q, cache, plan, window=64)
    with pytest.raises(ValueError, match="not filled"):
        ncb.paged_attention(q, cache, plan)
    plan.filled = True
    with pytest.raises(ValueError, match="15 pages"):
        ncb.paged_attention(q, ncb.PagedKVCache(15, 2, device="cpu"), plan)
    with pytest.raises(AssertionError):  # not on a GPU
        ncb.paged_attention(q, cache, plan)
    with pytest.raises(AssertionError):
        ncb.paged_attention(q[:7], cache, plan)
    with pytest.raises(AssertionError):
        ncb.paged_attention(q.float(), cache, plan)


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.bfloat16])
def test_pool_write_read_round_trip(dtype):
    gen = torch.Generator().manual_seed(3)
    cache = ncb.PagedKVCache(9, 3, dtype, device="cpu")
    row = torch.tensor([7, 2, 5, -1], dtype=torch.int32)
    k, v = (torch.randn(3, 140, 128, generator=gen).bfloat16() for _ in range(2))
    if dtype == torch.bfloat16:
        cache.write(row, k, v, start=30)
        want = k.float(), v.float()
        assert torch.equal(cache.pages[7, 1, 1, 33], v[1, 3])
    else:
        (kb, ks), (vb, vs) = (okv.quant_rows(x.view(torch.int16).numpy().view("uint16")) for x in (k, v))
        cache.write(row, *(torch.from_numpy(x) for x in (kb, vb)), *(torch.from_numpy(x) for x in (ks, vs)), start=30)
        want = tuple(torch.from_numpy(okv.e4m3_to_f32(b) * s[..., None]) for b, s in ((kb, ks), (vb, vs)))
    got = cache.read(row, 140, start=30)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert not cache.pages[[0, 1, 3, 4, 6, 8]].any()
    with pytest.raises(AssertionError):
        cache.read(row, 70, start=150)
