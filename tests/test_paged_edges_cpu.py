"""Refusals of the paged operators that need no GPU, beside test_paged_cpu.py."""

import pytest
import torch

import nanochat_b200 as ncb
from nanochat_b200 import native
from tests import paged_cases as plain

P, NUL = 4096, None  # a non-NULL, aligned stand-in: validation fails before any use


def test_page_trim_refuses():
    trim = native.cuda_library("page_plan").page_trim
    assert trim(P, P, P, P, P, 0, 8, 32, NUL, NUL) == 1 and trim(P, P, P, P, P, 8193, 8, 32, NUL, NUL) == 1
    assert trim(P, P, P, P, P, 4, 0, 32, NUL, NUL) == 1 and trim(P, P, P, P, P, 4, 8, 0, NUL, NUL) == 1
    for i in range(5):
        assert trim(*[NUL if j == i else P for j in range(5)], 4, 8, 32, NUL, NUL) == 1
    pages = ncb.PageTable(16, 4, 200, device="cpu")
    for keep in (torch.zeros(4), torch.zeros(3, dtype=torch.int32), torch.zeros(8, dtype=torch.int32)[::2], torch.zeros(4, dtype=torch.int32)):
        with pytest.raises(AssertionError):  # the last: not on a GPU
            pages.trim(keep)


@pytest.mark.parametrize("part", ["table", "lens", "free", "free_count"])
def test_a_table_lives_on_one_device(part):
    """Kernels take its parts' addresses; a part elsewhere would be an address of another memory."""
    shape = {"table": (4, 4), "lens": (4,), "free": (16,), "free_count": (1,)}[part]
    with pytest.raises(AssertionError, match="one device"):
        ncb.PageTable(16, 4, 200, device="cpu", **{part: torch.zeros(shape, dtype=torch.int32, device="meta")})


def test_a_workspace_is_as_large_as_it_says():
    """An expanded tensor has more elements than memory behind it."""
    pages = ncb.PageTable(16, 4, 64 * 64, device="cpu")
    plan = ncb.PagePlan(pages, 8, 8, 8, 2)
    plan.filled = True
    cache, q = ncb.PagedKVCache(16, 2, device="cpu"), torch.zeros(8, 8, 128, dtype=torch.bfloat16)
    assert plan.workspace_bytes > 0
    for workspace in (torch.zeros(1, dtype=torch.uint8).expand(plan.workspace_bytes), torch.zeros(2 * plan.workspace_bytes, dtype=torch.uint8)[::2]):
        with pytest.raises(AssertionError, match="contiguous"):
            ncb.paged_attention(q, cache, plan, workspace=workspace)


@pytest.mark.parametrize("terms", [1, 2])
def test_the_bound_for_few_slots_tells_one_term_from_two(terms):
    """Attention of few query slots over bf16 pages, restated: probabilities that enter the products as two bf16 terms keep the bound that the
    GPU's test has for them, one term does not."""
    gen = torch.Generator().manual_seed(41)
    q, k, v = (torch.randn(*shape, generator=gen).bfloat16().double() for shape in ((2, 8, 128), (2, 200, 128), (2, 200, 128)))
    want, size = plain.attention(q, k, v, 198, 0)
    out = torch.empty_like(want)
    for i in range(2):
        kk, vv = (x[:, :199 + i].repeat_interleave(4, 0) for x in (k, v))
        p = torch.einsum("hd,hkd->hk", q[i], kk) * 128 ** -0.5
        p = torch.exp(p - p.amax(-1, keepdim=True)).float()
        hi = p.bfloat16()
        rounded = hi.double() + ((p - hi.float()).bfloat16().double() if terms == 2 else 0)
        out[i] = (torch.einsum("hk,hkd->hd", rounded, vv) / p.double().sum(-1, keepdim=True)).bfloat16().double()
    off = (out - want).abs() - plain.few_slots_bound(want, size)
    assert (off.max() <= 0) == (terms == 2)


def test_a_pool_says_its_size():
    """As the slot caches do: pages of a length, bytes of the pool."""
    assert [ncb.PagedKVCache.pages_for(n) for n in (0, 1, 64, 65, 8191)] == [ncb.Fp8KVCache.pages_for(n) for n in (0, 1, 64, 65, 8191)] == [0, 1, 1, 2, 128]
    assert ncb.PagedKVCache(5, 3, device="cpu").nbytes() == 5 * 3 * 64 * 264
    assert ncb.PagedKVCache(5, 3, torch.bfloat16, device="cpu").nbytes() == 5 * 3 * 64 * 512
