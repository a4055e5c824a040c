"""A paged KV cache: pages of 64 positions taken from one pool by requests of any length, where Fp8KVCache cuts the memory into
slots of one size (as the reference does, inference/decoder.py:112-121). One step of a server runs

    plan = page_plan(pages, pages.lens, fresh, rows, ..., lens=pages.lens)     once: pages, positions, places, schedules
    for every layer:
        q = paged_append(qkv, ..., plan.pos, plan.place, cache, Hq)
        out = paged_attention(q, cache, plan, window=...)

with any mixture of decoding requests (one fresh token), drafted tokens (a few) and chunks of prompts (hundreds); a finished request's
pages go back with pages.release(), those behind rejected drafts with pages.trim(). Lengths stay on the device, so a captured step serves lengths that change. Like attention.py's
operators, each launches on the current stream and returns without synchronising; a non-zero native status raises
NativeError, what only the device can see is ORed into `status` (NCB_DEV_* bits)."""

import contextlib
import ctypes
import functools

import torch
from torch import Tensor

from .kv_cache import HEAD_DIM, PAGE_TOKENS, PagedKVCache, cache_pages
from .native import PLAN_WINDOWS, Paged, Plan, check, cuda_library, pointer, stream

_READY = contextlib.nullcontext()
_INT, _BF16, _F32 = torch.int32, torch.bfloat16, torch.float32
_SCALE = HEAD_DIM ** -0.5


def on_device_of(*operands: "Tensor | None"):
    """The launches below go to the current stream of the current device: make it the tensors' one."""
    device = operands[0].get_device()  # -1 for what is not on a GPU
    for t in operands:
        assert t is None or t.get_device() == device >= 0, "the operands live on one CUDA device"
    return _READY if device == torch._C._cuda_getDevice() else torch.cuda.device(device)


def _words(t: Tensor, *shape: int) -> bool:
    return t.dtype is _INT and t.shape == shape and t.is_contiguous()


def address(t: "Tensor | None") -> "int | None":
    return None if t is None else t.data_ptr()


@functools.lru_cache(maxsize=1024)
def _layout(requests: int, rows: int, width: int, max_new: int, Hq: int, Hkv: int, windows: "tuple[int, ...]"):
    """Of plans of this size: (blocks, words of a window's schedule, bytes of a workspace, words of the plan's parts, the native arguments that only
    sizes decide); words -1: none."""
    assert Hkv > 0 and Hq > 0 and Hq % Hkv == 0 and 0 < len(windows) <= PLAN_WINDOWS and len(set(windows)) == len(windows)
    attn = cuda_library("paged_attn")
    blocks = attn.paged_attn_blocks()
    words = cuda_library("page_plan").page_plan_words(requests, rows, max_new, Hq // Hkv, Hkv, blocks)
    workspace = attn.paged_attn_workspace_bytes(requests, rows, width, max_new, Hq, Hkv, blocks)
    parts = [words * len(windows), requests + 1, requests, requests, rows, rows, rows]
    sizes = Plan(rows=rows, requests=requests, max_fresh=max_new, group=Hq // Hkv, kv_heads=Hkv, blocks=blocks, n_windows=len(windows),
                 windows=(ctypes.c_int * PLAN_WINDOWS)(*windows))
    return blocks, words, workspace, parts, bytes(sizes)


class PageTable:
    """Which pages the requests hold, for the pools of every layer, on the device: `table` int32 (requests, width), -1 where there is
    none; `lens` int32 (requests,), positions held; `free` int32 (n_pages,) and `free_count` int32 (1,), the pages nobody holds.
    A page belongs to one request, which holds the pages of its `lens` positions: lengths go up by page_plan and back by trim and release only, since an
    entry behind a request's length counts as empty and its page would be lost. At most 8,192 requests. What changes a table (page_plan, release, trim) is
    one call after the other."""

    def __init__(self, n_pages: int, requests: int, max_len: int, device: "torch.device | str" = "cuda", table: Tensor | None = None,
                 lens: Tensor | None = None, free: Tensor | None = None, free_count: Tensor | None = None):
        self.n_pages, self.requests, self.width = n_pages, requests, cache_pages(max_len)
        new = dict(dtype=torch.int32, device=device)
        self.table = torch.full((requests, self.width), -1, **new) if table is None else table
        self.lens = torch.zeros(requests, **new) if lens is None else lens
        # taken from the end: the first request gets pages 0, 1, ..
        self.free = torch.arange(n_pages - 1, -1, -1, **new) if free is None else free
        self.free_count = torch.full((1,), n_pages, **new) if free_count is None else free_count
        assert _words(self.table, requests, self.width) and _words(self.lens, requests)
        assert _words(self.free, n_pages) and _words(self.free_count, 1)
        assert self.table.device == self.lens.device == self.free.device == self.free_count.device, "a table lives on one device"
        self.ticket = torch.zeros(1, dtype=torch.int32, device=self.device)

    @property
    def device(self) -> torch.device:
        return self.table.device

    @property
    def capacity(self) -> int:
        """Positions a request can hold."""
        return self.width * PAGE_TOKENS

    def release(self, which: Tensor, status: Tensor | None = None) -> None:
        """Requests with which[b] != 0 (int32 (requests,)) give back the pages of their lens[b] positions and hold none."""
        self._give_back("page_release", which, status)

    def trim(self, keep: Tensor, status: Tensor | None = None) -> None:
        """Request b keeps its first keep[b] positions (int32 (requests,); all that it has where that is more, or negative: NCB_DEV_BAD_LENGTH), its new
        lens[b], and gives back the pages behind them: after a step of drafts, pages.trim(pages.lens - rejected)."""
        self._give_back("page_trim", keep, status)

    def _give_back(self, call: str, words: Tensor, status: Tensor | None) -> None:
        assert _words(words, self.requests)
        with on_device_of(self.table, words, status):
            check(getattr(cuda_library("page_plan"), call)(
                pointer(self.table), pointer(self.lens), pointer(words), pointer(self.free), pointer(self.free_count), self.requests, self.width,
                self.n_pages, pointer(status), stream()), call)


class PagePlan:
    """One step of a PageTable's requests, in device memory that page_plan fills (and may fill again):
    row_start (requests + 1,) first rows; fresh (requests,) rows that are served, 0 for a request that is not; lens (requests,)
    positions after the step; pos, place, request (rows,) of every row: its position, page * 64 + position % 64, its request; -1 in pos
    and place of a row that is not served, in all three behind the last request. All int32. Schedules of paged_attention for
    each of `windows`, for Hq query heads over Hkv."""

    def __init__(self, pages: PageTable, rows: int, max_new: int, Hq: int, Hkv: int, windows: "tuple[int, ...]" = (0,)):
        self.pages, self.rows, self.max_new, self.Hq, self.Hkv, self.windows = pages, rows, max_new, Hq, Hkv, tuple(windows)
        n = pages.requests
        self.blocks, words, self.workspace_bytes, parts, sizes = _layout(n, rows, pages.width, max_new, Hq, Hkv, self.windows)
        if words < 0:
            raise ValueError(f"no plan for {n} requests, {rows} rows, at most {max_new} a request, {Hq} heads over {Hkv}")
        flat = pages.table.new_empty(sum(parts))
        self.work, self.row_start, self.fresh, self.lens, self.pos, self.place, self.request = flat.split_with_sizes(parts)
        self.own_lens = self.lens
        self.filled = False  # by page_plan: before, the schedules are whatever was in memory
        self._args = args = Plan.from_buffer_copy(sizes)
        args.width, args.n_pages = pages.width, pages.n_pages
        args.work = work = flat.data_ptr()
        args.row_start = at = work + 4 * parts[0]
        args.served, args.pos = at + 4 * (n + 1), at + 4 * (3 * n + 1)
        args.place, args.request = args.pos + 4 * rows, args.pos + 8 * rows
        self._schedules = {w: work + 4 * words * i for i, w in enumerate(self.windows)}


def page_plan(pages: PageTable, cached: Tensor, new: Tensor, rows: int, *, max_new: int, Hq: int, Hkv: int, windows: "tuple[int, ...]" = (0,),
              lens: Tensor | None = None, free_left: Tensor | None = None, plan: PagePlan | None = None, status: Tensor | None = None) -> PagePlan:
    """One step's bookkeeping in one launch: request b holds cached[b] positions and adds new[b] (int32 (requests,) on the device, 0 for
    a request that idles), whose rows follow the rows of request b - 1 in the step's `rows` rows. Takes the new pages off pages.free
    into pages.table, and returns the step's PagePlan (`plan`: one of the same sizes to fill again, as a captured step does).
    max_new: an upper bound of new known to the host (a step that only decodes says 1: longer requests cost attention a launch). lens: where the new lengths go (may be
    `cached`); free_left: where the count of free pages goes. By default pages.lens and pages.free_count, so that the table is the step's; with free_left elsewhere
    lens is the plan's own by default, and neither moves: the new pages are in pages.table and still on the list, for a caller who keeps both apart.
    Requests are served in order. One that would need more pages than are left (NCB_DEV_NO_PAGES), or that passes the table's
    width, max_new or `rows` or has a negative length (NCB_DEV_BAD_LENGTH), is not served: it keeps its length, and its rows are idle in the operators below."""
    n = pages.requests
    assert _words(cached, n) and _words(new, n)
    assert lens is None or _words(lens, n)
    assert free_left is None or _words(free_left, 1)
    with on_device_of(pages.table, cached, new, lens, free_left, status):
        if plan is None:
            plan = PagePlan(pages, rows, max_new, Hq, Hkv, windows)
        elif plan.pages is not pages or (plan.rows, plan.max_new, plan.Hq, plan.Hkv, plan.windows) != (rows, max_new, Hq, Hkv, tuple(windows)):
            raise ValueError("the plan was made for other sizes or another table")
        plan.lens = lens if lens is not None else pages.lens if free_left is None else plan.own_lens
        args = Plan.from_buffer_copy(plan._args)  # a call's own
        args.table, args.free_pages, args.free_count, args.ticket = pages.table.data_ptr(), pages.free.data_ptr(), pages.free_count.data_ptr(), pages.ticket.data_ptr()
        args.cached, args.fresh, args.lens = cached.data_ptr(), new.data_ptr(), plan.lens.data_ptr()
        args.free_left = (pages.free_count if free_left is None else free_left).data_ptr()
        if status is not None:
            args.status = status.data_ptr()
        check(cuda_library("page_plan").page_plan(ctypes.byref(args), stream()), "page_plan")
        plan.filled = True
    return plan


def paged_append(qkv: Tensor, q_gain: Tensor, k_gain: Tensor, cos: Tensor, sin: Tensor, pos: Tensor, place: Tensor, cache: PagedKVCache,
                 Hq: int, q_out: Tensor | None = None, status: Tensor | None = None) -> Tensor:
    """kv_append into a pool of pages: norm + rotate q and k, and store k and v at place[row] = page * 64 + position % 64 (a plan's
    pos and place; int32 (rows,), no place twice), quantised to e4m3 with a scale per row and head, or in bf16, as the pool is.
    Same bits as kv_append without value embeddings, which this has not. Rows with a negative position or place are idle: nothing is written for them. q_out overlaps nothing
    that is read. Returns q_out (rows, Hq, 128) bf16."""
    (rows, width), Hkv, pages = qkv.shape, cache.kv_heads, cache.pages
    stride, step = qkv.stride()
    assert qkv.dtype is _BF16 and step == 1 and width == (Hq + 2 * Hkv) * HEAD_DIM
    if rows <= 1:
        stride = width  # of a single row it says nothing
    assert _words(pos, rows) and _words(place, rows)
    length, half = table = cos.shape
    assert half == HEAD_DIM // 2 and sin.shape == table and cos.is_contiguous() and sin.is_contiguous()
    assert q_gain.dtype is k_gain.dtype is cos.dtype is sin.dtype is _F32
    assert q_gain.numel() == k_gain.numel() == HEAD_DIM and q_gain.is_contiguous() and k_gain.is_contiguous()
    if q_out is None:
        q_out = qkv.new_empty((rows, Hq, HEAD_DIM))
    else:
        assert q_out.dtype is _BF16 and q_out.shape == (rows, Hq, HEAD_DIM) and q_out.is_contiguous()
    with on_device_of(qkv, q_gain, k_gain, cos, sin, pos, place, pages, q_out, status):
        check(cuda_library("paged_append").paged_append(
            qkv.data_ptr(), q_gain.data_ptr(), k_gain.data_ptr(), cos.data_ptr(), sin.data_ptr(), pos.data_ptr(), place.data_ptr(),
            q_out.data_ptr(), pages.data_ptr(), rows, Hq, Hkv, stride, length, cache.n_pages, cache.e4m3, address(status), stream()),
            "paged_append")
    return q_out


def paged_attention(q: Tensor, cache: PagedKVCache, plan: PagePlan, window: int = 0, softmax_scale: float | None = None,
                    out: Tensor | None = None, workspace: Tensor | None = None, status: Tensor | None = None) -> Tensor:
    """Causal attention of a step's rows over their requests' pages, whose positions already hold the step's own (paged_append): the
    row at position p attends (p - window, p], or [0, p] with window 0. q (rows, Hq, 128) bf16, heads contiguous, row stride free;
    `window` is one that the plan was made with. Rows of requests that the plan did not serve become zeros; rows behind the last
    request are left as they were in `out`. workspace: uint8, plan.workspace_bytes long, for calls that no other stream overlaps
    (default: a new one). `out` overlaps nothing that is read. Scores and sums are fp32; a probability meets the values as f16 (e4m3 pages), as two bf16 terms (bf16 pages, requests of
    at most 16 rows times heads a group) or as one (longer ones), so that a row's last bits may depend on how many rows its request has. Returns out (rows, Hq, 128) bf16."""
    rows, Hq, pages = plan.rows, plan.Hq, plan.pages
    shape = (rows, Hq, HEAD_DIM)
    ldq, head, step = q.stride()
    assert q.dtype is _BF16 and q.shape == shape and step == 1 and (head == HEAD_DIM or Hq == 1)
    if rows <= 1:
        ldq = Hq * HEAD_DIM  # strides of single rows say nothing
    assert cache.kv_heads == plan.Hkv
    work = plan._schedules.get(window)
    if work is None:
        raise ValueError(f"the plan has schedules for windows {plan.windows}, not {window}")
    if not plan.filled:
        raise ValueError("page_plan has not filled this plan")
    if cache.n_pages != pages.n_pages:
        raise ValueError(f"a pool of {cache.n_pages} pages, a table over {pages.n_pages}")
    if out is None:
        out, ldo = q.new_empty(shape), Hq * HEAD_DIM
    else:
        ldo, head, step = out.stride()
        assert out.dtype is _BF16 and out.shape == shape and step == 1 and (head == HEAD_DIM or Hq == 1)
        if rows <= 1:
            ldo = Hq * HEAD_DIM
    size = plan.workspace_bytes
    if workspace is not None:
        assert workspace.is_contiguous(), "a workspace is contiguous: its size says what may be written"
        size = workspace.numel() * workspace.element_size()
    elif size:
        workspace = q.new_empty(size, dtype=torch.uint8)
    args = Paged(q.data_ptr(), cache.pages.data_ptr(), out.data_ptr(), address(workspace), pages.table.data_ptr(), work,
                 address(status), rows, ldq, ldo, size, pages.requests, pages.width, pages.n_pages,
                 plan.max_new, Hq, plan.Hkv, cache.e4m3, window, plan.blocks, _SCALE if softmax_scale is None else softmax_scale)
    with on_device_of(q, cache.pages, pages.table, out, workspace, status):
        check(cuda_library("paged_attn").paged_attn(ctypes.byref(args), stream()), "paged_attn")
    return out
