"""The operators of the paged KV cache, timed: page tables and slot maps made on the GPU from request lengths, the fused append
into pages, and attention of each request's new tokens over its pages.

A cache's positions lie in pages of 64; a pool of pages belongs to one layer, and one block table (request, page number) -> page
serves every layer. Kinds of cases:

plan      one step's bookkeeping: each request has `cached` positions and adds `new` ones; pages are taken off the free list, and
          every new row gets its position and its place (page * 64 + position in the page)
append    QK-norm, rotation and the store of a step's k and v rows in their places; e4m3 with a scale per row and head, or bf16
attend    causal attention of the new rows of every request over its pages, whose positions already hold the new rows

A page of e4m3 is, per key/value head, 16,896 bytes: K rows with swizzled 16-byte chunks, V transposed in blocks of 16 positions,
64 K scales and 64 V scales in fp32; a page of bf16 is [2][64][128], keys then values."""

import math

import torch

own = False
DEV, HEAD, HALF, PAGE, CODES = "cuda", 128, 64, 64, 16384
F64, I64, I32 = torch.float64, torch.int64, torch.int32
EPS, THETA = 1.1920928955078125e-07, 10000.0


def listed() -> list:
    return [
        # one decode step of the benchmark's batch: a full batch of long chats, one token each
        {"name": "plan_decode_64", "kind": "plan", "requests": 64, "shortest": 200, "longest": 8192, "new": 1, "chunk": 1, "chunks": 0, "idle": 3,
         "heads": 32, "kv_heads": 8, "window": 0, "spare": True},
        # a large server's step: a thousand requests, prompts being read in chunks beside them
        {"name": "plan_server_1025", "kind": "plan", "requests": 1025, "shortest": 16, "longest": 4000, "new": 1, "chunk": 509, "chunks": 120,
         "idle": 40, "heads": 32, "kv_heads": 8, "window": 0, "spare": True},
        # one layer of that decode step: 64 rows
        {"name": "append_decode_e4m3", "kind": "append", "dtype": "e4m3", "requests": 64, "shortest": 200, "longest": 8191, "new": 1, "chunk": 1,
         "chunks": 0, "idle": 0, "heads": 32, "kv_heads": 8, "window": 0},
        # one layer of eight prompts read at once
        {"name": "append_prompts_bf16", "kind": "append", "dtype": "bf16", "requests": 8, "shortest": 0, "longest": 0, "new": 1023, "chunk": 1023,
         "chunks": 0, "idle": 0, "heads": 32, "kv_heads": 8, "window": 0},
        # the smallest call: three users of the small model, a few hundred positions each
        {"name": "attend_three_bf16", "kind": "attend", "dtype": "bf16", "requests": 3, "shortest": 300, "longest": 700, "new": 1, "chunk": 1,
         "chunks": 0, "idle": 0, "heads": 10, "kv_heads": 10, "window": 0},
        # the benchmark's default workload, paged
        {"name": "attend_decode_e4m3", "kind": "attend", "dtype": "e4m3", "requests": 64, "shortest": 8191, "longest": 8191, "new": 1, "chunk": 1,
         "chunks": 0, "idle": 0, "heads": 32, "kv_heads": 8, "window": 0},
        # contexts from a question to a long document in one batch, an odd number of requests
        {"name": "attend_ragged_bf16", "kind": "attend", "dtype": "bf16", "requests": 47, "shortest": 130, "longest": 16384, "new": 1, "chunk": 1,
         "chunks": 0, "idle": 2, "heads": 16, "kv_heads": 4, "window": 0},
        # drafted tokens checked together, in a layer with a sliding window
        {"name": "attend_drafts_window", "kind": "attend", "dtype": "e4m3", "requests": 33, "shortest": 500, "longest": 6000, "new": 5, "chunk": 5,
         "chunks": 0, "idle": 0, "heads": 16, "kv_heads": 4, "window": 1024},
        # a chunk of a long document behind what was read before
        {"name": "attend_chunk_bf16", "kind": "attend", "dtype": "bf16", "requests": 1, "shortest": 16384, "longest": 16384, "new": 512, "chunk": 512,
         "chunks": 0, "idle": 0, "heads": 32, "kv_heads": 8, "window": 0},
        # a server's mixed step: chats that decode, two prompts in chunks
        {"name": "attend_mixed_e4m3", "kind": "attend", "dtype": "e4m3", "requests": 17, "shortest": 300, "longest": 4000, "new": 1, "chunk": 509,
         "chunks": 2, "idle": 0, "heads": 16, "kv_heads": 4, "window": 0},
        # one layer of a long document's prefill
        {"name": "attend_prompt_bf16", "kind": "attend", "dtype": "bf16", "requests": 1, "shortest": 0, "longest": 0, "new": 8190, "chunk": 8190,
         "chunks": 0, "idle": 0, "heads": 16, "kv_heads": 4, "window": 0},
    ]


def draw(rng) -> dict:
    def spread(low: int, high: int) -> int:
        return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))

    kv_heads, ratio = rng.choice([(10, 1), (4, 4), (8, 4), (6, 2), (16, 1), (2, 8), (5, 3), (1, 12)])
    case = {"kind": rng.choice(["plan", "append", "attend", "attend", "attend"]), "dtype": rng.choice(["e4m3", "bf16"]), "heads": kv_heads * ratio,
            "kv_heads": kv_heads, "window": rng.choice([0, 0, 0, 100, 1024]), "idle": 0}
    if case["kind"] == "plan":
        requests = spread(1, 1200)
        longest = spread(64, 8192)
        chunks = rng.choice([0, 0, requests // 9, requests // 3])
        return case | {"requests": requests, "shortest": spread(1, longest), "longest": longest, "new": rng.choice([1, 1, 4]),
                       "chunk": spread(2, max(2, min(2048, 61000 // max(chunks, 1)))), "chunks": chunks, "idle": rng.choice([0, requests // 10]),
                       "spare": rng.random() < 0.7}
    if case["kind"] == "append":
        new = spread(1, 2048)
        requests = max(1, min(spread(1, 64), 8184 // new))
        longest = spread(1, 4096)
        return case | {"requests": requests, "shortest": rng.choice([0, longest]), "longest": longest, "new": new, "chunk": new, "chunks": 0}
    form = rng.choice(["decode", "decode", "drafts", "chunk", "mixed", "prompt"])
    if form in ("decode", "drafts"):
        requests = spread(1, 64)
        longest = spread(32, 16384 if requests * kv_heads <= 192 else 8192)
        new = 1 if form == "decode" else rng.randint(2, 20)
        return case | {"requests": requests, "shortest": spread(16, longest), "longest": longest, "new": new, "chunk": new, "chunks": 0,
                       "idle": requests // 8}
    if form == "chunk":
        longest, new = spread(100, 16384), spread(8, 700)
        requests = max(1, min(rng.randint(1, 6), 40_000_000 // ((longest + new) * new * kv_heads)))
        return case | {"requests": requests, "shortest": spread(16, longest), "longest": longest, "new": new, "chunk": new, "chunks": 0}
    if form == "mixed":
        longest, chunk = spread(100, 4096), spread(20, 400)
        requests = rng.randint(2, 16)
        return case | {"requests": requests, "shortest": spread(16, longest), "longest": longest, "new": rng.choice([1, 1, 3]), "chunk": chunk,
                       "chunks": rng.randint(1, 2)}
    new = spread(16, 4096)
    requests = max(1, min(rng.randint(1, 8), 4096 // new))
    return case | {"requests": requests, "shortest": 0, "longest": 0, "new": new, "chunk": new, "chunks": 0}


def lengths(case: dict) -> tuple:
    """(cached, new) of every request: contexts from the shortest to the longest by equal factors; the last `chunks` requests add a
    chunk (sizes a little apart), the first `idle` nothing."""
    n, low, high = case["requests"], case["shortest"], case["longest"]
    cached = [int(round((low + 1) * ((high + 1) / (low + 1)) ** (i / max(n - 1, 1)))) - 1 for i in range(n - 1)] + [high]
    new = [case["new"]] * n
    for i in range(min(case["chunks"], n)):
        new[n - 1 - i] = max(1, case["chunk"] - 3 * (i % 5))
    for i in range(min(case["idle"], n - 1)):
        new[i] = 0
    return cached, new


def pages_of(positions: int) -> int:
    return -(-positions // PAGE)


# ---- inputs -----------------------------------------------------------------------------------------------------------------


def k_index() -> torch.Tensor:
    """Where the code of (position, dimension) of a key lies in an e4m3 page, flat."""
    j, d = torch.arange(PAGE, device=DEV)[:, None], torch.arange(HEAD, device=DEV)[None, :]
    return (j * HEAD + (((d >> 4) ^ ((j >> 2) & 7)) << 4) + (d & 15)).reshape(-1)


def v_index() -> torch.Tensor:
    j, d = torch.arange(PAGE, device=DEV)[:, None], torch.arange(HEAD, device=DEV)[None, :]
    return (8192 + (j >> 5) * 4096 + ((j >> 4) & 1) * 2048 + d * 16 + (j & 15)).reshape(-1)


def quantised(x: torch.Tensor) -> tuple:
    """(e4m3 codes, fp32 scales) of rows of 128."""
    scale = x.abs().amax(-1) / 448
    return (x / torch.where(scale > 0, scale, 1.0)[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn), scale


def filled_pool(case: dict, pages: int, gen: torch.Generator) -> torch.Tensor:
    """Pages full of keys and values as a model leaves them: around a mean of their own per head."""
    heads = case["kv_heads"]
    mean = torch.randn(heads, 2, 1, HEAD, device=DEV, generator=gen) * 0.5
    e4m3 = case["dtype"] == "e4m3"
    pool = torch.empty((pages, heads, CODES + 512) if e4m3 else (pages, heads, 2, PAGE, HEAD), dtype=torch.uint8 if e4m3 else torch.bfloat16, device=DEV)
    for at in range(0, pages, 1024):
        part = pool[at:at + 1024]
        x = torch.randn(len(part), heads, 2, PAGE, HEAD, device=DEV, generator=gen) + mean
        if e4m3:
            codes, scale = quantised(x.bfloat16().float())
            codes = codes.view(torch.uint8)
            part[..., k_index()] = codes[:, :, 0].flatten(2)
            part[..., v_index()] = codes[:, :, 1].flatten(2)
            part.view(torch.float32)[..., CODES // 4:] = scale.flatten(2)
        else:
            part.copy_(x)
    return pool


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device=DEV).manual_seed(seed)
    cached, new = (torch.tensor(v, device=DEV) for v in lengths(case))
    order = torch.randperm(len(cached), device=DEV, generator=gen)
    cached, new = cached[order], new[order]
    have, need = (cached + 63) // PAGE, torch.where(new > 0, (cached + new + 63) // PAGE - (cached + 63) // PAGE, 0)
    total = int(have.sum() + need.sum())
    width = int(((cached + new + 63) // PAGE).max()) + 1
    extra = 5 if case.get("spare", True) else -(int(need.sum()) // 4)  # not spare: the pool runs out for some requests
    pages = max(total + extra, 1)
    shuffled = torch.randperm(pages, device=DEV, generator=gen).to(I32)
    table = torch.full((len(cached), width), -1, dtype=I32, device=DEV)
    held = torch.arange(width, device=DEV)[None] < have[:, None]
    taken = int(have.sum())
    table[held] = shuffled[:taken]
    rows = int(new.sum())
    rows += (-rows) % 64 if case["kind"] == "plan" else 0  # a captured step's rows are rounded up
    free = torch.zeros(pages, dtype=I32, device=DEV)
    free[:pages - taken] = shuffled[taken:]
    state = {"case": case, "table": table, "free": free, "free_count": torch.tensor([pages - taken], dtype=I32, device=DEV),
             "cached": cached.to(I32), "new": new.to(I32), "rows": rows, "max_new": max(lengths(case)[1])}
    heads, kv_heads, dim = case["heads"], case["kv_heads"], HEAD
    if case["kind"] != "plan":
        state.update(plain_plan(state))
        state["pool"] = filled_pool(case, pages, gen)
    if case["kind"] == "append":
        state["qkv"] = torch.randn(rows, (heads + 2 * kv_heads) * dim, device=DEV, generator=gen).bfloat16()
        state["gain"] = [1 + 0.1 * torch.randn(dim, device=DEV, generator=gen) for _ in "qk"]
        angles = torch.arange(max(a + b for a, b in zip(*lengths(case))), dtype=F64, device=DEV)[:, None] * THETA ** -(torch.arange(0, dim, 2, dtype=F64, device=DEV) / dim)
        state["cos"], state["sin"] = angles.cos().float(), angles.sin().float()
    if case["kind"] == "attend":
        state["q"] = (torch.randn(rows, heads, dim, device=DEV, generator=gen) + 0.5 * torch.randn(heads, dim, device=DEV, generator=gen)).bfloat16()
    if own:  # the handles that a server keeps, and for a layer's attention the step's plan
        import nanochat_b200 as ncb

        state["pages"] = ncb.PageTable(pages, len(cached), width * PAGE, device=DEV, table=state["table"], free=free, free_count=state["free_count"])
        state["free_left"] = torch.empty(1, dtype=I32, device=DEV)
        if case["kind"] != "plan":
            state["cache"] = ncb.PagedKVCache(pages, kv_heads, torch.bfloat16 if case["dtype"] == "bf16" else torch.float8_e4m3fn, device=DEV, pages=state["pool"])
        if case["kind"] == "attend":
            state["plan"] = ncb.page_plan(state["pages"], state["cached"], state["new"], rows, max_new=state["max_new"], Hq=heads, Hkv=kv_heads,
                                          windows=(case["window"],), free_left=state["free_left"])
    return state


# ---- plain forms ------------------------------------------------------------------------------------------------------------


def plain_plan(s: dict) -> dict:
    """Requests are served in order while free pages last; a request that is not served keeps its length and its rows count for
    nothing. Pages come from the end of the free list."""
    table, cached, new, rows = s["table"].clone(), s["cached"].to(I64), s["new"].to(I64), s["rows"]
    free, count = s["free"].to(I64), s["free_count"].to(I64)
    row_end = new.cumsum(0)
    valid = (new > 0) & (cached >= 0) & (cached + new <= table.shape[1] * PAGE) & (row_end <= rows)
    have = (cached + PAGE - 1) // PAGE
    need = torch.where(valid, (cached + new + PAGE - 1) // PAGE - have, 0)
    upto = need.cumsum(0)
    served = valid & ((need == 0) | (upto <= count))
    col = torch.arange(table.shape[1], device=table.device)[None]
    fresh = served[:, None] & (col >= have[:, None]) & (col < (have + need)[:, None])
    source = count - 1 - ((upto - need)[:, None] + col - have[:, None])
    table = torch.where(fresh, free[source.clamp(0, len(free) - 1)].to(I32), table)
    at = torch.arange(rows, device=table.device)
    request = torch.searchsorted(row_end, at, right=True)
    inside = request < len(new)
    request = request.clamp(max=len(new) - 1)
    on = inside & served[request]
    pos = torch.where(on, cached[request] + at - (row_end - new)[request], -1)
    page = table[request, pos.clamp(min=0) // PAGE].to(I64)
    return {"table": table, "row_start": torch.cat([row_end.new_zeros(1), row_end]).to(I32), "fresh": torch.where(served, new, 0).to(I32),
            "lens": torch.where(served, cached + new, cached.clamp(min=0)).to(I32), "pos": pos.to(I32),
            "place": torch.where(on, page * PAGE + pos % PAGE, -1).to(I32), "request": torch.where(inside, request, -1).to(I32),
            "free_left": (count - torch.where(served, need, 0).sum()).to(I32)}


PLAN_OUT = ("table", "row_start", "fresh", "lens", "pos", "place", "request", "free_left")


def stored(s: dict) -> tuple:
    """The pool as the values it stands for."""
    pool = s["pool"]
    if s["case"]["dtype"] == "bf16":
        return (pool,)
    return pool[..., :CODES].view(torch.float8_e4m3fn), pool.view(torch.float32)[..., CODES // 4:]


def plain_append(s: dict) -> tuple:
    """q and k: RMS norm, gain, rotation by the row's position (pairs i, i + 64), one rounding to bf16; k and v into their places. The
    framework defines a cache's bytes and scales bit by bit: every operation in fp32 with its own rounding, and the squares summed in
    this order, so that no key next to a rounding border falls to its other side."""
    case, place = s["case"], s["place"].to(I64)
    heads, kv_heads = case["heads"], case["kv_heads"]
    x = s["qkv"].float().view(len(place), -1, HEAD)
    qk = x[:, :heads + kv_heads]
    square = qk * qk
    pair = (square[..., :HALF] + square[..., HALF:]).unflatten(-1, (8, 8))
    eighth = pair[..., 0] + pair[..., 1] + pair[..., 2] + pair[..., 3] + pair[..., 4] + pair[..., 5] + pair[..., 6] + pair[..., 7]
    quarter = eighth[..., :4] + eighth[..., 4:]
    half = quarter[..., :2] + quarter[..., 2:]
    qk = qk * (1.0 / torch.sqrt((half[..., :1] + half[..., 1:]) * (1 / HEAD) + EPS))
    qk = qk * torch.cat([s["gain"][0].expand(heads, HEAD), s["gain"][1].expand(kv_heads, HEAD)])
    cos, sin = (s[n][s["pos"].to(I64)][:, None] for n in ("cos", "sin"))
    a, b = qk[..., :HALF], qk[..., HALF:]
    qk = torch.cat([a * cos + b * sin, b * cos - a * sin], -1).bfloat16()
    page, j, pool = place // PAGE, place % PAGE, s["pool"]
    k, v = qk[:, heads:], s["qkv"].view(len(place), -1, HEAD)[:, heads + kv_heads:]
    head = torch.arange(kv_heads, device=page.device)
    if case["dtype"] == "bf16":
        pool[page[:, None], head, 0, j[:, None]] = k
        pool[page[:, None], head, 1, j[:, None]] = v
    else:
        dims = torch.arange(HEAD, device=page.device)
        for x, index, side in ((k, k_index(), 0), (v, v_index(), 1)):
            codes, scale = quantised(x.float())
            pool[page[:, None, None], head[:, None], index.view(PAGE, HEAD)[j][:, None, dims]] = codes.view(torch.uint8)
            pool.view(torch.float32)[page[:, None], head, CODES // 4 + side * PAGE + j[:, None]] = scale
    return qk[:, :heads].contiguous(), *stored(s)


def gathered(s: dict, dtype) -> tuple:
    """Keys and values of every request up to the longest, [requests, key/value heads, positions, 128]."""
    pool, lens = s["pool"], s["lens"].to(I64)
    table = s["table"].to(I64)[:, :-1].clamp(min=0)
    pages = pool[table].transpose(1, 2)  # [requests, heads, pages, ...]
    if s["case"]["dtype"] == "bf16":
        k, v = (pages[:, :, :, i].flatten(2, 3).to(dtype) for i in range(2))
    else:
        scales = pages.view(torch.float32)[..., CODES // 4:].to(dtype)
        k, v = (pages[..., index].view(torch.float8_e4m3fn).to(torch.float32).to(dtype).unflatten(-1, (PAGE, HEAD)) * scales[..., side * PAGE:side * PAGE + PAGE, None]
                for index, side in ((k_index(), 0), (v_index(), 1)))
        k, v = k.flatten(2, 3), v.flatten(2, 3)
    seen = (torch.arange(k.shape[2], device=k.device) < lens[:, None])[:, None, :, None]
    return torch.where(seen, k, 0), torch.where(seen, v, 0)


def plain_attend(s: dict) -> torch.Tensor:
    """softmax(q k / sqrt(128)) v over positions (p - window, p] of the request, p the row's own."""
    case, q = s["case"], s["q"]
    heads, kv_heads, window = case["heads"], case["kv_heads"], case["window"]
    group, most = heads // kv_heads, s["max_new"]
    row = s["row_start"].to(I64)[:-1, None] + torch.arange(most, device=q.device)
    used = torch.arange(most, device=q.device) < s["fresh"].to(I64)[:, None]
    row = torch.where(used, row, 0)
    pos = torch.where(used, s["pos"].to(I64)[row], -1)
    x = q.float()[row].unflatten(2, (kv_heads, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)  # [requests, kv heads, group * new, 128]
    k, v = gathered(s, torch.float32)
    score = (x * HEAD ** -0.5) @ k.transpose(2, 3)
    at = torch.arange(k.shape[2], device=q.device)
    mask = at > pos[..., None]
    if window:
        mask |= at <= pos[..., None] - window
    score = score.unflatten(2, (group, most)).masked_fill_(mask[:, None, None], -math.inf)
    score = torch.exp_(score.sub_(score.amax(-1, keepdim=True).clamp_(min=-3e38)))
    total = score.sum(-1, keepdim=True)
    o = (score.flatten(2, 3) @ v).unflatten(2, (group, most)) / torch.where(total > 0, total, 1.0)
    out = torch.zeros_like(q)
    out[row[used]] = o.permute(0, 3, 1, 2, 4).flatten(2, 3)[used].to(q.dtype)
    return out


# ---- one pass ---------------------------------------------------------------------------------------------------------------


def run(s: dict):
    case = s["case"]
    if not own:
        if case["kind"] == "plan":
            found = plain_plan(s)
            return [found[n] for n in PLAN_OUT]
        return plain_append(s) if case["kind"] == "append" else plain_attend(s)
    import nanochat_b200 as ncb

    if case["kind"] == "plan":
        plan = ncb.page_plan(s["pages"], s["cached"], s["new"], s["rows"], max_new=s["max_new"], Hq=case["heads"], Hkv=case["kv_heads"],
                             windows=(case["window"],), free_left=s["free_left"])
        return [s["pages"].table, plan.row_start, plan.fresh, plan.lens, plan.pos, plan.place, plan.request, s["free_left"]]
    if case["kind"] == "append":
        q = ncb.paged_append(s["qkv"], *s["gain"], s["cos"], s["sin"], s["pos"], s["place"], s["cache"], case["heads"])
        return (q, *stored(s))
    return ncb.paged_attention(s["q"], s["cache"], s["plan"], window=case["window"])


def work(case: dict) -> dict:
    cached, new = lengths(case)
    rows, heads, kv_heads = sum(new), case["heads"], case["kv_heads"]
    if case["kind"] == "plan":  # lengths in; table entries, row starts, lengths and four words a row out
        need = sum(pages_of(c + n) - pages_of(c) for c, n in zip(cached, new) if n)
        rows += (-rows) % 64
        return {"bytes": 4 * (2 * len(new) + 2 * need + 3 * len(new) + 3 * rows), "flops": 0}
    row = 2 * HEAD if case["dtype"] == "bf16" else HEAD + 4  # a key or a value in the cache
    if case["kind"] == "append":
        values = rows * HEAD
        table = 2 * 4 * HALF * len({p for c, n in zip(cached, new) for p in range(c, c + n)})
        return {"bytes": 2 * values * (2 * heads + 2 * kv_heads) + 2 * rows * kv_heads * row + table + 8 * rows, "flops": 12 * values * (heads + kv_heads)}
    span = pairs = 0
    for c, n in zip(cached, new):
        if n:
            first = max(0, c + 1 - case["window"]) if case["window"] else 0
            span += c + n - first
            pairs += sum(min(c + i + 1, case["window"] or c + i + 1) for i in range(n))
    return {"bytes": span * kv_heads * 2 * row + 2 * 2 * rows * heads * HEAD, "flops": 4 * pairs * heads * HEAD}


# ---- the same in 64 bits ----------------------------------------------------------------------------------------------------


def exact(case: dict, seed: int):
    s = prepare(case, seed)
    if case["kind"] == "plan":
        return None  # whole numbers
    heads, kv_heads, window = case["heads"], case["kv_heads"], case["window"]
    if case["kind"] == "append":
        x = s["qkv"].to(F64).view(s["rows"], -1, HEAD)
        turn = torch.complex(s["cos"].to(F64), -s["sin"].to(F64))[s["pos"].long()][:, None]

        def rotated(part, gain):
            part = part * torch.rsqrt((part * part).sum(-1, keepdim=True) / HEAD + EPS) * gain.to(F64)
            z = torch.complex(part[..., :HALF], part[..., HALF:]) * turn
            return torch.cat([z.real, z.imag], -1)

        q, k = rotated(x[:, :heads], s["gain"][0]), rotated(x[:, heads:heads + kv_heads], s["gain"][1])
        page, j = s["place"].long() // PAGE, s["place"].long() % PAGE
        if case["dtype"] == "bf16":
            pool = s["pool"].to(F64)
            for h in range(kv_heads):
                pool[page, h, 0, j], pool[page, h, 1, j] = k[:, h], x[:, heads + kv_heads + h]
            return q, pool
        codes = stored(s)[0].to(torch.float32).to(F64)
        k = k.to(torch.bfloat16).to(F64)  # the cache takes the rounded key
        for h in range(kv_heads):
            for side, index, row in ((0, k_index(), k[:, h]), (1, v_index(), x[:, heads + kv_heads + h])):
                scale = row.abs().amax(-1) / 448
                codes[page[:, None], h, index.view(PAGE, HEAD)[j]] = row / torch.where(scale > 0, scale, 1.0)[:, None]
        return q, codes, None  # a scale follows from the key's rounded bits, which 64 bits would place otherwise at a border
    out = torch.zeros(s["rows"], heads, HEAD, dtype=F64, device=DEV)
    group = heads // kv_heads
    for b in range(case["requests"]):
        n, length, first = int(s["fresh"][b]), int(s["lens"][b]), int(s["row_start"][b])
        if n == 0:
            continue
        pages = s["pool"][s["table"][b, :pages_of(length)].long()]
        for h in range(kv_heads):
            if case["dtype"] == "bf16":
                k, v = (pages[:, h, i].reshape(-1, HEAD)[:length].to(F64) for i in range(2))
            else:
                scale = pages[:, h].contiguous().view(torch.float32)[:, CODES // 4:].to(F64)
                k, v = ((pages[:, h][:, index].view(torch.float8_e4m3fn).float().to(F64).view(-1, PAGE, HEAD) * scale[:, i * PAGE:(i + 1) * PAGE, None])
                        .reshape(-1, HEAD)[:length] for i, index in ((0, k_index()), (1, v_index())))
            for at in range(0, n, 1024):
                rows = torch.arange(at, min(at + 1024, n), device=DEV)
                x = s["q"][first + rows].to(F64)[:, h * group:(h + 1) * group]
                z = torch.einsum("rgd,kd->rgk", x, k) / math.sqrt(HEAD)
                behind = (length - n + rows)[:, None] - torch.arange(length, device=DEV)  # how far back a position lies
                unseen = behind < 0 if window == 0 else (behind < 0) | (behind >= window)
                p = torch.softmax(z.masked_fill(unseen[:, None], -math.inf), -1)
                out[first + rows, h * group:(h + 1) * group] = torch.einsum("rgk,kd->rgd", p, v)
    return out
