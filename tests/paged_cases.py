"""Plain restatements of the paged operators for the tests: a step's bookkeeping as a loop over requests, attention in 64 bits."""

import numpy as np
import torch

PAGE = 64


def plan(table, cached, new, free, rows, max_new):
    """page_plan on lists: returns the dict of its outputs (table included, `left` free pages) and the NCB_DEV bits."""
    table, n_free, bits = [list(r) for r in table], len(free), 0
    width = len(table[0])
    out = {"row_start": [0], "fresh": [], "lens": [], "pos": [-1] * rows, "place": [-1] * rows, "request": [-1] * rows}
    wanted = 0
    taken = 0
    for b, (c, n) in enumerate(zip(cached, new)):
        start = out["row_start"][-1]
        out["row_start"].append(min(start + max(n, 0), 2 ** 31 - 1))  # 32-bit words
        ok = c >= 0 and 0 <= n <= max_new and c + n <= width * PAGE and (n == 0 or start + n <= rows)
        bits |= 0 if ok else 4
        need = -(-(c + n) // PAGE) - -(-c // PAGE) if ok and n else 0
        served = ok and n > 0
        if need and wanted + need > n_free:
            served = False
            bits |= 8
        if served:
            for i in range(need):
                table[b][-(-c // PAGE) + i] = free[n_free - 1 - wanted - i]
            taken += need
        wanted += need
        out["fresh"].append(n if served else 0)
        out["lens"].append(max(c, 0) + (n if served else 0))
        for i in range(min(n, rows - start)):
            out["request"][start + i] = b
            if served:
                out["pos"][start + i] = c + i
                out["place"][start + i] = table[b][(c + i) // PAGE] * PAGE + (c + i) % PAGE
    out["table"], out["left"] = table, n_free - taken
    return out, bits


def attention(q, k, v, first_pos, window):
    """Rows q (n, Hq, 128) at positions first_pos .. over keys, values (Hkv, len, 128), all fp64: (outputs, sums of p |v|)."""
    n, Hq, _ = q.shape
    group = Hq // k.shape[0]
    out, size = torch.zeros_like(q), torch.zeros_like(q)
    for i in range(n):
        last = first_pos + i
        begin = max(0, last + 1 - window) if window else 0
        kk, vv = (x[:, begin:last + 1].repeat_interleave(group, 0) for x in (k, v))
        p = torch.softmax(torch.einsum("hd,hkd->hk", q[i], kk) * 128 ** -0.5, -1)
        out[i] = torch.einsum("hk,hkd->hd", p, vv)
        size[i] = torch.einsum("hk,hkd->hd", p, vv.abs())
    return out, size


def few_slots_bound(want, size):
    """What requests of at most 16 query slots may be off over bf16 pages: a result's rounding 2^-8, a probability's two bf16 terms 2^-16 (2^-8 of
    the first one's 2^-8), scores, sums and exponentials in 32 bits 2^-14."""
    return 2.0 ** -8 * want.abs() + (2.0 ** -16 + 2.0 ** -14) * size


def schedule(words, requests, rows, max_new, group, sms):
    """[(rows an owner has at most, blocks, overhead, least share, [total, share, whole], owners, starts, joins, pieces)] of a schedule's classes."""
    w = np.asarray(words)
    few, each = 16 // group, min(requests, rows)
    classes = []
    tiles = max_new > few and rows > few
    if few and rows:
        per = min(few, max_new)
        classes.append((per, each if tiles else (rows + each * (per - 1)) // per, 3 * sms, 2, 6, 0))
    if tiles:
        per = 128 // group * 2
        classes.append((per, rows // per + min(rows // (few + 1), each), sms, 4, 8, 9 * sms))
    found, at = [], 0
    for per, most, blocks, overhead, least, room in classes:
        n = int(w[at])
        assert n <= most
        owners = w[at + 8:at + 8 + 8 * n].reshape(-1, 8)
        starts = at + 8 + 8 * most
        joins = starts + 4 * ((blocks + 2) // 2 * 2)
        pieces = joins + 8 * blocks
        found.append((per, blocks, overhead, least, w[at + 1:at + 4].tolist(), owners, w[starts:starts + 4 * (blocks + 1)].reshape(-1, 4),
                      w[joins:pieces].reshape(-1, 8), w[pieces:pieces + 8 * room].reshape(-1, 8)))
        at = pieces + 8 * room
    assert at == len(w)
    return found


def last_whole(weights, heads, blocks):
    """A bound of the last block's work if owners are whole: the heaviest, and what some block has of all owners of at least a weight."""
    top, last, n = int(weights.max()), int(weights.max()), 0
    steps = (weights.astype(np.int64) * 16 - 1) // top
    for i in range(15, -1, -1):
        here = weights[steps == i]
        n += len(here)
        if len(here):
            last = max(last, -(-n * heads // blocks) * int(here.min()))
    return last


def pieces(owners, heads, blocks, overhead, total, share):
    """What the blocks do with a class that is cut: (block, head, owner, page0, page1, part), and by (head, owner) the blocks whose parts are joined."""
    done, joined = [], {}
    for head in range(heads):
        for i, o in enumerate(owners.tolist()):
            first = head * total + o[6] + overhead
            stop = first + max(o[5], 1)
            b0, b1 = first // share, (stop - 1) // share
            assert b1 < blocks
            if b1 > b0:
                joined[head, i] = [2 * b + (b == b0) for b in range(b0, b1 + 1)]
            for b in range(b0, b1 + 1):
                x, y = max(b * share, first), min((b + 1) * share, stop)
                done.append((b, head, i, x - first, min(y - first, o[5]), -1 if b0 == b1 else 2 * b + (x == first)))
    return done, joined
