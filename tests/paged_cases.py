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


def schedule(words, requests, rows, max_new, group, units):
    """[(rows an owner has at most, entries, merges, most parts)] of a schedule: the small kernel's, the tile kernel's, where they run."""
    w = np.asarray(words)
    few, per = 16 // group, 128 // group
    each = min(requests, rows)
    found, at = [], 16
    small, tile = few > 0, max_new > few
    if small:
        merges = 8 * units[0]
        found.append((0, few, each + (0 if tile else rows // few) + 2 * merges, merges))
    if tile:
        found.append((2, per, max(rows // per + min(rows // (few + 1), each), 2 * units[1]), units[1]))
    out = []
    for head, limit, entries, merges in found:
        m = at + 8 * entries
        out.append((limit, w[at:at + 8 * w[head]].reshape(-1, 8), w[m:m + 4 * w[head + 1]].reshape(-1, 4), 2 * merges))
        at = m + 4 * merges
    assert len(w) == -(-at // 4) * 4
    assert small or not w[:2].any()
    assert tile or not w[2:4].any()
    return out
