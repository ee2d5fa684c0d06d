"""Steps of a page pool and their plans, sequence by sequence in plain Python."""
from __future__ import annotations

import numpy as np

NAMES = ("took", "q_start", "len_out", "next_pos_out", "n_free_out", "slot", "pos", "seq", "table", "free_pages")


def pool(r, lens, page, extra, max_pages, spare=0):
    """table, free_pages, n_free of a pool whose sequences hold `lens` rows and that has `extra` free pages; `spare`
    pages are of neither."""
    counts = [-(-n // page) for n in lens]
    n_pages = sum(counts) + extra + spare
    order = r.permutation(n_pages).astype(np.int32)
    table = np.full((len(lens), max_pages), -9, np.int32)       # (entries behind the last page hold anything)
    at = 0
    for b, c in enumerate(counts):
        table[b, :c] = order[at:at + c]
        at += c
    free = np.full(max(n_pages, 1), -8, np.int32)
    free[:extra] = order[at:at + extra]
    return table, free, extra


def plan(lens, new, table, free, n_free, page, n_tok, ended=None, next_pos=None):
    """The definition of vx27_hip_paged_plan."""
    B, max_pages = table.shape
    ended = [0] * B if ended is None else ended
    table, free, lens, new = table.copy(), free.copy(), list(lens), list(new)
    nxt = list(lens) if next_pos is None else list(next_pos)
    stack = [int(x) for x in free[:n_free]]
    for b in range(B):
        if ended[b]:
            stack += [int(x) for x in table[b, :-(-lens[b] // page)]]
            lens[b] = new[b] = nxt[b] = 0
    total, wanted, tokens = len(stack), 0, 0
    out = {n: [] for n in NAMES}
    start = [0]
    for b in range(B):
        n, t = int(lens[b]), int(new[b])
        need = -(-(n + t) // page) - -(-n // page)
        if n + t > max_pages * page:
            t = 0
        else:
            wanted += need
            if need and wanted > total:
                t = 0
        tokens += t
        if tokens > n_tok:
            t = 0
        if t:
            for i in range(need):
                table[b, -(-n // page) + i] = stack.pop()
        out["took"].append(t)
        out["len_out"].append(n + t)
        out["next_pos_out"].append(int(nxt[b]) + t)
        start.append(start[-1] + t)
        for r in range(n, n + t):
            out["slot"].append(int(table[b, r // page]) * page + r % page)
            out["pos"].append(int(nxt[b]) + r - n)
            out["seq"].append(b)
    out["q_start"], out["n_free_out"] = start, [len(stack)]
    if len(stack) > n_free:
        free[n_free:len(stack)] = stack[n_free:]
    for n in ("slot", "pos", "seq"):
        out[n] += [-1] * (n_tok - len(out[n]))
    out["table"], out["free_pages"] = table, free
    return {n: np.array(x, np.int32) for n, x in out.items()}
