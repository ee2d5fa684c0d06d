"""The operators of a paged cache held in 4 bits, as timed cases.

A server of many conversations that keeps their key-value rows in 4 bits, per step

  plan     gives the sequences their new tokens' rows: releases the pages of
           ended ones, takes pages from the free ones, extends the page tables,
           and leaves the ragged ranges, slots and positions that the other
           calls read (vx27_hip_paged_plan)

and per GQA layer

  append   norms and rotates the new tokens' queries and keys and rounds keys
           and values to 4 bits in the pages (vx27_hip_paged_append_q4)
  attn     attends from the new tokens to the cached rows: all of them, or a
           sliding window and the first few rows (vx27_hip_paged_attn_q4)
  read     gives the values of rows by slot, as a program does that moves a
           conversation out of the pool (vx27_hip_paged_read_q4)

The heads are those of the Qwen 27B hybrid's attention layers (24 query and 4
KV heads of 256, RoPE over 64 dimensions); draws take other groupings too.

A page holds P / 32 blocks of 32 rows for each KV head, [n_pages][n_kv][P/32]
of 4608 bytes each of K and of V. A row's 256 dims are four groups of 64; the
value of a dim is m + s c, with s and m of its row and group (bf16) and a 4-bit
code c:  m is the largest bf16 number not above the group's values, s the
smallest bf16 number at least (largest value - m) / 15, c the integer nearest
to (x - m) / s (ties to even). Bytes of a block, from the slowest index:
  K   0     codes [row/4%2][dim/128][dim/8%4][row/8][row%4][dim/32%4][dim%4], dims 4..7 of 8 in the high halves
      4096  s [dim/64][row]     4352  m [row][dim/64]
  V   0     codes [dim/64][row/8][dim%16][dim/16%4][row%4], rows 4..7 of 8 in the high halves
      4096  s [dim/64][row]     4352  m [dim/64][row]
"""
from __future__ import annotations

import ctypes as C
import math
import random

import torch

own = False

HD = 256                       # head dim
ROPE, THETA, EPS = 64, 1e7, 1e-6
BLOCK = 4608                   # bytes of 32 rows of K or of V
DEV = "cuda"
BF = torch.bfloat16
DBL = torch.float64


# ------------------------------------------------------------------- cases
def _case(kind, **kw):
    c = {"kind": kind, "n_q": 24, "n_kv": 4, "page": 64}
    if kind == "attn":
        c.update(T=1, ragged=False, out="bf16", gate="bf16", window=0, sink=0)
    if kind == "plan":
        c.update(T=1, ended=False, short=False)
    c.update(kw)
    return c


def listed():
    return [
        # one user's short conversation: the smallest call, latency counts
        _case("attn", name="q4_attn_b1_1k", B=1, ctx=1000, out="f32", gate="f32"),
        # four long documents, full attention: the cache's bytes
        _case("attn", name="q4_attn_b4_128k", B=4, ctx=131072, page=256, out="f32", gate="f32"),
        # a busy server with a window and sinks, every conversation of another length
        _case("attn", name="q4_window_b32", B=32, ctx=30001, ragged=True, window=4096, sink=4, page=32),
        # a drafter's tokens are verified
        _case("attn", name="q4_verify_b8_t6", B=8, ctx=20011, T=6, ragged=True),
        # continuous batching: chunks of several prompts and some decoding tokens in one call
        _case("attn", name="q4_chunks_b7", B=7, ctx=6000, T=701, ragged=True, window=2048, sink=16, page=128),
        # a long prompt through a window
        _case("attn", name="q4_window_prompt_8k", B=1, ctx=8192, T=8192, window=1024, sink=4),
        # one decode step of a small server
        _case("append", name="q4_append_b13", B=13, T=1, ctx=5000, dtype="f32"),
        # a prompt of two conversations
        _case("append", name="q4_append_prompt_4k", B=2, T=4096, ctx=4500, dtype="bf16"),
        # the last rows of a conversation, looked at
        _case("read", name="q4_read_77", rows=77, out="f32"),
        # a long conversation leaves the pool
        _case("read", name="q4_read_32k", rows=32768, out="bf16", page=128),
        # the next token of a small server
        _case("plan", name="plan_b13", B=13, ctx=5000),
        # a large server: prompts come in chunks, some conversations end
        _case("plan", name="plan_b2000_chunks", B=2000, T=500, ctx=9000, ended=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "window", "few", "prompt", "prompt", "append", "append", "read", "plan"])
    n_q, n_kv = rng.choice([(24, 4), (24, 4), (24, 4), (24, 4), (16, 1), (8, 8), (10, 2)])
    kw = {"n_q": n_q, "n_kv": n_kv, "page": rng.choice([32, 64, 128, 256])}
    rows = 524288 * 4 // max(4, n_kv)                          # (as many as the largest listed cache has)
    if kind == "plan":
        B = _log_int(rng, 1, 4096)
        return _case("plan", page=kw["page"], B=B, T=rng.choice([1, 1, _log_int(rng, 2, max(2, min(8192, 400000 // B)))]),
                     ctx=_log_int(rng, 30, 12000), ended=rng.random() < 0.5, short=rng.random() < 0.3)
    if kind == "read":
        return _case("read", **kw, rows=_log_int(rng, 1, 32768), out=rng.choice(["f32", "bf16"]))
    if kind == "append":
        B = _log_int(rng, 1, 64)
        T = rng.choice([1, rng.randint(2, 8), _log_int(rng, 9, max(9, 8192 // B))])
        return _case("append", **kw, B=B, T=T, ctx=T + rng.randint(0, 6000), dtype=rng.choice(["f32", "bf16"]))
    if kind == "attn":
        B = _log_int(rng, 1, 64)
        return _case("attn", **kw, B=B, ctx=_log_int(rng, 20, rows // max(B, 4)), ragged=rng.random() < 0.7,
                     out=rng.choice(["f32", "bf16"]), gate=rng.choice(["none", "f32", "bf16"]))
    if kind == "window":
        B = _log_int(rng, 1, 64)
        return _case("attn", **kw, B=B, ctx=_log_int(rng, 500, rows // max(B, 4)), ragged=True,
                     window=_log_int(rng, 60, 8192), sink=rng.choice([0, 1, 4, 70]), out=rng.choice(["f32", "bf16"]),
                     gate=rng.choice(["none", "f32", "bf16"]))
    if kind == "few":
        B, T = _log_int(rng, 1, 16), rng.randint(2, 24)
        return _case("attn", **kw, B=B, T=T, ctx=T + _log_int(rng, 200, rows // 4 // max(B, 8)), ragged=True,
                     window=rng.choice([0, 0, 2048]), sink=4, out=rng.choice(["f32", "bf16"]))
    B = rng.choice([1, 1, 2, 5])
    windowed = rng.random() < 0.7
    most = (8192 if windowed else 4096) // B                   # (as many operations as the listed prompt has)
    T = _log_int(rng, 9, most)
    return _case("attn", **kw, B=B, T=T, ctx=rng.choice([T, rng.randint(T, most)]), ragged=B > 1,
                 window=_log_int(rng, 60, min(4096, 8388608 // (B * T))) if windowed else 0, sink=rng.choice([0, 4, 70]),
                 gate=rng.choice(["none", "bf16"]))


def _lengths(case):
    """(rows, new tokens) of every sequence: from the case alone. The first sequence is always whole."""
    r = random.Random("%d %d %d" % (case["B"], case["ctx"], case["T"]))
    lens, new = [], []
    for b in range(case["B"]):
        n, t = case["ctx"], case["T"]
        if b and case.get("ragged", True):
            n = _log_int(r, max(1, n // 16), n)
            t = min(n, t if t <= 8 else max(1, int(t * r.random())))
            t = 1 if case["T"] > 8 and b % 3 == 2 else t         # (a decoding token among the prompts)
        lens.append(n)
        new.append(t)
    return lens, new


def _pages(case, n):
    return -(-n // case["page"])


# ------------------------------------------------------------------ inputs
class _Rand:
    """Device tensors from the seed alone, in call order."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(1000003 * int(seed) + 31)

    def normal(self, *shape, std=1.0, mean=0.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=self.g, device=DEV) * std + mean).to(dtype)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device=DEV)

    def pages(self, n_pages, n_kv, P, by_row):
        """Pages of rows as N(0, 1) values leave them: codes of a middle-heavy distribution, scales of a group's range,
        minima at its lower end."""
        shape = (n_pages, n_kv, P // 32)
        pg = torch.empty(*shape, BLOCK, device=DEV, dtype=torch.uint8)
        each = max(1, (1 << 27) // (4096 * n_kv * (P // 32)))
        for p in range(0, n_pages, each):
            n = min(each, n_pages - p)
            c = [torch.empty(n, *shape[1:], 4096, device=DEV, dtype=torch.float16).normal_(7.5, 3.2, generator=self.g)
                 .round_().clamp_(0, 15).to(torch.uint8) for _ in range(2)]
            pg[p:p + n, ..., :4096] = c[0] | (c[1] << 4)
        s = torch.exp(self.normal(*shape, 4, 32, std=0.12)) * 0.31
        m = -7.5 * s + self.normal(*shape, 4, 32, std=0.1)
        if by_row:
            m = m.transpose(-1, -2)
        pg[..., 4096:4352] = s.to(BF).reshape(*shape, 128).contiguous().view(torch.uint8)
        pg[..., 4352:] = m.to(BF).reshape(*shape, 128).contiguous().view(torch.uint8)
        return pg

    def table(self, counts, width):
        """A page table [B][width]: the sequences' pages are 0 .. sum(counts) - 1 in random order, the entries behind a
        sequence's last page 0."""
        pages = self.perm(sum(counts))
        t = torch.zeros(len(counts), width, device=DEV, dtype=torch.int32)
        at = torch.arange(width, device=DEV)[None] < torch.tensor(counts, device=DEV)[:, None]
        t[at] = pages.int()
        return t


def _dtype(name):
    return torch.float32 if name == "f32" else BF


def _i32(v):
    return torch.tensor(v, device=DEV, dtype=torch.int32)


def _prepare_plan(case, r):
    lens, new = _lengths(case)
    B = case["B"]
    counts = [_pages(case, n) for n in lens]
    more = [_pages(case, n + t) - c for n, t, c in zip(lens, new, counts)]
    held = sum(counts)
    free = sum(more) // 2 if case["short"] else sum(more) + 7
    s = {"case": case, "kind": "plan", "B": B, "page": case["page"], "n_tok": sum(new) + 3, "n_pages": held + free,
         "max_pages": max(c + m for c, m in zip(counts, more)) + 1}
    s["len"], s["new_tok"] = _i32(lens), _i32(new)
    s["ended"] = _i32([int(case["ended"] and b % 16 == 5) for b in range(B)])
    s["next_pos"] = s["len"] + 11
    s["table"] = r.table(counts, s["max_pages"])
    s["free_pages"] = torch.zeros(held + free, device=DEV, dtype=torch.int32)
    s["free_pages"][:free] = (r.perm(free) + held).int()
    s["n_free"] = _i32([free])
    for name, n in (("took", B), ("q_start", B + 1), ("len_out", B), ("next_pos_out", B), ("n_free_out", 1),
                    ("slot", s["n_tok"]), ("pos", s["n_tok"]), ("seq", s["n_tok"])):
        s[name] = torch.zeros(n, device=DEV, dtype=torch.int32)
    return s


def prepare(case, seed):
    r, kind = _Rand(seed), case["kind"]
    if kind == "plan":
        s = _prepare_plan(case, r)
    else:
        n_q, n_kv, P = case["n_q"], case["n_kv"], case["page"]
        s = {"case": case, "kind": kind, "n_q": n_q, "n_kv": n_kv, "page": P}
        lens, new = ([case["rows"]], [0]) if kind == "read" else _lengths(case)
        counts = [_pages(case, n) for n in lens]
        s["table"] = r.table(counts, max(counts))
        s["k"] = r.pages(sum(counts), n_kv, P, True)
        s["v"] = r.pages(sum(counts), n_kv, P, False)
        s["len"], s["B"], s["max_T"] = _i32(lens), len(lens), max(new)
        start = [0]
        for t in new:
            start.append(start[-1] + t)
        N = start[-1]
        s["q_start"], s["n_tok"] = _i32(start), N
        rows = torch.cat([torch.arange(n - t, n, device=DEV) for n, t in zip(lens, new)])
        owner = torch.repeat_interleave(torch.arange(len(lens), device=DEV), torch.tensor(new, device=DEV))
        if kind == "read":
            rows = torch.arange(case["rows"], device=DEV)
            owner = torch.zeros_like(rows)
        # slots, as the plan leaves them
        s["slot"] = (s["table"].long()[owner, rows // P] * P + rows % P).int()
        if kind == "append":
            dt = _dtype(case["dtype"])
            s["qg"] = r.normal(N, n_q, 2 * HD, dtype=dt)       # a q_proj row: q and gate interleaved by head
            s["kv"] = r.normal(N, 2, n_kv, HD, dtype=dt)
            s["q_norm_w"], s["k_norm_w"] = r.normal(HD, std=0.1), r.normal(HD, std=0.1)
            s["q_out"] = torch.empty(N, n_q, HD, device=DEV, dtype=BF)
            s["k_out"], s["v_out"] = (torch.empty(N, n_kv, HD, device=DEV) for _ in range(2))
        if kind == "read":
            s["k_out"], s["v_out"] = (torch.empty(case["rows"], n_kv, HD, device=DEV, dtype=_dtype(case["out"]))
                                      for _ in range(2))
        if kind == "attn":
            s["window"], s["sink"] = case["window"], case["sink"]
            s["q"] = r.normal(N, n_q, HD, std=2.0, dtype=BF)   # (scores of std 2: some rows weigh much more than others)
            s["gate"] = r.normal(N, n_q, HD, dtype=_dtype(case["gate"])) if case["gate"] != "none" else None
            s["out"] = torch.empty(N, n_q, HD, device=DEV, dtype=_dtype(case["out"]))
    if own:
        s["calls"] = _calls(s)
    return s


# ------------------------------------------------------ the framework's calls
_ctx = None


def _p(t):
    return t.data_ptr() if t is not None else None


def _code(t, L):
    return L.BF16 if t.dtype == BF else L.F32


def _calls(s):
    """(entry point, context, descriptor, check) of a state's calls, as a program keeps them from step to step."""
    global _ctx
    from vx27_amd import lib as L
    if _ctx is None:
        _ctx = L.Ctx(0)
    kind, lib = s["kind"], L.lib()
    if kind == "plan":
        d = L.PagedPlanDesc()
        d.B, d.page_size, d.n_pages, d.max_pages, d.n_tok = s["B"], s["page"], s["n_pages"], s["max_pages"], s["n_tok"]
        for name in ("new_tok", "ended", "len", "next_pos", "table", "free_pages", "n_free", "took", "q_start", "len_out",
                     "next_pos_out", "n_free_out", "slot", "pos", "seq"):
            setattr(d, name, _p(s[name]))
        return [(lib.vx27_hip_paged_plan, _ctx.h, d, L.check)]
    calls = []
    if kind != "read":
        d = L.PagedAppendDesc() if kind == "append" else L.PagedAttnDesc()
        d.B, d.n_q, d.n_kv, d.hd, d.page_size = s["B"], s["n_q"], s["n_kv"], HD, s["page"]
        d.n_pages, d.max_pages = s["k"].shape[0], s["table"].shape[1]
        d.table, d.len, d.k_pages, d.v_pages = _p(s["table"]), _p(s["len"]), _p(s["k"]), _p(s["v"])
        d.q_start, d.n_tok, d.max_T = _p(s["q_start"]), s["n_tok"], s["max_T"]
    if kind == "append":
        d.rope_dim, d.rope_theta, d.rope_yarn, d.in_dtype = ROPE, THETA, 1.0, _code(s["qg"], L)
        d.q, d.q_tok_stride, d.q_head_stride = _p(s["qg"]), s["qg"].stride(0), s["qg"].stride(1)
        d.k_new, d.v_new, d.kv_tok_stride = _p(s["kv"]), _p(s["kv"][0, 1]), s["kv"].stride(0)
        d.q_norm_w, d.k_norm_w, d.q_out = _p(s["q_norm_w"]), _p(s["k_norm_w"]), _p(s["q_out"])
        calls.append((lib.vx27_hip_paged_append_q4, _ctx.h, d, L.check))
    if kind == "attn":
        d.window, d.n_sink = s["window"], s["sink"]
        d.q, d.q_tok_stride, d.q_head_stride = _p(s["q"]), s["q"].stride(0), s["q"].stride(1)
        if s["gate"] is not None:
            d.gate, d.gate_dtype = _p(s["gate"]), _code(s["gate"], L)
            d.gate_tok_stride, d.gate_head_stride = s["gate"].stride(0), s["gate"].stride(1)
        d.out, d.out_dtype = _p(s["out"]), _code(s["out"], L)
        return [(lib.vx27_hip_paged_attn_q4, _ctx.h, d, L.check)]
    # what the pages hold now: the values of the slots
    d = L.PagedReadDesc()
    d.n_kv, d.hd, d.page_size, d.n_pages, d.n_rows = s["n_kv"], HD, s["page"], s["k"].shape[0], s["slot"].numel()
    d.slots, d.k_pages, d.v_pages = _p(s["slot"]), _p(s["k"]), _p(s["v"])
    d.k_out, d.v_out, d.out_dtype = _p(s["k_out"]), _p(s["v_out"]), _code(s["k_out"], L)
    calls.append((lib.vx27_hip_paged_read_q4, _ctx.h, d, L.check))
    return calls


PLANNED = ("took", "q_start", "len_out", "next_pos_out", "n_free_out", "slot", "pos", "seq", "table", "free_pages")


def run(s):
    kind = s["kind"]
    if own:
        for fn, h, d, check in s["calls"]:
            check(fn(h, C.byref(d)), kind)
    else:
        {"append": _append, "attn": _attn, "read": _read, "plan": _plan}[kind](s)
    if kind == "plan":
        return {name: s[name] for name in PLANNED}
    if kind == "attn":
        return {"out": s["out"]}
    out = {"k": s["k_out"], "v": s["v_out"]}                   # the values that the pages hold for the call's rows
    if kind == "append":
        out["q"] = s["q_out"]
    return out


# ------------------------------------------------------------ the plain form
def _scales(blk, by_row):
    lead = blk.shape[:-1]
    s = blk[..., 4096:4352].contiguous().view(BF).view(*lead, 4, 32).transpose(-1, -2)
    m = blk[..., 4352:].contiguous().view(BF)
    m = m.view(*lead, 32, 4) if by_row else m.view(*lead, 4, 32).transpose(-1, -2)
    return s, m                                                # [..., row, group]


def _codes(blk, by_row):
    """[..., 32 rows, 256 dims] codes of blocks [..., 4608]: K's if by_row, else V's."""
    lead, n = blk.shape[:-1], blk.dim() - 1
    b = blk[..., :4096]
    c = torch.stack((b & 15, b >> 4), dim=-1)                  # [..., 4096, half]
    if by_row:
        c = c.view(*lead, 2, 2, 4, 4, 4, 4, 4, 2)              # row/4%2, dim/128, dim/8%4, row/8, row%4, dim/32%4, dim%4, half
        order = (3, 0, 4, 1, 5, 2, 7, 6)
    else:
        c = c.view(*lead, 4, 4, 16, 4, 4, 2)                   # dim/64, row/8, dim%16, dim/16%4, row%4, half
        order = (1, 5, 4, 0, 3, 2)
    return c.permute(*range(n), *(n + i for i in order)).reshape(*lead, 32, HD)


def _packed(c, by_row):
    """The code bytes of [..., 32 rows, 256 dims]."""
    lead, n = c.shape[:-2], c.dim() - 2
    if by_row:
        c = c.view(*lead, 4, 2, 4, 2, 4, 4, 2, 4)              # row/8, row/4%2, row%4, dim/128, dim/32%4, dim/8%4, half, dim%4
        order = (1, 3, 5, 0, 2, 4, 7, 6)
    else:
        c = c.view(*lead, 4, 2, 4, 4, 4, 16)                   # row/8, half, row%4, dim/64, dim/16%4, dim%16
        order = (3, 0, 5, 4, 2, 1)
    c = c.permute(*range(n), *(n + i for i in order)).reshape(*lead, 4096, 2)
    return c[..., 0] | (c[..., 1] << 4)


def _values(blk, by_row):
    s, m = _scales(blk, by_row)
    c = _codes(blk, by_row).float().unflatten(-1, (4, 64))
    return c.mul_(s.float()[..., None]).add_(m.float()[..., None]).flatten(-2)


def _rows(s, pages, by_row):
    """The cached rows of every sequence in 32 bits, [B][n_kv][rows][256]."""
    t = s["table"].long()
    x = _values(pages[t], by_row)                              # [B][pages][n_kv][P/32][32][256]
    return x.permute(0, 2, 1, 3, 4, 5).reshape(s["B"], s["n_kv"], -1, HD)


def _owner(s):
    """(sequence, number within it) of every token."""
    n = torch.arange(s["n_tok"], device=DEV)
    b = torch.searchsorted(s["q_start"].long(), n, right=True) - 1
    return b, n - s["q_start"].long()[b]


def _attn(s):
    B, T, n_kv, grp = s["B"], s["max_T"], s["n_kv"], s["n_q"] // s["n_kv"]
    ob, ot = _owner(s)
    new = s["q_start"].diff().long()
    q = torch.zeros(B, T, n_kv, grp, HD, device=DEV)
    q[ob, ot] = s["q"].view(-1, n_kv, grp, HD).float()
    k = _rows(s, s["k"], True)
    sc = (q.permute(0, 2, 3, 1, 4).reshape(B, n_kv, grp * T, HD) @ k.transpose(2, 3)) / 16.0
    del k
    t, j = torch.arange(T, device=DEV), torch.arange(sc.shape[3], device=DEV)
    i = (s["len"].long() - new)[:, None, None] + t[None, :, None]                     # the tokens' rows
    seen = (j <= i) & (t[None, :, None] < new[:, None, None])
    if s["window"]:
        seen &= (j > i - s["window"]) | (j < s["sink"])
    sc = sc.view(B, n_kv, grp, T, -1).masked_fill_(~seen[:, None, None], -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = sc.sub_(torch.where(m > -math.inf, m, torch.zeros_like(m))).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_min(1e-30))
    v = _rows(s, s["v"], False)
    o = (p.view(B, n_kv, grp * T, -1) @ v).view(B, n_kv, grp, T, HD)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, T, s["n_q"], HD)[ob, ot]
    if s["gate"] is not None:
        o = o * torch.sigmoid(s["gate"].float())
    s["out"].copy_(o)


def _angles(pos):
    """cos and sin of every token's angles. The angle is the framework's: the position (32 bits) times the frequency
    (32 bits), rounded to 32 bits; its cosine and sine are taken in 64."""
    e = torch.arange(ROPE // 2, dtype=torch.float32) * -2.0 / ROPE
    f = (torch.tensor(THETA, dtype=DBL) ** e.double()).float().to(DEV)
    a = (pos.float()[:, None] * f).double()
    return a.cos()[:, None], a.sin()[:, None]


def _norm_rope(x, w, cs, sn):
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1 + w)
    a, b, h = x[..., :ROPE // 2], x[..., ROPE // 2:ROPE], x[..., ROPE:]
    return torch.cat((a * cs - b * sn, a * sn + b * cs, h), -1)


def _toward(x, up):
    """bf16 at or beyond x (64 bits): the largest not above it, or with `up` the smallest not below it."""
    y = x.to(BF)
    off = (y.double() < x) if up else (y.double() > x)
    return torch.where(off, torch.nextafter(y, torch.full_like(y, math.inf if up else -math.inf)), y)


def _quantised(x):
    """(codes, s, m) of rows [..., 256] in 64 bits (a value next to a border would get another code in 32)."""
    g = x.unflatten(-1, (4, 64))
    m = _toward(g.amin(-1), False)
    s = _toward((g.amax(-1) - m.double()) / 15, True)
    d = s.double()[..., None]
    c = torch.where(d > 0, (g - m.double()[..., None]) / torch.where(d > 0, d, torch.ones_like(d)), torch.zeros_like(d))
    return c.round().to(torch.uint8).flatten(-2), s, m


def _place(s, pages, rows, by_row):
    """Rows [N][n_kv][256] into their slots."""
    c, sc, mn = _quantised(rows)
    n_kv, P = s["n_kv"], s["page"]
    slot = s["slot"].long()
    blocks, which = torch.unique(slot // 32, return_inverse=True)
    page, blk = blocks // (P // 32), blocks % (P // 32)
    old = pages[page, :, blk]                                  # [blocks][n_kv][4608]
    codes, (ps, pm) = _codes(old, by_row), (t.clone() for t in _scales(old, by_row))
    at = slot % 32
    codes[which, :, at], ps[which, :, at], pm[which, :, at] = c, sc, mn
    old[..., :4096] = _packed(codes, by_row)
    lead = old.shape[:2]
    old[..., 4096:4352] = ps.transpose(-1, -2).contiguous().view(*lead, 128).view(torch.uint8)
    pm = pm if by_row else pm.transpose(-1, -2)
    old[..., 4352:] = pm.contiguous().view(*lead, 128).view(torch.uint8)
    pages[page, :, blk] = old


def _append(s):
    ob, ot = _owner(s)
    row = (s["len"].long() - s["q_start"].diff().long())[ob] + ot
    cs, sn = _angles(row)
    s["q_out"].copy_(_norm_rope(s["qg"][..., :HD].float(), s["q_norm_w"], cs.float(), sn.float()))
    _place(s, s["k"], _norm_rope(s["kv"][:, 0].double(), s["k_norm_w"].double(), cs, sn), True)
    _place(s, s["v"], s["kv"][:, 1].double(), False)
    _read(s)


def _read(s):
    slot, P = s["slot"].long(), s["page"]
    for pages, out, by_row in ((s["k"], s["k_out"], True), (s["v"], s["v_out"], False)):
        for i in range(0, slot.numel(), 4096):
            a = slot[i:i + 4096]
            blocks, which = torch.unique(a // 32, return_inverse=True)
            x = _values(pages[blocks // (P // 32), :, blocks % (P // 32)], by_row)
            out[i:i + 4096] = x[which, :, a % 32].to(out.dtype)


def _plan(s):
    P, n_tok, B = s["page"], s["n_tok"], s["B"]
    ceil = lambda n: (n + P - 1) // P  # noqa: E731
    ended, length, new = s["ended"] != 0, s["len"].long(), s["new_tok"].long()
    held = ceil(length)
    width = torch.arange(s["max_pages"], device=DEV)
    back = s["table"][ended[:, None] & (width < held[:, None])]                       # released pages, in order
    free = s["n_free"].long()
    stack = torch.cat((s["free_pages"], s["free_pages"].new_zeros(s["n_pages"])))
    stack[free + torch.arange(back.numel(), device=DEV)] = back
    total = free + back.numel()
    length = torch.where(ended, 0, length)
    held = torch.where(ended, 0, held)
    new = torch.where(ended, 0, new)
    fits = length + new <= s["max_pages"] * P
    need = torch.where(fits, ceil(length + new) - held, 0)
    new = torch.where(fits & ((need == 0) | (need.cumsum(0) <= total)), new, 0)
    new = torch.where(new.cumsum(0) <= n_tok, new, 0)
    need = torch.where(new > 0, need, 0)
    end = new.cumsum(0)
    s["took"].copy_(new)
    s["q_start"].copy_(torch.cat((end.new_zeros(1), end)))
    s["len_out"].copy_(length + new)
    s["next_pos_out"].copy_(torch.where(ended, 0, s["next_pos"].long()) + new)
    s["n_free_out"].copy_(total - need.sum())
    # pages from the top of the stack, in the order of the sequences and their rows
    b = torch.repeat_interleave(torch.arange(B, device=DEV), need)
    k = torch.arange(b.numel(), device=DEV)
    within = k - (need.cumsum(0) - need)[b]
    s["table"][b, held[b] + within] = stack[total - 1 - k]
    put = torch.arange(s["n_pages"], device=DEV)
    s["free_pages"].copy_(torch.where((put >= free) & (put < s["n_free_out"]), stack[:s["n_pages"]], s["free_pages"]))
    b = torch.repeat_interleave(torch.arange(B, device=DEV), new)
    t = torch.arange(b.numel(), device=DEV) - (end - new)[b]
    row = length[b] + t
    for name, x in (("slot", s["table"].long()[b, row // P] * P + row % P),
                    ("pos", torch.where(ended, 0, s["next_pos"].long())[b] + t), ("seq", b)):
        s[name].fill_(-1)
        s[name][:b.numel()] = x.int()


# --------------------------------------------------------------------- work
def _seen(case, i):
    """How many rows the token at row i sees."""
    if i < 0:
        return 0
    if not case["window"]:
        return i + 1
    lo = max(0, i - case["window"] + 1)
    return i + 1 - lo + min(case["sink"], lo)


def work(case):
    n_q, n_kv, kind = case["n_q"], case["n_kv"], case["kind"]
    row = n_kv * 2 * BLOCK // 32                               # (K and V of a row)
    if kind == "read":
        e = 4 if case["out"] == "f32" else 2
        return {"bytes": case["rows"] * (row + 4 + n_kv * HD * 2 * e), "flops": case["rows"] * n_kv * HD * 4}
    lens, new = _lengths(case)
    N = sum(new)
    if kind == "plan":
        pages = sum(_pages(case, n + t) - _pages(case, n) for n, t in zip(lens, new))
        return {"bytes": case["B"] * 4 * 8 + N * 12 + pages * 8, "flops": 0}
    if kind == "append":
        e = 4 if case["dtype"] == "f32" else 2
        values = N * (row + n_kv * HD * 2 * 4)                 # (read back)
        return {"bytes": N * ((n_q + 2 * n_kv) * HD * e + n_q * HD * 2 + row) + values, "flops": N * (n_q + n_kv) * HD * 6}
    b, f = 0, 0
    for n, t in zip(lens, new):
        first, last = n - t, n - 1
        # rows that any of the tokens sees
        rows = n
        if case["window"]:
            lo = max(0, first - case["window"] + 1)
            rows = last + 1 - lo + min(case["sink"], lo)
        b += rows * row
        f += sum(_seen(case, i) for i in range(first, n)) * n_q * HD * 4
    out = 4 if case["out"] == "f32" else 2
    gate = {"none": 0, "f32": 4, "bf16": 2}[case["gate"]]
    return {"bytes": b + N * n_q * HD * (2 + out + gate), "flops": f}


# ------------------------------------------------------------ in 64 bits
def _where(by_row):
    """Byte and shift of the code of (row, dim), byte offsets of its s and m: [32][256] each, from the format."""
    r, d = torch.arange(32, device=DEV)[:, None], torch.arange(HD, device=DEV)[None]
    if by_row:
        byte = r // 4 % 2 * 2048 + d // 128 * 1024 + d // 8 % 4 * 256 + r // 8 * 64 + r % 4 * 16 + d // 32 % 4 * 4 + d % 4
        return byte, d // 4 % 2 * 4 + 0 * r, 4096 + d // 64 * 64 + r * 2, 4352 + r * 8 + d // 64 * 2
    byte = d // 64 * 1024 + r // 8 * 256 + d % 16 * 16 + d // 16 % 4 * 4 + r % 4
    return byte, r // 4 % 2 * 4 + 0 * d, 4096 + d // 64 * 64 + r * 2, 4352 + d // 64 * 64 + r * 2


def _bf16_at(blk, at):
    """The bf16 numbers at byte offsets `at` of blocks [n][4608], in 64 bits."""
    bits = blk[:, at].int() | (blk[:, at + 1].int() << 8)
    return (bits << 16).view(torch.float32).double()


def _decoded(blk, by_row):
    """[n][4608] -> [n][32][256] in 64 bits."""
    byte, shift, s_at, m_at = _where(by_row)
    c = ((blk[:, byte] >> shift.to(torch.uint8)) & 15).double()
    return c.mul_(_bf16_at(blk, s_at)).add_(_bf16_at(blk, m_at))


def _held(x):
    """What rows [..., 256] in 64 bits become when held in 4 bits."""
    out = torch.empty_like(x)
    for g in range(0, HD, 64):
        v = x[..., g:g + 64]
        lo, hi = v.min(-1, keepdim=True).values, v.max(-1, keepdim=True).values

        def bf(x, up):
            """Truncated bits of the nearest 32-bit number, then a step where that is on the wrong side."""
            b = x.float().view(torch.int32) & -65536
            for _ in range(2):
                y = b.view(torch.float32).double()
                wrong = y < x if up else y > x
                away = ((b < 0) ^ up)                          # a larger magnitude is the way to go
                zero = (b & 0x7fffffff) == 0
                step = torch.where(away | zero, b + 65536, b - 65536)
                step = torch.where(zero, torch.full_like(b, 65536 if up else -2147483648 + 65536), step)
                b = torch.where(wrong, step, b)
            return b.view(torch.float32).double()

        m = bf(lo, False)
        s = bf((hi - m) / 15, True)
        t = (v - m) / torch.where(s > 0, s, torch.ones_like(s))
        c = torch.floor(t)
        r = t - c
        c += (r > 0.5) | ((r == 0.5) & (c % 2 == 1))
        out[..., g:g + 64] = torch.where(s > 0, m + s * c, m.expand_as(v))
    return out


def exact(case, seed):
    """From the definitions, sequence by sequence and head by head, in 64 bits."""
    s = prepare(case, seed)
    n_kv, grp, P, kind = case["n_kv"], case["n_q"] // case["n_kv"], case["page"], case["kind"]
    if kind == "plan":
        return _exact_plan(s)
    if kind == "read":
        out = {}
        for name, by_row in (("k", True), ("v", False)):
            x = torch.empty(case["rows"], n_kv, HD, device=DEV, dtype=DBL)
            for p in range(0, s["table"].shape[1], 64):
                pages = s["table"][0, p:p + 64].long()
                for h in range(n_kv):
                    y = _decoded(s[name][pages, h].reshape(-1, BLOCK), by_row).reshape(-1, HD)
                    n = min(len(y), case["rows"] - p * P)
                    x[p * P:p * P + n, h] = y[:n]
            out[name] = x
        return out
    lens, new = _lengths(case)
    if kind == "append":
        e = [THETA ** (-2.0 * i / ROPE) for i in range(ROPE // 2)]
        freq = torch.tensor(e, device=DEV, dtype=torch.float32)
        rows = torch.cat([torch.arange(n - t, n, device=DEV) for n, t in zip(lens, new)])
        ang = (rows.to(torch.float32)[:, None] * freq).double()[:, None, :]
        turn = torch.complex(ang.cos(), ang.sin())

        def rotated(x, w):
            x = x.double()
            x = x / torch.sqrt((x * x).sum(-1, keepdim=True) / HD + EPS) * (w.double() + 1)
            z = torch.complex(x[..., :ROPE // 2], x[..., ROPE // 2:ROPE]) * turn
            return torch.cat((z.real, z.imag, x[..., ROPE:]), -1)

        return {"k": _held(rotated(s["kv"][:, 0], s["k_norm_w"])), "v": _held(s["kv"][:, 1].double()),
                "q": rotated(s["qg"][:, :, :HD], s["q_norm_w"])}
    out = torch.zeros(s["n_tok"], case["n_q"], HD, device=DEV, dtype=DBL)
    at = 0
    for b, (n, t) in enumerate(zip(lens, new)):
        pages = s["table"][b, :_pages(case, n)].long()
        rows = torch.arange(n, device=DEV)
        for h in range(n_kv):
            k = _decoded(s["k"][pages, h].reshape(-1, BLOCK), True).reshape(-1, HD)[:n]
            v = _decoded(s["v"][pages, h].reshape(-1, BLOCK), False).reshape(-1, HD)[:n]
            for c in range(at, at + t, 512):                   # 512 tokens at a time
                m = min(512, at + t - c)
                i = (n - t + c - at + torch.arange(m, device=DEV))[:, None]
                seen = rows <= i
                if case["window"]:
                    seen = seen & ((i - rows < case["window"]) | (rows < case["sink"]))
                for g in range(h * grp, (h + 1) * grp):
                    x = s["q"][c:c + m, g].double() @ k.t() * (HD ** -0.5)
                    out[c:c + m, g] = torch.softmax(torch.where(seen, x, torch.full_like(x, -math.inf)), 1) @ v
        at += t
    if s["gate"] is not None:
        out /= 1 + torch.exp(-s["gate"].double())
    return {"out": out}


def _exact_plan(s):
    """One sequence after the other, on the host."""
    P, cap = s["page"], s["max_pages"] * s["page"]
    x = {name: s[name].tolist() for name in (*PLANNED, "len", "new_tok", "ended", "next_pos", "n_free")}
    free, n_free, B = x["free_pages"], x["n_free"][0], s["B"]
    stack = free[:n_free]
    for b in range(B):
        if x["ended"][b]:
            stack += x["table"][b][:-(-x["len"][b] // P)]
            x["len"][b] = x["next_pos"][b] = x["new_tok"][b] = 0
    total = len(stack)
    wanted = tokens = 0
    x["slot"], x["pos"], x["seq"] = [], [], []
    for b in range(B):
        n, t = x["len"][b], x["new_tok"][b]
        need = -(-(n + t) // P) - -(-n // P)
        if n + t > cap:
            t = 0
        else:
            wanted += need
            if need and wanted > total:
                t = 0
        tokens += t
        if tokens > s["n_tok"]:
            t = 0
        if t:
            for i in range(need):
                x["table"][b][-(-n // P) + i] = stack.pop()
        x["took"][b], x["len_out"][b], x["next_pos_out"][b] = t, n + t, x["next_pos"][b] + t
        x["q_start"][b + 1] = x["q_start"][b] + t
        for r in range(n, n + t):
            x["slot"].append(x["table"][b][r // P] * P + r % P)
            x["pos"].append(x["next_pos"][b] + r - n)
            x["seq"].append(b)
    x["n_free_out"][0] = len(stack)
    free[n_free:max(n_free, len(stack))] = stack[n_free:]
    for name in ("slot", "pos", "seq"):
        x[name] += [-1] * (s["n_tok"] - len(x[name]))
    return {name: _i32(x[name]) for name in PLANNED}
