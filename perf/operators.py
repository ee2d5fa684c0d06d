"""The paged-cache operators that a serving program calls, as timed cases.

A server of many conversations keeps their key-value rows in pages and, per
GQA layer and step,

  append   norms and rotates the new tokens' queries and keys and writes keys
           and values into the pages (vx27_hip_paged_append)
  attn     attends from the new tokens to the cached rows: all of them, or a
           sliding window and the first few rows (sinks); where it means to
           evict later, it has the call add every row's attention weights up
           (vx27_hip_paged_attn)
  evict    keeps the sinks, the recent rows and the heaviest of the others and
           lays them out in fresh pages (vx27_hip_paged_evict)

The heads are those of the Qwen 27B hybrid's attention layers (24 query and 4
KV heads of 256, RoPE over 64 dimensions); draws take other groupings too.

Pages: K [n_pages][n_kv][P][256], V [n_pages][n_kv][P/32][256][32], bf16; row r
of sequence b is row r % P of page table[b][r // P].
"""
from __future__ import annotations

import ctypes as C
import math
import random

import torch

own = False

HD = 256                       # head dim
ROPE, THETA, EPS = 64, 1e7, 1e-6
DEV = "cuda"
BF = torch.bfloat16


# ------------------------------------------------------------------- cases
def _case(kind, **kw):
    c = {"kind": kind, "n_q": 24, "n_kv": 4, "page": 64, "window": 0, "sink": 0}
    if kind == "attn":
        c.update(T=1, ragged=False, out="bf16", gate="bf16", acc=False)
    c.update(kw)
    return c


def listed():
    return [
        # one user's short conversation: the smallest call, latency counts
        _case("attn", name="attn_b1_1k", B=1, ctx=1000, out="f32", gate="f32"),
        # four long documents, full attention: the cache's bytes
        _case("attn", name="attn_b4_128k", B=4, ctx=131072, page=256, out="f32", gate="f32"),
        # a busy server: an odd batch, every conversation of another length
        _case("attn", name="attn_b61_ragged", B=61, ctx=16000, ragged=True),
        # the same with a window and sinks: what is read no longer grows with the conversation
        _case("attn", name="window_b32", B=32, ctx=30001, ragged=True, window=4096, sink=4, page=32),
        # a long prompt through a window
        _case("attn", name="window_prompt_8k", B=1, ctx=8192, T=8192, window=1024, sink=4),
        # continuous batching: chunks of several prompts and some decoding tokens in one call
        _case("attn", name="window_chunks_b7", B=7, ctx=6000, T=701, ragged=True, window=2048, sink=16, page=128),
        # decoding under an eviction budget: the weights are added up
        _case("attn", name="weights_b16_8k", B=16, ctx=8190, ragged=True, acc=True),
        # the last tokens of a prompt weigh its rows before the first eviction
        _case("attn", name="weights_window_t64", B=4, ctx=9000, T=64, acc=True),
        # one conversation over its budget
        _case("evict", name="evict_b1_1k", B=1, ctx=1030, budget=512, sink=4, recent=64, ragged=False),
        # a batch of long ones
        _case("evict", name="evict_b8_32k", B=8, ctx=32768, budget=8192, sink=4, recent=1024, page=128, ragged=True),
        # one decode step of a small server
        _case("append", name="append_b13", B=13, T=1, ctx=5000, dtype="f32", ragged=True),
        # a prompt of two conversations
        _case("append", name="append_prompt_4k", B=2, T=4096, ctx=4500, dtype="bf16", ragged=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "window", "prompt", "prompt", "weights", "evict", "append"])
    n_q, n_kv = rng.choice([(24, 4), (24, 4), (24, 4), (24, 4), (16, 1), (8, 8), (10, 2)])
    kw = {"n_q": n_q, "n_kv": n_kv, "page": rng.choice([32, 64, 128, 256])}
    rows = 524288 * 4 // max(4, n_kv)                          # (K and V of them: 2.1 GB at most)
    if kind == "evict":
        B = _log_int(rng, 1, 16)
        ctx = _log_int(rng, 200, rows // 2 // max(B, 8))
        budget = rng.randint(max(40, ctx // 8), ctx)
        sink = rng.choice([0, 1, 4, 16])
        return _case("evict", **kw, B=B, ctx=ctx, budget=budget, sink=sink, recent=rng.randint(0, budget - sink),
                     ragged=True)
    if kind == "append":
        B = _log_int(rng, 1, 64)
        T = rng.choice([1, rng.randint(2, 8), _log_int(rng, 9, max(9, 8192 // B))])
        return _case("append", **kw, B=B, T=T, ctx=T + rng.randint(0, 6000), dtype=rng.choice(["f32", "bf16"]),
                     ragged=True)
    if kind == "attn":
        B = _log_int(rng, 1, 64)
        return _case("attn", **kw, B=B, ctx=_log_int(rng, 20, rows // max(B, 4)), ragged=rng.random() < 0.7,
                     out=rng.choice(["f32", "bf16"]), gate=rng.choice(["none", "f32", "bf16"]))
    if kind == "window":
        B = _log_int(rng, 1, 64)
        return _case("attn", **kw, B=B, ctx=_log_int(rng, 500, rows // max(B, 4)), ragged=True,
                     window=_log_int(rng, 60, 8192), sink=rng.choice([0, 1, 4, 70]), out=rng.choice(["f32", "bf16"]),
                     gate=rng.choice(["none", "f32", "bf16"]))
    if kind == "weights":
        B = _log_int(rng, 1, 16)
        T = rng.choice([1, 1, rng.randint(2, 64)])
        return _case("attn", **kw, B=B, T=T, ctx=T + _log_int(rng, 200, rows // 4 // max(B, 8)), ragged=True, acc=True,
                     window=rng.choice([0, 0, 2048]), sink=4)
    B = rng.choice([1, 1, 2, 5])
    windowed = rng.random() < 0.7
    most = (8192 if windowed else 4096) // B                   # (as many operations as the listed prompt has)
    T = _log_int(rng, 2, most)
    return _case("attn", **kw, B=B, T=T, ctx=rng.choice([T, rng.randint(T, most)]), ragged=B > 1,
                 window=_log_int(rng, 60, min(4096, 8388608 // (B * T))) if windowed else 0, sink=rng.choice([0, 4, 70]),
                 gate=rng.choice(["none", "bf16"]))


def _plan(case):
    """(rows, new tokens) of every sequence: from the case alone. The first sequence is always whole."""
    r = random.Random("%d %d %d" % (case["B"], case["ctx"], case.get("T", 0)))
    lens, new = [], []
    for b in range(case["B"]):
        n, t = case["ctx"], case.get("T", 1)
        if case["ragged"] and b:
            n = _log_int(r, max(1, n // 16), n)
            t = min(n, t if t <= 8 else max(1, int(t * r.random())))
            t = 1 if case.get("T", 1) > 8 and b % 3 == 2 else t      # (a decoding token among the prompts)
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
        self.g.manual_seed(1000003 * int(seed) + 29)

    def normal(self, *shape, std=1.0, mean=0.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=self.g, device=DEV) * std + mean).to(dtype)

    def bf16(self, *shape):
        """N(0, 1) in bf16, made in place (for large caches)."""
        return torch.empty(*shape, device=DEV, dtype=BF).normal_(generator=self.g)

    def table(self, counts, width, lo=0):
        """A page table [B][width]: the sequences' pages are lo .. lo + sum(counts) - 1 in random order, the entries
        behind a sequence's last page 0."""
        perm = torch.randperm(sum(counts), generator=self.g, device=DEV) + lo
        t = torch.zeros(len(counts), width, device=DEV, dtype=torch.int32)
        at = torch.arange(width, device=DEV)[None] < torch.tensor(counts, device=DEV)[:, None]
        t[at] = perm.int()
        return t


def _dtype(name):
    return torch.float32 if name == "f32" else BF


def _i32(v):
    return torch.tensor(v, device=DEV, dtype=torch.int32)


def prepare(case, seed):
    r, kind = _Rand(seed), case["kind"]
    lens, new = _plan(case)
    B, n_q, n_kv, P = case["B"], case["n_q"], case["n_kv"], case["page"]
    counts = [_pages(case, n) for n in lens]
    n_pages, width = sum(counts), max(counts)
    s = {"case": case, "kind": kind, "len": _i32(lens), "max_T": max(new), "B": B, "n_q": n_q, "n_kv": n_kv, "page": P,
         "window": case["window"], "sink": case["sink"]}
    s["table"] = r.table(counts, width)
    if kind == "evict":
        kept = [_pages(case, min(n, case["budget"])) for n in lens]
        s["dst_table"] = r.table(kept, max(kept), lo=n_pages)
        n_pages += sum(kept)
        # what decoding leaves: a few heavy rows, many light ones, some that no token ever weighed
        acc = torch.exp(r.normal(B, n_kv, width * P, std=2.0))
        s["acc"] = torch.where(r.normal(B, n_kv, width * P) < -1.5, torch.zeros_like(acc), acc)
        s["acc_out"] = torch.zeros(B, n_kv, case["budget"], device=DEV)
        s["kept"] = torch.full((B, n_kv, case["budget"]), -1, device=DEV, dtype=torch.int32)
        s["len_out"] = torch.zeros(B, device=DEV, dtype=torch.int32)
        s["budget"], s["recent"] = case["budget"], case["recent"]
    s["k"] = r.bf16(n_pages, n_kv, P, HD)
    s["v"] = r.bf16(n_pages, n_kv, P // 32, HD, 32)
    if kind != "evict":
        start = [0]
        for t in new:
            start.append(start[-1] + t)
        N = start[-1]
        s["q_start"], s["n_tok"] = _i32(start), N
    if kind == "append":
        dt = _dtype(case["dtype"])
        s["qg"] = r.normal(N, n_q, 2 * HD, dtype=dt)           # a q_proj row: q and gate interleaved by head
        s["kv"] = r.normal(N, 2, n_kv, HD, dtype=dt)
        s["q_norm_w"], s["k_norm_w"] = r.normal(HD, std=0.1), r.normal(HD, std=0.1)
        s["q_out"] = torch.empty(N, n_q, HD, device=DEV, dtype=BF)
    if kind == "attn":
        s["q"] = r.normal(N, n_q, HD, std=2.0, dtype=BF)       # (scores of std 2: some rows weigh much more than others)
        s["gate"] = r.normal(N, n_q, HD, dtype=_dtype(case["gate"])) if case["gate"] != "none" else None
        s["out"] = torch.empty(N, n_q, HD, device=DEV, dtype=_dtype(case["out"]))
        s["acc"] = torch.exp(r.normal(B, n_kv, width * P)) if case["acc"] else None
    if own:
        s["call"] = _call(s)
    return s


# ------------------------------------------------------ the framework's calls
_ctx = None


def _p(t):
    return t.data_ptr() if t is not None else None


def _call(s):
    """(entry point, context, descriptor) of a state's call, as a program keeps them from step to step."""
    global _ctx
    from vx27_amd import lib as L
    if _ctx is None:
        _ctx = L.Ctx(0)
    code = lambda t: L.BF16 if t is not None and t.dtype == BF else L.F32  # noqa: E731
    kind, lib = s["kind"], L.lib()
    d = {"append": L.PagedAppendDesc, "attn": L.PagedAttnDesc, "evict": L.PagedEvictDesc}[kind]()
    d.B, d.n_kv, d.hd, d.page_size = s["B"], s["n_kv"], HD, s["page"]
    d.n_pages, d.max_pages = s["k"].shape[0], s["table"].shape[1]
    d.table, d.len, d.k_pages, d.v_pages = _p(s["table"]), _p(s["len"]), _p(s["k"]), _p(s["v"])
    if kind == "evict":
        d.budget, d.n_sink, d.n_recent = s["budget"], s["sink"], s["recent"]
        d.acc, d.acc_stride, d.acc_out, d.acc_out_stride = _p(s["acc"]), s["acc"].shape[2], _p(s["acc_out"]), s["budget"]
        d.dst_table, d.dst_max_pages = _p(s["dst_table"]), s["dst_table"].shape[1]
        d.dst_len, d.kept = _p(s["len_out"]), _p(s["kept"])
        return lib.vx27_hip_paged_evict, _ctx.h, d, L.check
    d.n_q, d.q_start, d.n_tok, d.max_T = s["n_q"], _p(s["q_start"]), s["n_tok"], s["max_T"]
    if kind == "append":
        d.rope_dim, d.rope_theta, d.rope_yarn, d.in_dtype = ROPE, THETA, 1.0, code(s["qg"])
        d.q, d.q_tok_stride, d.q_head_stride = _p(s["qg"]), s["qg"].stride(0), s["qg"].stride(1)
        d.k_new, d.v_new, d.kv_tok_stride = _p(s["kv"]), _p(s["kv"][0, 1]), s["kv"].stride(0)
        d.q_norm_w, d.k_norm_w, d.q_out = _p(s["q_norm_w"]), _p(s["k_norm_w"]), _p(s["q_out"])
        return lib.vx27_hip_paged_append, _ctx.h, d, L.check
    d.window, d.n_sink = s["window"], s["sink"]
    d.q, d.q_tok_stride, d.q_head_stride = _p(s["q"]), s["q"].stride(0), s["q"].stride(1)
    if s["gate"] is not None:
        d.gate, d.gate_dtype = _p(s["gate"]), code(s["gate"])
        d.gate_tok_stride, d.gate_head_stride = s["gate"].stride(0), s["gate"].stride(1)
    d.out, d.out_dtype = _p(s["out"]), code(s["out"])
    if s["acc"] is not None:
        d.acc, d.acc_stride = _p(s["acc"]), s["acc"].shape[2]
    return lib.vx27_hip_paged_attn, _ctx.h, d, L.check


def run(s):
    if own:
        fn, h, d, check = s["call"]
        check(fn(h, C.byref(d)), s["kind"])
    else:
        {"append": _append, "attn": _attn, "evict": _evict}[s["kind"]](s)
    if s["kind"] == "append":
        return {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    if s["kind"] == "attn":
        return {"out": s["out"], "acc": s["acc"]}
    return {"kept": s["kept"], "len": s["len_out"], "acc": s["acc_out"], "k": s["k"], "v": s["v"]}


# ------------------------------------------------------------ the plain form
def _owner(s):
    """(sequence, number within it) of every token."""
    n = torch.arange(s["n_tok"], device=DEV)
    b = torch.searchsorted(s["q_start"].long(), n, right=True) - 1
    return b, n - s["q_start"].long()[b]


def _rows(s):
    """The cached rows of every sequence in 32 bits, [B][n_kv][rows][256] each."""
    t, n_kv, P = s["table"].long(), s["n_kv"], s["page"]
    n = t.shape[1] * P
    k = s["k"][t].permute(0, 2, 1, 3, 4).reshape(s["B"], n_kv, n, HD).float()
    v = s["v"][t].permute(0, 2, 1, 3, 5, 4).reshape(s["B"], n_kv, n, HD).float()
    return k, v


def _attn(s):
    B, T, n_kv, grp = s["B"], s["max_T"], s["n_kv"], s["n_q"] // s["n_kv"]
    ob, ot = _owner(s)
    new = s["q_start"].diff().long()
    q = torch.zeros(B, T, n_kv, grp, HD, device=DEV)
    q[ob, ot] = s["q"].view(-1, n_kv, grp, HD).float()
    k, v = _rows(s)
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
    o = (p.view(B, n_kv, grp * T, -1) @ v).view(B, n_kv, grp, T, HD)
    o = o.permute(0, 3, 1, 2, 4).reshape(B, T, s["n_q"], HD)[ob, ot]
    if s["gate"] is not None:
        o = o * torch.sigmoid(s["gate"].float())
    s["out"].copy_(o)
    if s["acc"] is not None:
        s["acc"] += p.sum((2, 3))


def _angles(pos):
    """cos and sin of every token's angles. The angle is the framework's: the position (32 bits) times the frequency
    (32 bits), rounded to 32 bits; its cosine and sine are taken in 64."""
    e = torch.arange(ROPE // 2, dtype=torch.float32) * -2.0 / ROPE
    f = (torch.tensor(THETA, dtype=torch.float64) ** e.double()).float().to(DEV)
    a = (pos.float()[:, None] * f).double()
    return a.cos().float()[:, None], a.sin().float()[:, None]


def _norm_rope(x, w, cs, sn):
    x = x.float()
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1 + w)
    a, b, h = x[..., :ROPE // 2], x[..., ROPE // 2:ROPE], x[..., ROPE:]
    return torch.cat((a * cs - b * sn, a * sn + b * cs, h), -1)


def _append(s):
    ob, ot = _owner(s)
    row = (s["len"].long() - s["q_start"].diff().long())[ob] + ot
    cs, sn = _angles(row)
    s["q_out"].copy_(_norm_rope(s["qg"][..., :HD], s["q_norm_w"], cs, sn))
    page, at = s["table"].long()[ob, row // s["page"]], row % s["page"]
    s["k"][page, :, at] = _norm_rope(s["kv"][:, 0], s["k_norm_w"], cs, sn).to(BF)
    s["v"][page, :, at // 32, :, at % 32] = s["kv"][:, 1].to(BF)


def _evict(s):
    B, n_kv, P, C_ = s["B"], s["n_kv"], s["page"], s["budget"]
    n = s["table"].shape[1] * P
    j, length = torch.arange(n, device=DEV), s["len"].long()[:, None, None]
    held = (j < s["sink"]) | (j >= length - s["recent"]) | (length <= C_)
    rank = torch.where(held, torch.full_like(s["acc"], math.inf), s["acc"]).masked_fill(j >= length, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :C_]
    if n < C_:
        order = torch.nn.functional.pad(order, (0, C_ - n), value=n)
    order = torch.where(order < length, order, torch.full_like(order, n)).sort(-1).values
    kept_n = s["len"].long().clamp(max=C_)
    s["len_out"].copy_(kept_n)
    some = (torch.arange(C_, device=DEV) < kept_n[:, None])[:, None].expand(B, n_kv, C_)
    b, h, d = some.nonzero(as_tuple=True)
    r = order[some]
    s["kept"][some] = r.int()
    s["acc_out"][some] = s["acc"][b, h, r]
    src, dst = s["table"].long()[b, r // P], s["dst_table"].long()[b, d // P]
    r, d = r % P, d % P
    s["k"][dst, h, d] = s["k"][src, h, r]
    s["v"][dst, h, d // 32, :, d % 32] = s["v"][src, h, r // 32, :, r % 32]


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
    lens, new = _plan(case)
    n_q, n_kv = case["n_q"], case["n_kv"]
    N, row = sum(new), n_kv * HD * 2 * 2                       # (K and V of a row)
    if case["kind"] == "append":
        e = 4 if case["dtype"] == "f32" else 2
        return {"bytes": N * (n_q + 2 * n_kv) * HD * (e + 2), "flops": N * (n_q + n_kv) * HD * 6}
    if case["kind"] == "evict":
        kept = sum(min(n, case["budget"]) for n in lens)
        return {"bytes": kept * (2 * row + 8 * n_kv) + sum(lens) * 4 * n_kv, "flops": sum(lens) * n_kv}
    b, f = 0, 0
    for n, t in zip(lens, new):
        first, last = n - t, n - 1
        # rows that any of the tokens sees
        rows = n
        if case["window"]:
            lo = max(0, first - case["window"] + 1)
            rows = last + 1 - lo + min(case["sink"], lo)
        b += rows * row + (rows * n_kv * 8 if case["acc"] else 0)
        f += sum(_seen(case, i) for i in range(first, n)) * n_q * HD * 4
    out = 4 if case["out"] == "f32" else 2
    gate = {"none": 0, "f32": 4, "bf16": 2}[case["gate"]]
    return {"bytes": b + N * n_q * HD * (2 + out + gate), "flops": f}


# ------------------------------------------------------------ in 64 bits
def exact(case, seed):
    """From the definitions, sequence by sequence and head by head, in 64 bits."""
    s = prepare(case, seed)
    lens, new = _plan(case)
    n_kv, grp, P = case["n_kv"], case["n_q"] // case["n_kv"], case["page"]
    dbl = torch.float64
    if case["kind"] == "attn":
        out = torch.zeros(s["n_tok"], case["n_q"], HD, device=DEV, dtype=dbl)
        acc = s["acc"].double() if s["acc"] is not None else None
        at = 0
        for b, (n, t) in enumerate(zip(lens, new)):
            pages = s["table"][b, :_pages(case, n)].long()
            rows = torch.arange(n, device=DEV)
            for h in range(n_kv):
                k = s["k"][pages, h].reshape(-1, HD)[:n].double()
                v = s["v"][pages, h].transpose(2, 3).reshape(-1, HD)[:n].double()
                for c in range(at, at + t, 512):               # 512 tokens at a time
                    m = min(512, at + t - c)
                    i = (n - t + c - at + torch.arange(m, device=DEV))[:, None]
                    seen = rows <= i
                    if case["window"]:
                        seen = seen & ((i - rows < case["window"]) | (rows < case["sink"]))
                    for g in range(h * grp, (h + 1) * grp):
                        x = s["q"][c:c + m, g].double() @ k.t() * (HD ** -0.5)
                        x = torch.softmax(torch.where(seen, x, torch.full_like(x, -math.inf)), 1)
                        out[c:c + m, g] = x @ v
                        if acc is not None:
                            acc[b, h, :n] += x.sum(0)
            at += t
        if s["gate"] is not None:
            out /= 1 + torch.exp(-s["gate"].double())
        return {"out": out, "acc": acc}
    if case["kind"] == "append":
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

        q, kn = rotated(s["qg"][:, :, :HD], s["q_norm_w"]), rotated(s["kv"][:, 0], s["k_norm_w"])
        k, v, at = s["k"].double(), s["v"].double(), 0
        for b, (n, t) in enumerate(zip(lens, new)):
            r = torch.arange(n - t, n, device=DEV)
            page = s["table"][b].long()[r // P]
            k[page, :, r % P] = kn[at:at + t]
            v[page, :, r % P // 32, :, r % 32] = s["kv"][at:at + t, 1].double()
            at += t
        return {"q": q, "k": k, "v": v}
    # eviction moves values: what it writes are copies, and which ones are whole numbers
    k, v = s["k"].double(), s["v"].double()
    kept, acc, C_ = s["kept"].clone(), s["acc_out"].double(), case["budget"]
    for b, n in enumerate(lens):
        for h in range(n_kv):
            if n <= C_:
                keep = list(range(n))
            else:
                w = s["acc"][b, h, :n].tolist()
                middle = sorted(range(case["sink"], n - case["recent"]), key=lambda r: (-w[r], r))
                keep = sorted([*range(case["sink"]), *middle[:C_ - case["sink"] - case["recent"]],
                               *range(n - case["recent"], n)])
            r = torch.tensor(keep, device=DEV)
            d = torch.arange(len(keep), device=DEV)
            kept[b, h, :len(keep)] = r.int()
            acc[b, h, :len(keep)] = s["acc"][b, h, r].double()
            src, dst = s["table"][b].long()[r // P], s["dst_table"][b].long()[d // P]
            k[dst, h, d % P] = k[src, h, r % P]
            v[dst, h, d % P // 32, :, d % 32] = v[src, h, r % P // 32, :, r % 32]
    return {"kept": kept, "len": _i32([min(n, C_) for n in lens]), "acc": acc, "k": k, "v": v}
