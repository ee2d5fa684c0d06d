"""The 4-bit paged cache on the GPU against plain float64 results: the append's
codes byte for byte, attention (one token, ragged windows and prompts, sliding
windows with sinks), rows read by slot; then faulty tables and values, captured
graphs and other streams."""
import ctypes as C

import numpy as np
import pytest

from gpu_common import say
from paged_common import HD, f64, score_err
from q4_common import BF16_MAX, K_AT, V_AT, Batch4, get, norm_rope, out_tol, put, quantise, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from vx27_amd import lib as L
    c = L.Ctx(0)
    yield c
    c.close()


# --------------------------------------------------------------- attention
class Attn4:
    """A batch on the device and its attention call."""

    def __init__(self, ctx, bt, out_bf16=False, gate="f32", interleaved=False, device=None):
        from vx27_amd import lib as L, workloads as W
        self.ctx, self.bt, self.L, self.out_bf16, self.gated = ctx, bt, L, out_bf16, interleaved or gate != "none"
        n = bt.N * bt.n_q * HD
        self.bufs = dict(k=ctx.put(bt.kq), v=ctx.put(bt.vq), table=ctx.put(bt.table), len=ctx.put(np.asarray(bt.lens, np.int32)),
                         start=ctx.put(bt.start))
        d = self.d = L.PagedAttnDesc()
        d.B, d.n_q, d.n_kv, d.hd, d.page_size, d.n_pages, d.max_pages = bt.B, bt.n_q, bt.n_kv, HD, bt.page, bt.n_pages, bt.max_pages
        d.table, d.len, d.q_start = (self.bufs[x].ptr for x in ("table", "len", "start"))
        d.n_tok, d.max_T, d.window, d.n_sink = bt.N, max(bt.new), bt.window, bt.sink
        d.k_pages, d.v_pages = self.bufs["k"].ptr, self.bufs["v"].ptr
        if interleaved:      # q and gate of a head side by side, both bf16
            qg = np.concatenate([bt.q, W.bf16_bits(bt.gate)], axis=-1)
            bt.gate = W.bf16_to_f32(W.bf16_bits(bt.gate))
            self.bufs["q"] = ctx.put(qg)
            d.q, d.q_tok_stride, d.q_head_stride = self.bufs["q"].ptr, bt.n_q * 2 * HD, 2 * HD
            d.gate, d.gate_dtype, d.gate_tok_stride, d.gate_head_stride = d.q + 2 * HD, L.BF16, bt.n_q * 2 * HD, 2 * HD
        else:
            self.bufs["q"] = ctx.put(bt.q)
            d.q = self.bufs["q"].ptr
            if gate != "none":
                self.bufs["gate"] = ctx.put(W.bf16_bits(bt.gate) if gate == "bf16" else bt.gate)
                if gate == "bf16":
                    bt.gate = W.bf16_to_f32(W.bf16_bits(bt.gate))
                d.gate, d.gate_dtype = self.bufs["gate"].ptr, L.BF16 if gate == "bf16" else L.F32
        self.sentinel = np.full(n, 0x7FA5, np.uint16) if out_bf16 else np.full(n, -777.25, np.float32)
        self.bufs["out"] = ctx.put(self.sentinel)
        d.out, d.out_dtype = self.bufs["out"].ptr, L.BF16 if out_bf16 else L.F32
        self.bufs["lse"] = ctx.put(np.full(bt.N * bt.n_q, -777.25, np.float32))
        d.lse = self.bufs["lse"].ptr

    def call(self):
        self.L.check(self.L.lib().vx27_hip_paged_attn_q4(self.ctx.h, C.byref(self.d)), "paged_attn_q4")

    def out(self):
        bt = self.bt
        if self.out_bf16:
            return f64(self.bufs["out"].download((bt.N, bt.n_q, HD), np.uint16))
        return self.bufs["out"].download((bt.N, bt.n_q, HD), np.float32).astype(np.float64)

    def lse(self):
        return self.bufs["lse"].download((self.bt.N, self.bt.n_q), np.float32).astype(np.float64)

    def raw(self):
        return [self.bufs[n].download((self.bufs[n].nbytes,), np.uint8) for n in ("out", "lse")]

    def tiled(self):
        """Whether the call runs the tile kernel."""
        rows = max(self.bt.new) * self.bt.qg
        return rows > (self.L.Q4_SPLIT_ROWS if self.out_bf16 else self.L.Q4_SPLIT_ROWS_F32)

    def tol(self, ref, keys):
        """Weights are rounded to one bf16 part (2^-8), or two in the split kernel's fp32 outputs (2^-16)."""
        return out_tol(ref, keys, self.out_bf16, 2.0 ** -8 if self.out_bf16 or self.tiled() else 2.0 ** -16, self.tiled())

    def free(self):
        for b in self.bufs.values():
            b.free()

    def check(self, tag):
        self.ctx.sync()
        bt = self.bt
        ref, out = bt.result(self.gated), self.out()
        lo, hi = bt.start[0], bt.start[-1]
        err, tol = np.abs(out - ref["out"])[lo:hi], self.tol(ref, max(max(bt.lens), 1))[lo:hi]
        if err.size:
            say(f"  {tag}: max err/tol {np.nanmax(err / tol):.3f}, rel {np.linalg.norm(err) / max(np.linalg.norm(ref['out'][lo:hi]), 1e-30):.2e}")
        assert bool(np.all(err <= tol)), tag                # (a NaN fails it)
        got = self.bufs["out"].download((bt.N, bt.n_q, HD), self.sentinel.dtype)
        keep = self.sentinel.reshape(got.shape)
        assert np.array_equal(got[:lo], keep[:lo]) and np.array_equal(got[hi:], keep[hi:]), "rows of no sequence were written"
        lse, want = self.lse(), ref["lse"]
        assert np.all(lse[:lo] == -777.25) and np.all(lse[hi:] == -777.25)
        lse, want = lse[lo:hi], want[lo:hi]
        assert np.array_equal(np.isinf(lse), np.isinf(want)), tag
        f = np.isfinite(want)
        ltol = score_err(ref["S"][lo:hi]) + 2.0 ** -20 * (1 + np.abs(want)) + max(bt.lens) * 2.0 ** -24
        if self.tiled():
            ltol += 2.0 ** -8 * ref["S"][lo:hi]              # (keys rounded to bf16)
        assert np.all(np.abs(lse[f] - want[f]) <= ltol[f]), tag
        return ref


SHAPES = [   # lens, new, n_q, n_kv, page, window, sink
    ([1], [1], 24, 4, 64, 0, 0),
    ([0, 1, 31, 32, 33], [1, 1, 1, 1, 1], 24, 4, 32, 0, 0),          # a token that sees nothing
    ([1000, 7, 257], [1, 0, 1], 24, 4, 64, 0, 0),                    # a sequence without new tokens
    ([2, 1, 64, 700], [2, 1, 2, 0], 24, 4, 64, 0, 0),                # two tokens of some
    ([517, 90, 1300], [1, 1, 1], 16, 1, 128, 0, 0),                  # 16 rows a KV head
    ([333] * 5, [1] * 5, 8, 8, 96, 0, 0),                            # one row a KV head; pages no power of two
    ([900, 40, 64, 3, 700], [1] * 5, 24, 4, 64, 100, 4),             # sinks, a gap, the window
    ([900, 901, 902, 963], [1] * 4, 10, 2, 32, 64, 70),              # sinks past two tiles
    ([900, 129, 131], [2, 2, 1], 24, 4, 64, 1, 0),                   # a token sees itself alone
    ([900, 129, 131], [1, 2, 1], 24, 4, 64, 128, 1000),              # more sinks than rows
    ([50] * 70, [1] * 70, 24, 4, 32, 0, 0),                          # more than 64 sequences
    ([0, 0], [1, 0], 24, 4, 64, 7, 3),
    ([5, 6], [3, 2], 4, 2, 32, 0, 0),                                # three tokens, six rows
    ([1 + 37 * i for i in range(70)], [1 + i % 3 for i in range(70)], 24, 4, 64, 0, 0),
    ([600, 77, 6, 3000], [6, 6, 6, 5], 24, 4, 64, 0, 0),             # a drafter's tokens: blocks of query rows
    ([600, 77, 11, 0], [11, 1, 11, 2], 16, 1, 64, 40, 2),
    ([2500, 5], [9, 5], 24, 4, 96, 700, 40),
    ([130, 70, 1, 33], [130, 1, 1, 30], 24, 4, 64, 0, 0),            # prompts beside decoding tokens
    ([300, 500, 64], [260, 77, 64], 24, 4, 32, 90, 7),
    ([700], [129], 8, 8, 64, 0, 0),
    ([1200, 900], [43, 200], 16, 1, 128, 300, 33),
    ([3, 257], [3, 257], 10, 2, 64, 0, 5),
    ([0, 40, 5], [3, 60, 5], 24, 4, 64, 0, 0),                       # tokens before the first row see nothing
    ([2000, 1990], [300, 1], 24, 4, 64, 1, 0),
    ([1500, 40], [150, 20], 24, 4, 64, 64, 2000),
    ([1100, 700], [1000, 33], 16, 1, 64, 500, 9),                    # rows past the fp32 outputs' limit
    ([5000], [43], 24, 4, 256, 0, 0),                                # a short chunk over a long cache, cut into parts
]


@pytest.mark.parametrize("out_bf16", [False, True])
@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_attention(ctx, i, out_bf16):
    lens, new, n_q, n_kv, page, window, sink = SHAPES[i]
    say(f"q4 attn {i} {lens[:6]} {new[:6]} heads {n_q}/{n_kv} page {page} window {window} sink {sink} bf16 {out_bf16}")
    bt = Batch4(lens, new, n_q, n_kv, page, window, sink, seed=900 + i, lead=2, tail=3)
    at = Attn4(ctx, bt, out_bf16, gate=("f32", "bf16", "none")[i % 3], interleaved=i % 4 == 3)
    at.call()
    at.check(f"{i}")
    at.free()


@pytest.mark.parametrize("T", [1, 5, 40])
def test_tokens_without_rows(ctx, T):
    """More tokens than rows: those before the first row see nothing and get 0."""
    say(f"tokens without rows T={T}")
    bt = Batch4([3, 2, 0], [T, T, T], 24, 4, 32, seed=31 + T)
    at = Attn4(ctx, bt, False, gate="none")
    at.call()
    at.check(f"T={T}")
    at.free()


@pytest.mark.parametrize("lens,new,window,sink", [
    ([40, 9], [2, 2], 0, 0), ([300, 70], [2, 1], 33, 4), ([300, 90], [7, 3], 0, 0),
    ([90, 33], [60, 33], 0, 0), ([400, 90], [130, 90], 50, 4), ([3000, 10], [40, 3], 0, 0)])
@pytest.mark.parametrize("what", ["k", "v"])
def test_groups_held_as_nan_stay_with_the_rows_that_see_them(ctx, lens, new, window, sink, what):
    """A group of a key or value row that is held as NaN: the tokens that see it have NaN there, no other has."""
    say(f"nan groups {what} {lens} {new} window {window}")
    bt = Batch4(lens, new, 24, 4, 64, window, sink, seed=600 + new[0])
    hit = np.zeros((bt.N, 24, HD), bool)
    q, where = (bt.kq, K_AT) if what == "k" else (bt.vq, V_AT)
    clean = q.copy()
    for b in range(bt.B):
        seen = bt.seen(b)
        part = np.nonzero(seen.any(0) & ~seen.all(0))[0]
        picks = [part[0], part[len(part) // 2], part[-1]] if len(part) else []
        if seen.all(0).any():
            picks.append(np.nonzero(seen.all(0))[0][-1])
        for i, j in enumerate(dict.fromkeys(picks)):
            p, at, h, g = bt.table[b, j // 64], j % 64, i % 4, (i + b) % 4
            c, s, m = get(q[p, h, at // 32], where, at % 32)
            c2, s2, m2 = c.copy(), s.copy(), m.copy()
            c2[64 * g:64 * g + 64], s2[g], m2[g] = 0, 0, 0x7FC0
            put(q[p, h, at // 32], where, at % 32, c2, s2, m2)
            m2[g] = 0
            put(clean[p, h, at // 32], where, at % 32, c2, s2, m2)
            tokens = bt.start[b] + np.nonzero(seen[:, j])[0]
            dims = range(HD) if what == "k" else range(64 * g, 64 * g + 64)
            hit[np.ix_(tokens, range(6 * h, 6 * h + 6), dims)] = True
    assert hit.any()
    at = Attn4(ctx, bt, False, gate="none")
    at.call()
    ctx.sync()
    out = at.out()
    if what == "k":
        bt.kq = clean
    else:
        bt.vq = clean
    ref = bt.result(False)
    tol = at.tol(ref, max(lens))
    assert np.isnan(out[hit]).all()
    assert np.all(np.abs(out[~hit] - ref["out"][~hit]) <= tol[~hit])
    at.free()


@pytest.mark.parametrize("scale,offset", [(1e30, 0.0), (1e-35, 0.0), (1.0, 3000.0), (1e-3, -50.0)])
@pytest.mark.parametrize("new", [1, 3, 40])
def test_values_of_other_sizes(ctx, scale, offset, new):
    """Values far from 1 and groups far from 0 (a large minimum under a small range)."""
    say(f"values x {scale} + {offset}, {new} tokens")
    bt = Batch4([300, 45], [new, new], 24, 4, 64, seed=650 + new)
    for b, j in bt.where:
        r = bt.r.standard_normal((2, 4, HD))
        bt.set_row(b, j, r[0], (r[1] * scale + offset).astype(np.float32))
    for out_bf16 in (False, True):
        at = Attn4(ctx, bt, out_bf16, gate="none")
        at.call()
        at.check(f"bf16 {out_bf16}")
        at.free()


def test_large_scores(ctx):
    """Scores in the thousands: one key takes all the weight; nothing overflows."""
    say("large scores")
    for new in (1, 4, 50):
        bt = Batch4([400, 60], [new, new], 24, 4, 64, seed=660 + new, q_std=900.0)
        at = Attn4(ctx, bt, False, gate="none")
        at.call()
        ctx.sync()
        ref, out = bt.result(False), at.out()
        # a score's error is score_err(S), about 0.1 here: weights may be off by that factor, the outputs stay weighted
        # means of the values
        assert not at.tiled()
        e = np.expm1(2 * score_err(ref["S"]))[..., None]
        assert np.all(np.abs(out - ref["out"]) <= 2 * e * ref["W"] + 2.0 ** -8 * ref["W"] + 1e-5)
        at.free()


# ------------------------------------------------------------------ append
APPENDS = [   # lens, new, n_q, n_kv, page, rope_dim, flags (1: NORM_W), with_pos, with_q
    ([1], [1], 24, 4, 64, 64, 0, False, True),
    ([500, 31, 32, 33, 64], [1] * 5, 24, 4, 32, 64, 0, False, True),
    ([70, 3, 0, 200], [70, 3, 0, 131], 24, 4, 64, 64, 0, True, True),
    ([100, 65], [35, 2], 8, 8, 96, 128, 1, False, True),
    ([100, 65], [34, 1], 16, 1, 64, 0, 0, False, True),
    ([90], [33], 10, 2, 128, 36, 0, True, True),
    ([257, 8], [40, 8], 24, 4, 256, 256, 0, False, False),
    ([40, 41, 42, 43, 44, 45, 46, 47], [8, 7, 6, 5, 4, 3, 2, 1], 4, 2, 32, 6, 0, False, False),
]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("i", range(len(APPENDS)))
def test_append(ctx, i, dtype):
    """Codes, scales and minima byte for byte, everything else of the pages as it was; q within a bf16 rounding."""
    from vx27_amd import lib as L, workloads as W
    lens, new, n_q, n_kv, page, rope, flags, with_pos, with_q = APPENDS[i]
    say(f"append {i} {dtype} {lens} {new} heads {n_q}/{n_kv} page {page} rope {rope}")
    bt = Batch4(lens, new, n_q, n_kv, page, seed=700 + i, lead=1, tail=2)
    r, N = bt.r, bt.N
    qg, kv = W.normal(r, (N, n_q, 2 * HD)), W.normal(r, (N, 2, n_kv, HD))
    if dtype == "bf16":
        qg, kv = W.bf16_to_f32(W.bf16_bits(qg)), W.bf16_to_f32(W.bf16_bits(kv))
    qn, kn = W.normal(r, HD, 0.1), W.normal(r, HD, 0.1)
    yarn = 2.0 if with_pos else 1.0
    ps = r.integers(0, 200000, N).astype(np.int32)
    up = lambda x: ctx.put(W.bf16_bits(x) if dtype == "bf16" else x)   # noqa: E731
    bufs = dict(qg=up(qg), kv=up(kv), qn=ctx.put(qn), kn=ctx.put(kn), pos=ctx.put(ps), k=ctx.put(bt.kq), v=ctx.put(bt.vq),
                table=ctx.put(bt.table), len=ctx.put(np.asarray(lens, np.int32)), start=ctx.put(bt.start),
                out=ctx.put(np.full((N, n_q, HD), 0x7FA5, np.uint16)))
    d = L.PagedAppendDesc()
    d.B, d.n_q, d.n_kv, d.hd, d.rope_dim, d.rope_theta, d.rope_yarn, d.flags = bt.B, n_q, n_kv, HD, rope, 1e7, yarn, flags
    d.page_size, d.n_pages, d.max_pages, d.n_tok, d.max_T = page, bt.n_pages, bt.max_pages, N, max(new)
    d.table, d.len, d.q_start, d.pos = bufs["table"].ptr, bufs["len"].ptr, bufs["start"].ptr, bufs["pos"].ptr if with_pos else None
    e = 2 if dtype == "bf16" else 4
    d.in_dtype, d.k_new, d.v_new, d.kv_tok_stride = L.BF16 if dtype == "bf16" else L.F32, bufs["kv"].ptr, bufs["kv"].ptr + n_kv * HD * e, 2 * n_kv * HD
    if with_q:
        d.q, d.q_tok_stride, d.q_head_stride, d.q_norm_w, d.q_out = bufs["qg"].ptr, n_q * 2 * HD, 2 * HD, bufs["qn"].ptr, bufs["out"].ptr
    d.k_norm_w, d.k_pages, d.v_pages = bufs["kn"].ptr, bufs["k"].ptr, bufs["v"].ptr
    L.check(L.lib().vx27_hip_paged_append_q4(ctx.h, C.byref(d)), "paged_append_q4")
    ctx.sync()
    own = np.zeros(N, bool)
    row = np.zeros(N, np.int64)
    for b, (n, t) in enumerate(zip(lens, new)):
        s0 = bt.start[b]
        own[s0:s0 + t], row[s0:s0 + t] = True, np.arange(n - t, n)
    pos = ps if with_pos else row.astype(np.int32)
    k = norm_rope(kv[:, 0], kn, pos, rope, 1e7, yarn, plus_one=not flags)
    for b, t in enumerate(new):
        for x in range(bt.start[b], bt.start[b] + t):
            bt.set_row(b, row[x], k[x], kv[x, 1])
    for name, want in (("k", bt.kq), ("v", bt.vq)):
        got = bufs[name].download(want.shape, np.uint8)
        assert np.array_equal(got, want), (name, int((got != want).sum()))
    q = bufs["out"].download((N, n_q, HD), np.uint16)
    keep = ~own if with_q else np.ones(N, bool)
    assert np.all(q[keep] == 0x7FA5)
    if with_q:
        want = norm_rope(qg[..., :HD], qn, pos, rope, 1e7, yarn, plus_one=not flags)
        # bf16 rounding, and fp32's of the norm (2^-20 of the row's largest value with the angles' sine)
        tol = 2.0 ** -8 * np.abs(want) + 2.0 ** -18 * np.abs(want).max(-1, keepdims=True)
        assert np.all(np.abs(f64(q) - want)[own] <= tol[own])
    for x in bufs.values():
        x.free()


def append_v(ctx, rows, B_rows=None, k=None):
    """Appends value rows [n][1][256] (fp32) to an empty page; the bytes of K and V."""
    from vx27_amd import lib as L
    n = len(rows)
    pages = -(-n // 32)
    k = np.ones_like(rows) if k is None else k
    bufs = dict(k=ctx.put(np.zeros((pages, 1, 1, 4608), np.uint8)), v=ctx.put(np.zeros((pages, 1, 1, 4608), np.uint8)), kn=ctx.put(k),
                vn=ctx.put(rows), w=ctx.put(np.zeros(HD, np.float32)), t=ctx.put(np.arange(pages, dtype=np.int32)[None]),
                len=ctx.put(np.array([n], np.int32)), start=ctx.put(np.array([0, n], np.int32)))
    d = L.PagedAppendDesc(B=1, n_q=1, n_kv=1, hd=HD, rope_theta=1e7, rope_yarn=1.0, page_size=32, n_pages=pages, max_pages=pages,
                          n_tok=n, max_T=n)
    d.table, d.len, d.q_start, d.k_new, d.v_new, d.k_norm_w = (bufs[x].ptr for x in ("t", "len", "start", "kn", "vn", "w"))
    d.k_pages, d.v_pages = bufs["k"].ptr, bufs["v"].ptr
    L.check(L.lib().vx27_hip_paged_append_q4(ctx.h, C.byref(d)), "paged_append_q4")
    ctx.sync()
    out = [bufs[x].download((pages, 4608), np.uint8) for x in ("k", "v")]
    for x in bufs.values():
        x.free()
    return out


def test_codes_of_special_values(ctx):
    """Ties, equal values, zeros of both signs, denormals, groups far from 0, the ends of the range."""
    say("codes of special values")
    r = np.random.default_rng(41)
    f = np.float32
    rows = [np.zeros(HD), np.full(HD, 0.1), np.full(HD, -3.0), np.tile([0.0, 15.0], 128), np.tile(np.arange(16), 16) + 0.5,
            np.tile([0, 15, *np.arange(14) + 0.5], 16), np.tile([-7.5, 7.5, *np.arange(14) - 6.5], 16),     # ties: codes go to even
            np.tile([0.0, -0.0], 128), r.standard_normal(HD) * 1e-38, r.standard_normal(HD) * 1e-44, r.standard_normal(HD) * 1e37,
            1000 + r.standard_normal(HD), -1e5 + r.standard_normal(HD), np.tile([BF16_MAX, -BF16_MAX], 128),
            np.where(r.random(HD) < 0.02, 100.0, r.standard_normal(HD)), np.full(HD, 1e-45), np.tile([3e38, 1e-30], 128),
            np.round(r.standard_normal(HD) * 4) / 4, np.tile([1.0, np.nextafter(f(1), f(2))], 128)]
    rows += [r.integers(-40, 40, HD) / 2.0 ** r.integers(0, 6) for _ in range(45)]                       # many ties
    rows = np.array(rows, f)[:, None]
    got = append_v(ctx, rows)[1]
    c, s, m = quantise(rows[:, 0].astype(np.float64))
    for i in range(len(rows)):
        gc, gs, gm = get(got[i // 32], V_AT, i % 32)
        # (a minimum of zero may have either sign)
        assert np.array_equal(gs, s[i]) and np.array_equal(gc, c[i]), i
        assert np.all((gm == m[i]) | ((gm | m[i]) & 0x7FFF == 0)), i
        x = rows[i, 0].astype(np.float64)
        off = np.abs(values(c[i], s[i], m[i]) - x).reshape(4, 64)
        assert np.all(off <= f64(s[i])[:, None] / 2 * (1 + 2.0 ** -40)), i


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3.4e38])
def test_groups_that_cannot_be_held(ctx, bad):
    """A group with an infinity, a NaN or a value past bf16's range is held as NaN; the row's others as without it. Of a
    key, the norm takes a NaN to the whole row and an infinity to NaN and zeros."""
    say(f"groups with {bad}")
    r = np.random.default_rng(42)
    rows = r.standard_normal((40, 1, HD)).astype(np.float32)
    rows[5, 0, 70] = rows[33, 0, 255] = bad
    with np.errstate(all="ignore"):
        kb, vb = append_v(ctx, rows, k=rows)
        k = norm_rope(rows, np.zeros(HD, np.float32), np.arange(40), 0, 1e7)[:, 0]
        for got, at, x in ((vb, V_AT, rows[:, 0].astype(np.float64)), (kb, K_AT, k)):
            c, s, m = quantise(x)
            for i in range(40):
                gc, gs, gm = get(got[i // 32], at, i % 32)
                nan = np.isnan(f64(m[i]))
                assert np.array_equal(np.isnan(f64(gm)), nan), i
                ok = np.repeat(~nan, 64)
                assert np.array_equal(gc[ok], c[i][ok]) and np.array_equal(gs, s[i]), i
                assert np.all((gm == m[i]) | nan | ((gm | m[i]) & 0x7FFF == 0)), i
    assert np.isnan(f64(quantise(rows[5].astype(np.float64))[2])).any()


# -------------------------------------------------------------------- read
@pytest.mark.parametrize("out_bf16", [False, True])
@pytest.mark.parametrize("n_kv,page,n", [(4, 64, 1), (4, 32, 77), (1, 96, 300), (8, 128, 1000)])
def test_read(ctx, n_kv, page, n, out_bf16):
    """Rows by slot, in any order, twice and not at all (-1)."""
    from vx27_amd import lib as L, workloads as W
    say(f"read {n} rows of {n_kv} heads, page {page}")
    bt = Batch4([300, 129], [300, 129], n_kv, n_kv, page, seed=800 + n)
    r = bt.r
    sets = [np.arange(300), np.arange(129)]
    slots = np.concatenate([bt.table[b, x // page] * page + x % page for b, x in enumerate(sets)]).astype(np.int32)
    owner = np.concatenate([np.stack([np.full(len(x), b), x]) for b, x in enumerate(sets)], axis=1)
    pick = r.integers(0, len(slots), n) if n != 300 else np.arange(300)      # (300: a whole sequence in order)
    use = slots[pick].copy()
    gone = r.random(n) < 0.1
    use[gone] = -1
    e = 2 if out_bf16 else 4
    bufs = dict(k=ctx.put(bt.kq), v=ctx.put(bt.vq), slots=ctx.put(use), ko=ctx.put(np.full(n * n_kv * HD * e, 0x5A, np.uint8)),
                vo=ctx.put(np.full(n * n_kv * HD * e, 0x5A, np.uint8)))
    held = [bt.held(b) for b in range(2)]
    for skip in (None, "ko", "vo"):
        d = L.PagedReadDesc(n_kv=n_kv, hd=HD, page_size=page, n_pages=bt.n_pages, n_rows=n, slots=bufs["slots"].ptr, k_pages=bufs["k"].ptr,
                            v_pages=bufs["v"].ptr, out_dtype=L.BF16 if out_bf16 else L.F32,
                            k_out=None if skip == "ko" else bufs["ko"].ptr, v_out=None if skip == "vo" else bufs["vo"].ptr)
        for x in ("ko", "vo"):
            bufs[x].upload(np.full(bufs[x].nbytes, 0x5A, np.uint8))
        L.check(L.lib().vx27_hip_paged_read_q4(ctx.h, C.byref(d)), "paged_read_q4")
        ctx.sync()
        for w, name in enumerate(("ko", "vo")):
            raw = bufs[name].download((n, n_kv, HD * e), np.uint8)
            if skip == name:
                assert np.all(raw == 0x5A)
                continue
            assert np.all(raw[gone] == 0x5A)
            got = np.frombuffer(raw.tobytes(), np.uint16 if out_bf16 else np.float32).reshape(n, n_kv, HD)
            want = np.stack([values(*(x[j] for x in held[b][w])) for b, j in owner[:, pick].T])
            want = want.astype(np.float32)
            live = ~gone
            if out_bf16:
                assert np.array_equal(got[live], W.bf16_bits(want)[live])
            else:
                assert np.array_equal(got[live], want[live])
    for x in bufs.values():
        x.free()
