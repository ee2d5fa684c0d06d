"""The 4-bit paged attention where values and sizes are extreme."""
import ctypes as C

import numpy as np
import pytest

import q4_bounds as Q
from gpu_common import say
from paged_common import HD, f64
from q4_bounds import run, widen
from q4_common import BF16_MAX, BLOCK, Batch4, quantise, values
from test_gpu_paged_q4 import Attn4, ctx  # noqa: F401
from vx27_amd import workloads as W

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kernel,lens,new,window,sink,wide", [
    ("paged_rows_q4", [90, 33], [60, 33], 0, 0, True), ("paged_rows_q4", [900, 400, 300], [100, 100, 100], 50, 4, False),
    ("paged_rows_q4", [3000, 10], [40, 3], 0, 0, True), ("paged_rows_flat", [400, 90], [130, 90], 50, 4, False),
    ("paged_q4_split", [300, 90], [7, 3], 0, 0, False), ("paged_q4_split", [300, 70], [2, 1], 33, 4, False)])
def test_values_that_come_back_infinite(ctx, kernel, lens, new, window, sink, wide):  # noqa: F811
    """A value that rounds to an infinity in bf16, at rows that some tokens see and others do not: the tokens that see it
    do not lose it, and the others' outputs are as without it."""
    say(f"infinite values {kernel} {lens} {new} window {window}")
    bt = Batch4(lens, new, 24, 4, 64, window, sink, seed=1700 + new[0])
    if wide:
        widen(bt)
    seen = bt.seen(0)
    part = np.nonzero(seen.any(0) & ~seen.all(0))[0]
    picks = sorted({int(part[0]), int(part[len(part) // 2]), int(part[-1])})
    rows = bt.r.standard_normal((len(picks), 2, 4, HD))
    for j, (k, v) in zip(picks, rows):
        bt.set_row(0, j, k, v)
    clean = Attn4(ctx, bt, True, gate="none")
    assert run(clean) == kernel
    ctx.sync()
    want = clean.out()
    for j, (k, v) in zip(picks, rows):
        v = v.astype(np.float32).astype(np.float64)
        # (range 319 2^120, s 21.375 2^120: the largest value comes back as 256.6 2^120)
        v[1, 70], v[1, 90] = BF16_MAX, -2.0 ** 126
        c, s, m = quantise(v)
        with np.errstate(over="ignore"):
            x = values(c, s, m)[1]
            assert np.nonzero(np.isinf(f64(W.bf16_bits(x.astype(np.float32)))))[0].tolist() == [70]
        bt.set_row(0, j, k, v)
    at = Attn4(ctx, bt, True, gate="none")
    assert run(at) == kernel
    ctx.sync()
    out = at.out()
    hit = np.zeros((bt.N, 24), bool)
    for j in picks:
        hit[np.ix_(bt.start[0] + np.nonzero(seen[:, j])[0], range(6, 12))] = True
    assert hit.any() and not hit.all()
    # (weights of scores of std 2 over 3000 rows are above 2^-40)
    big = out[..., 70]
    assert np.all(~np.isfinite(big[hit]) | (big[hit] > 2.0 ** 80)), "an infinite value was lost"
    assert np.array_equal(out[~hit], want[~hit])
    clean.free()
    at.free()


class Wide:
    """B sequences that all read one page of 2^18 rows, of which 32 are there: sequence b has its first lens[b], and its
    last new[b] are the call's tokens."""

    def __init__(self, ctx, lens, new, n_q, n_kv, out_bf16, seed):
        from vx27_amd import lib as L
        self.ctx, self.L, self.out_bf16 = ctx, L, out_bf16
        src = Batch4([32], [32], n_q, n_kv, 32, seed=seed)
        pools = [np.zeros((1, n_kv, 1 << 13, BLOCK), np.uint8) for _ in range(2)]
        for pool, q in zip(pools, (src.kq, src.vq)):
            pool[0, :, 0] = q[src.table[0, 0], :, 0]
        bt = self.bt = Batch4.__new__(Batch4)
        r, bt.B, bt.lens, bt.new, bt.n_q, bt.n_kv, bt.qg, bt.window, bt.sink = src.r, len(lens), lens, new, n_q, n_kv, n_q // n_kv, 0, 0
        bt.start = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
        bt.N = int(bt.start[-1])
        bt.q = W.bf16_bits(W.normal(r, (bt.N, n_q, HD), 2.0))
        held = src.held(0)
        bt.held = lambda b: [[x[:bt.lens[b]] for x in part] for part in held]
        up = dict(k=pools[0], v=pools[1], table=np.zeros((bt.B, 1), np.int32), len=np.asarray(lens, np.int32), start=bt.start, q=bt.q)
        self.buf = {n: ctx.put(x) for n, x in up.items()}
        self.buf["out"] = ctx.buf(bt.N * n_q * HD * (2 if out_bf16 else 4))
        d = self.d = L.PagedAttnDesc(B=bt.B, n_q=n_q, n_kv=n_kv, hd=HD, page_size=1 << 18, n_pages=1, max_pages=1, n_tok=bt.N, max_T=max(new))
        d.table, d.len, d.q_start, d.q, d.k_pages, d.v_pages, d.out = (self.buf[x].ptr for x in ("table", "len", "start", "q", "k", "v", "out"))
        d.out_dtype = L.BF16 if out_bf16 else L.F32

    def call(self):
        self.L.check(self.L.lib().vx27_hip_paged_attn_q4(self.ctx.h, C.byref(self.d)), "paged_attn_q4")

    def check(self, kernel, tokens):
        self.ctx.sync()
        bt = self.bt
        res = Q.result(bt, kernel, False, tokens=tokens)
        out = self.buf["out"].download((bt.N, bt.n_q, HD), np.uint16 if self.out_bf16 else np.float32)
        out = f64(out) if self.out_bf16 else out.astype(np.float64)
        most, mean = Q.check(out[tokens], {n: x[tokens] for n, x in res.items()}, kernel, 32, self.out_bf16)
        say(f"  err {most:.3f}, mean {mean:.3f}")
        assert most <= 1 and mean <= 1

    def free(self):
        for b in self.buf.values():
            b.free()


def test_many_sequences_beside_one_with_many_tokens(ctx):  # noqa: F811
    """One sequence of 30 tokens beside 2199 of one, whose table has room for 8192 blocks: were all of 30 tokens, the list
    would be past 2^31, but they are not."""
    say("one of many sequences with more tokens")
    B = 2200
    w = Wide(ctx, [30] + [1 + b % 30 for b in range(B - 1)], [30] + [1] * (B - 1), 64, 4, False, 1800)
    assert B * 4 * 30 * 8192 >= 2 ** 31
    assert run(w) == "paged_q4_split"
    w.check("paged_q4_split", np.arange(w.bt.N) % 7 < 3)
    w.free()


@pytest.mark.parametrize("out_bf16", [False, True])
def test_lists_past_2_to_31_blocks(ctx, out_bf16):  # noqa: F811
    """65535 sequences with room for 8192 blocks of 4 KV heads each: the tile kernel needs no list of them."""
    say(f"lists past 2^31 blocks, bf16 {out_bf16}")
    B = 65535
    w = Wide(ctx, [1 + b % 32 for b in range(B)], [1] * B, 4, 4, out_bf16, 1810)
    assert B * 4 * 8192 >= 2 ** 31 - 65536
    assert run(w) == "paged_rows_q4"
    w.check("paged_rows_q4", np.arange(B) % 97 < 4)
    w.free()


def test_token_ranges_that_overlap_past_2_to_31_blocks(ctx):  # noqa: F811
    """Ranges that overlap can make a list longer than n_tok tokens do: nothing runs, and the next sync reports it."""
    from vx27_amd import lib as L
    say("overlapping ranges past 2^31 blocks")
    B, T = 4200, 32
    w = Wide(ctx, [32] * B, [T] + [0] * (B - 1), 64, 4, False, 1820)
    assert (B // 2) * 4 * 32 * 8192 >= 2 ** 31
    start, lens = np.zeros(B + 1, np.int32), np.full(B, 1 << 18, np.int32)
    start[1::2] = T
    for n, x in (("start", start), ("len", lens)):
        w.buf[n].upload(x)
    w.buf["out"].upload(np.full(w.buf["out"].nbytes, 0x5A, np.uint8))
    w.call()
    with pytest.raises(L.HipError, match="paged cache"):
        ctx.sync()
    assert np.all(w.buf["out"].download((w.buf["out"].nbytes,), np.uint8) == 0x5A)
    for n, x in (("start", w.bt.start), ("len", np.asarray(w.bt.lens, np.int32))):
        w.buf[n].upload(x)
    assert run(w) == "paged_q4_split"
    w.check("paged_q4_split", np.ones(w.bt.N, bool))
    w.free()


SIZES = [("paged_q4_split", [300, 70], [1, 1], False), ("paged_q4_split", [300, 70], [7, 2], False), ("paged_rows_q4", [300, 70], [40, 3], True),
         ("paged_rows_flat", [300, 170], [130, 90], False)]


def attend(ctx, bt, kernel, out_bf16):  # noqa: F811
    at = Attn4(ctx, bt, out_bf16, gate="none")
    ran = run(at)
    assert ran == kernel or (ran == "paged_q4_split" and not out_bf16)     # (fp32 outputs keep it for more tokens)
    ctx.sync()
    out = at.out()
    at.free()
    return out, ran


@pytest.mark.parametrize("out_bf16", [False, True])
@pytest.mark.parametrize("how", ["equal", "minus", "rising", "falling"])
@pytest.mark.parametrize("kernel,lens,new,wide", SIZES)
def test_scores_up_to_2_to_24(ctx, kernel, lens, new, wide, how, out_bf16):  # noqa: F811
    """Scores of just below 2^24, of either sign: equal ones weigh the same; of rising or falling ones the largest takes
    all the weight."""
    say(f"scores of 2^24 {kernel} {how} bf16 {out_bf16}")
    bt = Batch4(lens, new, 24, 4, 64, seed=1900 + new[0])
    if wide:
        widen(bt)
    sign = np.where(bt.r.random(HD) < 0.5, -1.0, 1.0)
    bt.q[:] = W.bf16_bits(np.broadcast_to(sign * 1000.0, bt.q.shape).astype(np.float32))
    for b in range(bt.B):
        n = bt.lens[b]
        for j in range(n):
            x = {"equal": 1.0, "minus": -1.0, "rising": 2 * j / n - 1, "falling": 1 - 2 * j / n}[how]
            bt.set_row(b, j, np.broadcast_to(x * 1000.0 * sign, (4, HD)), bt.r.standard_normal((4, HD)))
    out, ran = attend(ctx, bt, kernel, out_bf16)
    for b in range(bt.B):
        (kc, ks, km), v = bt.held(b)[0], values(*bt.held(b)[1])
        s = values(kc, ks, km)[:, 0] @ f64(bt.q)[0, 0] / 16
        assert 1.5e7 < np.abs(s).max() < 2 ** 24
        if ran != "paged_q4_split":
            v = Q.rounded(v)
        for t in range(bt.new[b]):
            i = bt.lens[b] - bt.new[b] + t
            pick = {"rising": slice(i, i + 1), "falling": slice(0, 1)}.get(how, slice(0, i + 1))
            want = np.repeat(v[pick].mean(0), 6, axis=0)
            # the weights are of one size: one rounding of each (two parts), fp32 sums of terms s c + |m| (twice the largest
            # value and what it is off by), the output's rounding
            part = Q.PART[ran] * np.repeat(np.abs(v[pick]).mean(0), 6, axis=0) + 2.0 ** -14 * 8
            assert np.all(np.abs(out[bt.start[b] + t] - want) <= part + (2.0 ** -8 * np.abs(want) if out_bf16 else 0.0))


@pytest.mark.parametrize("out_bf16", [False, True])
@pytest.mark.parametrize("kernel,lens,new,wide", SIZES)
def test_large_queries_of_small_keys(ctx, kernel, lens, new, wide, out_bf16):  # noqa: F811
    """Queries whose sum of 15 |q| over a group is just below 2^127, of keys as much smaller than 1."""
    say(f"large queries {kernel} bf16 {out_bf16}")
    bt = Batch4(lens, new, 24, 4, 64, seed=1930 + new[0], q_std=1.0)
    if wide:
        widen(bt)
    q = f64(bt.q)
    most = np.abs(q).reshape(bt.N, 24, 4, 64).sum(-1).max()
    up = 2.0 ** np.floor(np.log2(2.0 ** 127 / (15 * most)))
    bt.q[:] = W.bf16_bits((q * up).astype(np.float32))
    for b in range(bt.B):
        for j in range(bt.lens[b]):
            bt.set_row(b, j, (bt.r.standard_normal((4, HD)) * 2 / up).astype(np.float32), bt.r.standard_normal((4, HD)))
    out, ran = attend(ctx, bt, kernel, out_bf16)
    most, mean = Q.check(out, Q.result(bt, ran, False), ran, max(lens), out_bf16)
    assert most <= 1 and mean <= 1, (most, mean)


@pytest.mark.parametrize("out_bf16", [False, True])
@pytest.mark.parametrize("kernel,lens,new,wide", SIZES)
def test_values_up_to_2_to_127_in_all(ctx, kernel, lens, new, wide, out_bf16):  # noqa: F811
    """Values whose |s*15| + |m| times the rows seen is just below 2^127, under weights that are all the same."""
    say(f"large values {kernel} bf16 {out_bf16}")
    bt = Batch4(lens, new, 24, 4, 64, seed=1960 + new[0])
    if wide:
        widen(bt)
    bt.q[:] = 0
    r = [bt.r.standard_normal((n, 2, 4, HD)) for n in bt.lens]
    c, s, m = quantise(r[0][:, 1])
    up = 2.0 ** np.floor(np.log2(2.0 ** 127 / (max(lens) * (15 * f64(s) + np.abs(f64(m))).max())))
    for b in range(bt.B):
        for j in range(bt.lens[b]):
            bt.set_row(b, j, r[b][j, 0], (r[b][j, 1] * up).astype(np.float32))
    out, ran = attend(ctx, bt, kernel, out_bf16)
    most, mean = Q.check(out, Q.result(bt, ran, False), ran, max(lens), out_bf16)
    assert most <= 1 and mean <= 1, (most, mean)
