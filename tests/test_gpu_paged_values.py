"""The paged-cache operators where values and sizes are extreme: infinite and
NaN keys, values near the end of bf16's range, capacities at the limits, pages
past 2^32 elements, and work that is late on the caller's stream."""
import ctypes as C

import numpy as np
import pytest

from gpu_common import say
from paged_common import HD, Batch, out_tol
from test_gpu_paged import Attn, ctx  # noqa: F401

pytestmark = pytest.mark.gpu

NAN, MINUS_INF = 0x7FC1, 0xFF80


@pytest.mark.parametrize("lens,new,window,sink,rows", [
    ([1], [1], 0, 0, [0]),                           # all that the token sees
    ([0, 100, 7], [1, 1, 1], 1, 0, [99]),            # all of a window
    ([40, 9], [2, 2], 0, 0, [39]),                   # seen by one of two tokens
    ([3000], [1], 0, 0, range(32)),                  # a first tile
    ([3000, 50], [1, 1], 0, 0, range(3000)),         # every part of a cut sequence
    ([900, 40], [1, 1], 100, 4, range(4)),           # the sinks
    ([3], [3], 0, 0, [0]),                           # tile kernel
    ([90, 33], [60, 33], 0, 0, range(32)),
    ([90, 33], [60, 33], 0, 0, [80]),
    ([400, 90], [130, 90], 50, 4, range(300, 332)),
    ([3000, 10], [40, 3], 0, 0, range(64)),          # cut into parts: the first part's first step
    ([3000, 10], [40, 3], 0, 0, range(3000)),
])
def test_nan_keys_reach_the_tokens_that_see_them(ctx, lens, new, window, sink, rows):  # noqa: F811
    """NaN in one KV head's keys: the outputs and lse of that head's queries that see one are NaN, all others as without."""
    say(f"nan keys {lens} {new} window {window} rows {list(rows)[:3]}")
    bt = Batch(lens, new, 24, 4, 64, window, sink, seed=500 + len(rows) + lens[0])
    b = int(np.argmax(lens))
    hit = np.zeros((bt.N, 24), bool)
    clean = bt.k.copy()
    seen = bt.seen(b)
    for j in rows:
        p, at = bt.table[b, j // bt.page], j % bt.page
        bt.k[p, 1, at] = NAN
        clean[p, 1, at] = 0
        hit[np.ix_(bt.start[b] + np.nonzero(seen[:, j])[0], range(6, 12))] = True
    assert hit.any()
    at = Attn(ctx, bt, gate="none")
    at.call()
    ctx.sync()
    out, lse = at.out(), at.bufs["lse"].download((bt.N, 24), np.float32)
    bt.k = clean
    ref = bt.result(False)
    tol = out_tol(ref, max(lens), False, max(new) * 6 > 16)
    assert np.isnan(out[hit]).all() and np.isnan(lse[hit]).all()
    assert np.all(np.abs(out[~hit] - ref["out"][~hit]) <= tol[~hit])
    assert not np.isnan(lse[~hit]).any()
    at.free()


@pytest.mark.parametrize("lens,new,rows", [
    ([1, 40], [1, 1], 1), ([2, 40], [2, 2], 2), ([2, 40], [2, 2], 1),
    ([300, 40], [1, 1], 300), ([3, 70], [3, 9], 3), ([60, 70], [60, 9], 40)])
def test_scores_of_minus_infinity(ctx, lens, new, rows):  # noqa: F811
    """Keys whose scores are -inf weigh nothing; a token that sees no others gets 0, lse -inf, and adds nothing."""
    say(f"-inf scores {lens} {new} rows {rows}")
    bt = Batch(lens, new, 24, 4, 64, seed=520 + rows)
    bt.q[..., 0] = np.where(bt.q[..., 0] & 0x7FFF, bt.q[..., 0] & 0x7FFF, 0x3F80)      # q_0 > 0
    seen = bt.seen(0)
    none = bt.start[0] + np.nonzero(~seen[:, rows:].any(1))[0]                           # tokens without a finite score
    assert len(none)
    for j in range(rows):
        p, at = bt.table[0, j // 64], j % 64
        bt.k[p, :, at] = 0
        bt.k[p, :, at, 0] = MINUS_INF
    at = Attn(ctx, bt, gate="none", acc=True)
    at.call()
    ctx.sync()
    out, lse = at.out(), at.bufs["lse"].download((bt.N, 24), np.float32)
    acc = at.bufs["acc"].download((bt.B, 4, at.stride), np.float32).astype(np.float64)
    with np.errstate(invalid="ignore"):
        ref = bt.result(False)      # (its weights of these rows are exp(-inf - m) = 0)
    assert not out[none].any() and np.all(lse[none] == -np.inf)
    # (score magnitudes of the finite ones: sums of 256 products of std 2 and 1 over 16, 20.4 on average, below 64)
    S = np.where(np.isfinite(ref["S"]), ref["S"], 0).max()
    rel = 2 * 256 * 2.0 ** -24 * max(S, 64.0) + 2.0 ** -20 + 3 * max(lens) * 2.0 ** -24 + 2.0 ** -8
    some = np.setdiff1d(np.arange(bt.N), none)
    assert np.all(np.abs(out[some] - ref["out"][some]) <= 1.01 * rel * ref["W"][some] + 1e-30)
    for b, n in enumerate(lens):
        base, w = at.acc0[b, :, :n].astype(np.float64), ref["acc"][b]
        assert np.all(np.abs(acc[b, :, :n] - base - w) <= 2 * rel * w + 2.0 ** -23 * (base + w)), b
    at.free()


@pytest.mark.parametrize("T", [1, 2, 3, 60])
@pytest.mark.parametrize("power", [60, 100])
def test_large_values_and_rising_scores(ctx, T, power):  # noqa: F811
    """Values of 2^60 and 2^100 where the scores rise by 30 past those of the first keys: sums stay finite."""
    from vx27_amd import workloads as W
    say(f"values 2^{power} T={T}")
    bt = Batch([400, 130], [T, T], 24, 4, 64, seed=540 + T)
    q = np.zeros((bt.N, 24, HD), np.float32)
    q[..., 0] = 16.0
    bt.q = W.bf16_bits(q)
    for b, n in enumerate(bt.lens):
        for j in range(n):
            k = np.zeros((4, HD), np.float32)
            k[:, 0] = 0.0 if j < 64 else 30.0 + (j % 3) / 4     # (the scores: q.k / 16)
            v = W.normal(bt.r, (4, HD)) * np.float32(2.0 ** power)
            bt.put_row(b, j, W.bf16_bits(k), W.bf16_bits(v))
    at = Attn(ctx, bt, gate="none", acc=T == 60)
    at.call()
    at.check(f"values 2^{power} T={T}")
    at.free()


@pytest.mark.parametrize("lens,new", [([70], [40]), ([3000, 9], [40, 3]), ([70], [1]), ([3000, 9], [2, 1])])
@pytest.mark.parametrize("power", [10, 26, 30, 60])
def test_weights_of_huge_scores(ctx, lens, new, power):  # noqa: F811
    """One key whose score is 2^power, all others 0: it weighs 1 for every token, whatever a score's last place is."""
    from vx27_amd import workloads as W
    say(f"scores 2^{power} {lens} {new}")
    bt = Batch(lens, new, 24, 4, 64, seed=545)
    q = np.zeros((bt.N, 24, HD), np.float32)
    q[..., 0] = 2.0 ** (power // 2 + 4)                       # (over 16)
    bt.q = W.bf16_bits(q)
    for b, n in enumerate(bt.lens):
        for j in range(n):
            k = np.zeros((4, HD), np.float32)
            k[:, 0] = 2.0 ** (power - power // 2) if j == 0 else 0.0
            bt.put_row(b, j, W.bf16_bits(k), W.bf16_bits(W.normal(bt.r, (4, HD))))
    at = Attn(ctx, bt, gate="none", acc=True)
    at.call()
    ctx.sync()
    out, lse = at.out(), at.bufs["lse"].download((bt.N, 24), np.float32)
    acc = at.bufs["acc"].download((bt.B, 4, at.stride), np.float32).astype(np.float64)
    for b, n in enumerate(bt.lens):
        w = np.zeros((4, n))
        w[:, 0] = 6 * bt.new[b]
        base = at.acc0[b, :, :n].astype(np.float64)
        # (the others weigh less than e^-1000; sums, the division and the last place of the accumulated weight)
        assert np.all(np.abs(acc[b, :, :n] - base - w) <= 2.0 ** -20 * w + 2.0 ** -23 * (base + w)), b
        _, v = bt.rows(b)
        tok = slice(bt.start[b], bt.start[b + 1])
        want = np.repeat(W.bf16_to_f32(v[0]).astype(np.float64), 6, axis=0)
        assert np.all(np.abs(out[tok] - want) <= 2.0 ** -20 * np.abs(want)), b
        # (the maximum times log2 e and back: three roundings, and those of the two constants)
        assert np.all(np.abs(lse[tok] - 2.0 ** power) <= 2.0 ** power * 2.0 ** -22), b
    at.free()


def test_eviction_of_the_largest_capacity():
    """A capacity of 2^30 rows and a budget next to it: the short sequence is moved, whatever its capacity's launch would
    be."""
    from vx27_amd import lib as L
    page, n, cap = 1 << 20, 100, 1 << 30
    r = np.random.default_rng(560)
    rows_k = r.integers(0, 65536, (n, HD)).astype(np.uint16)
    block_v = r.integers(0, 65536, (4, HD, 32)).astype(np.uint16)
    with L.Ctx(0) as c:
        k, v, acc = c.buf(2 * page * HD * 2), c.buf(2 * page * HD * 2), c.buf(cap * 4)
        k.upload(rows_k)
        v.upload(block_v)
        acc.zero()
        table, dst = np.zeros((1, cap // page), np.int32), np.ones((1, cap // page), np.int32)
        tb, db, ln, dl = c.put(table), c.put(dst), c.put(np.array([n], np.int32)), c.put(np.array([-1], np.int32))
        d = L.PagedEvictDesc()
        d.B, d.n_kv, d.hd, d.page_size, d.n_pages, d.max_pages = 1, 1, HD, page, 2, cap // page
        d.table, d.len, d.budget, d.acc, d.acc_stride = tb.ptr, ln.ptr, cap - 1, acc.ptr, cap
        d.k_pages, d.v_pages, d.dst_table, d.dst_max_pages, d.dst_len = k.ptr, v.ptr, db.ptr, cap // page, dl.ptr
        L.check(L.lib().vx27_hip_paged_evict(c.h, C.byref(d)), "paged_evict")
        c.sync()
        assert dl.download((1,), np.int32)[0] == n
        got_k, got_v = np.empty((n, HD), np.uint16), np.empty((4, HD, 32), np.uint16)
        half = page * HD * 2
        L.check(L.lib().vx27_hip_d2h(c.h, got_k.ctypes.data, k.ptr + half, got_k.nbytes))
        L.check(L.lib().vx27_hip_d2h(c.h, got_v.ctypes.data, v.ptr + half, got_v.nbytes))
        assert np.array_equal(got_k, rows_k) and np.array_equal(got_v[:3], block_v[:3])
        assert np.array_equal(got_v[3, :, :4], block_v[3, :, :4])


class Step:
    """Append, attention with weights and eviction of one batch whose pool lies `off` pages into a larger one."""

    def __init__(self, ctx, lens, new, off=0):
        from vx27_amd import lib as L, workloads as W
        self.ctx, self.L, self.off = ctx, L, off
        bt = self.bt = Batch(lens, new, page=64, seed=580)
        N, n_kv, B = bt.N, 4, bt.B
        budget, dst = 96, 2
        pool = bt.n_pages + B * dst
        self.k = np.concatenate([bt.k, np.zeros((B * dst,) + bt.k.shape[1:], np.uint16)])
        self.v = np.concatenate([bt.v, np.zeros((B * dst,) + bt.v.shape[1:], np.uint16)])
        self.lo = off * n_kv * 64 * HD * 2
        self.up = dict(q=W.normal(bt.r, (N, 24, HD)), kv=W.normal(bt.r, (2, N, n_kv, HD)),
                       acc=bt.r.random((B, n_kv, bt.max_pages * 64)).astype(np.float32))
        self.outs = dict(rot=np.zeros((N, 24, HD), np.uint16), out=np.zeros((N, 24, HD), np.float32), dl=np.zeros(B, np.int32),
                         kept=np.full((B, n_kv, budget), -1, np.int32), ao=np.zeros((B, n_kv, budget), np.float32))
        table = np.where(bt.table >= 0, bt.table + off, bt.table)
        const = dict(table=table, len=np.asarray(lens, np.int32), start=bt.start, w=W.normal(bt.r, HD, 0.1),
                     dst=np.arange(bt.n_pages, pool, dtype=np.int32) + off)
        self.buf = {n: ctx.put(x) for n, x in {**self.up, **self.outs, **const}.items()}
        self.buf["k"], self.buf["v"] = ctx.buf(self.lo + self.k.nbytes), ctx.buf(self.lo + self.v.nbytes)
        u = {n: x.ptr for n, x in self.buf.items()}
        p, a, e = self.descs = L.PagedAppendDesc(), L.PagedAttnDesc(), L.PagedEvictDesc()
        for d in self.descs:
            d.B, d.n_kv, d.hd, d.page_size, d.n_pages, d.max_pages = B, n_kv, HD, 64, off + pool, bt.max_pages
            d.table, d.len, d.k_pages, d.v_pages = u["table"], u["len"], u["k"], u["v"]
        for d in (p, a):
            d.n_q, d.q_start, d.n_tok, d.max_T = 24, u["start"], N, max(new)
        p.rope_dim, p.rope_theta, p.rope_yarn, p.q = 64, 1e7, 1.0, u["q"]
        p.k_new, p.v_new, p.q_norm_w, p.k_norm_w, p.q_out = u["kv"], u["kv"] + N * n_kv * HD * 4, u["w"], u["w"], u["rot"]
        a.q, a.out, a.acc, a.acc_stride = u["rot"], u["out"], u["acc"], bt.max_pages * 64
        e.budget, e.n_sink, e.n_recent, e.acc, e.acc_stride = budget, 4, 16, u["acc"], bt.max_pages * 64
        e.dst_table, e.dst_max_pages, e.dst_len, e.kept = u["dst"], dst, u["dl"], u["kept"]
        e.acc_out, e.acc_out_stride = u["ao"], budget

    def h2d(self, name, host):
        self.L.check(self.L.lib().vx27_hip_h2d(self.ctx.h, self.buf[name].ptr + self.lo, host.ctypes.data, host.nbytes))

    def reset(self):
        self.h2d("k", self.k)
        self.h2d("v", self.v)
        for n, x in {**self.up, **self.outs}.items():
            self.buf[n].upload(x)

    def call(self):
        lib = self.L.lib()
        for fn, d in zip((lib.vx27_hip_paged_append, lib.vx27_hip_paged_attn, lib.vx27_hip_paged_evict), self.descs):
            self.L.check(fn(self.ctx.h, C.byref(d)))

    def results(self):
        self.ctx.sync()
        got = [self.buf[n].download(x.shape, x.dtype) for n, x in {**self.outs, "acc": self.up["acc"]}.items()]
        for n, x in (("k", self.k), ("v", self.v)):
            h = np.empty_like(x)
            self.L.check(self.L.lib().vx27_hip_d2h(self.ctx.h, h.ctypes.data, self.buf[n].ptr + self.lo, h.nbytes))
            got.append(h)
        return [x.view(np.uint8) for x in got]

    def free(self):
        for b in self.buf.values():
            b.free()


SHAPES = [([300, 95, 200], [1, 1, 1]), ([300, 95, 200], [2, 1, 2]), ([300, 95, 200], [130, 1, 9]), ([40 + i for i in range(70)], [1] * 70)]


@pytest.mark.parametrize("lens,new", SHAPES)
def test_pages_past_2_to_32_elements(ctx, lens, new):  # noqa: F811
    """A pool whose used pages begin past 2^32 elements (8 GiB) of K and of V: every output's and page's bytes are those
    of the same batch at the pool's start."""
    say(f"far pages {lens[:3]} {new[:3]}")
    got = []
    for off in (0, (1 << 32) // (4 * 64 * HD) + 3):
        s = Step(ctx, lens, new, off)
        s.reset()
        s.call()
        got.append(s.results())
        s.free()
    assert all(np.array_equal(x, y) for x, y in zip(*got))


@pytest.mark.parametrize("lens,new", SHAPES)
def test_inputs_that_are_late_on_the_callers_stream(ctx, lens, new):  # noqa: F811
    """Copies of 64 GB are queued on the caller's stream, then one that delivers the inputs, then the calls: kernels on any
    other stream would be done with zeros long before."""
    from vx27_amd import lib as L
    say(f"late inputs {lens[:3]} {new[:3]}")
    lib, other = L.lib(), L.Ctx(0)
    s = Step(ctx, lens, new)
    s.reset()
    s.call()
    want = s.results()
    s.reset()
    keep = {n: ctx.put(x) for n, x in s.up.items()}
    for n in s.up:
        s.buf[n].zero()
    ctx.sync()
    big = [ctx.buf(4 << 30) for _ in range(2)]
    try:
        L.check(lib.vx27_hip_set_stream(ctx.h, lib.vx27_hip_get_stream(other.h)))
        for _ in range(16):
            L.check(lib.vx27_hip_d2d(ctx.h, big[0].ptr, big[1].ptr, 4 << 30))
        for n, x in s.up.items():
            L.check(lib.vx27_hip_d2d(ctx.h, s.buf[n].ptr, keep[n].ptr, x.nbytes))
        s.call()
        assert all(np.array_equal(x, y) for x, y in zip(s.results(), want))
    finally:
        ctx.sync()
        L.check(lib.vx27_hip_set_stream(ctx.h, None))
        other.close()
        for b in [*big, *keep.values()]:
            b.free()
        s.free()
