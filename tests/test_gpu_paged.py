"""The paged-cache operators on the GPU against plain float64 results:
append, attention (one token, ragged windows and prompts, sliding windows
with sinks, accumulated weights) and eviction; then a conversation that uses
them together, captured graphs, other streams and bad tables."""
import ctypes as C

import numpy as np
import pytest

from gpu_common import say
from paged_common import HD, Batch, f64, out_tol, score_err

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    from vx27_amd import lib as L
    c = L.Ctx(0)
    yield c
    c.close()


class Attn:
    """A batch on the device and its attention call."""

    def __init__(self, ctx, bt, out_bf16=False, gate="f32", lse=True, acc=False, interleaved=False):
        from vx27_amd import lib as L, workloads as W
        self.ctx, self.bt, self.L, self.out_bf16, self.gated = ctx, bt, L, out_bf16, gate != "none"
        n = bt.N * bt.n_q * HD
        self.bufs = dict(k=ctx.put(bt.k), v=ctx.put(bt.v), table=ctx.put(bt.table), len=ctx.put(np.asarray(bt.lens, np.int32)),
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
            if gate == "bf16":
                self.bufs["gate"] = ctx.put(W.bf16_bits(bt.gate))
                bt.gate = W.bf16_to_f32(W.bf16_bits(bt.gate))
                d.gate, d.gate_dtype = self.bufs["gate"].ptr, L.BF16
            elif gate == "f32":
                self.bufs["gate"] = ctx.put(bt.gate)
                d.gate = self.bufs["gate"].ptr
        self.sentinel = np.full(n, 0x7FA5, np.uint16) if out_bf16 else np.full(n, -777.25, np.float32)
        self.bufs["out"] = ctx.put(self.sentinel)
        d.out, d.out_dtype = self.bufs["out"].ptr, L.BF16 if out_bf16 else L.F32
        if lse:
            self.bufs["lse"] = ctx.put(np.full(bt.N * bt.n_q, -777.25, np.float32))
            d.lse = self.bufs["lse"].ptr
        if acc:
            self.stride = bt.max_pages * bt.page + 5
            self.acc0 = bt.r.random((bt.B, bt.n_kv, self.stride)).astype(np.float32)
            self.bufs["acc"] = ctx.put(self.acc0)
            d.acc, d.acc_stride = self.bufs["acc"].ptr, self.stride

    def call(self):
        self.L.check(self.L.lib().vx27_hip_paged_attn(self.ctx.h, C.byref(self.d)), "paged_attn")

    def reset(self):
        self.bufs["out"].upload(self.sentinel)
        if self.d.acc:
            self.bufs["acc"].upload(self.acc0)

    def out(self):
        bt = self.bt
        if self.out_bf16:
            return f64(self.bufs["out"].download((bt.N, bt.n_q, HD), np.uint16))
        return self.bufs["out"].download((bt.N, bt.n_q, HD), np.float32).astype(np.float64)

    def raw(self):
        """Every output's bytes."""
        return [self.bufs[n].download((self.bufs[n].nbytes,), np.uint8) for n in ("out", "lse", "acc") if n in self.bufs]

    def free(self):
        for b in self.bufs.values():
            b.free()

    def check(self, tag):
        self.ctx.sync()
        bt = self.bt
        ref, out = bt.result(self.gated), self.out()
        lo, hi = bt.start[0], bt.start[-1]
        one_part = max(bt.new) * bt.qg > 16
        err, tol = np.abs(out - ref["out"])[lo:hi], out_tol(ref, max(max(bt.lens), 1), self.out_bf16, one_part)[lo:hi]
        if err.size:
            say(f"  {tag}: max err/tol {np.nanmax(err / tol):.3f}, rel {np.linalg.norm(err) / max(np.linalg.norm(ref['out'][lo:hi]), 1e-30):.2e}")
        assert np.all(err <= tol), tag                      # (a NaN fails it)
        got = self.bufs["out"].download((bt.N, bt.n_q, HD), self.sentinel.dtype)
        keep = self.sentinel.reshape(got.shape)
        assert np.array_equal(got[:lo], keep[:lo]) and np.array_equal(got[hi:], keep[hi:]), "rows of no sequence were written"
        if not self.out_bf16 and not one_part and err.size:
            # errors of the weights are independent: their 2-norm goes by the typical score error, 16 * 2^-24 of scores up to 16
            assert np.linalg.norm(err) <= 2e-5 * max(np.linalg.norm(ref["out"]), 1e-30), tag
        if "lse" in self.bufs:
            lse = self.bufs["lse"].download((bt.N, bt.n_q), np.float32).astype(np.float64)[lo:hi]
            want = ref["lse"][lo:hi]
            assert np.array_equal(np.isinf(lse), np.isinf(want)), tag
            f = np.isfinite(want)
            ltol = score_err(ref["S"][lo:hi]) + 2.0 ** -20 * (1 + np.abs(want)) + max(bt.lens) * 2.0 ** -24
            assert np.all(np.abs(lse[f] - want[f]) <= ltol[f]), tag
        if "acc" in self.bufs:
            acc = self.bufs["acc"].download((bt.B, bt.n_kv, self.stride), np.float32).astype(np.float64)
            serr = 4 * score_err(ref["S"]).max() + 2.0 ** -18 + max(bt.lens) * 2.0 ** -24
            for b in range(bt.B):
                seen = bt.seen(b).any(0)
                a0 = self.acc0[b].astype(np.float64)
                untouched = np.ones(self.stride, bool)
                untouched[:bt.lens[b]] = ~seen
                assert np.array_equal(acc[b][:, untouched], a0[:, untouched]), (tag, b)
                w = ref["acc"][b][:, seen]
                got_b, base = acc[b][:, :bt.lens[b]][:, seen], a0[:, :bt.lens[b]][:, seen]
                assert np.all(np.abs(got_b - base - w) <= serr * w + 2.0 ** -23 * (base + w)), (tag, b)
        return ref


DECODE = [   # lens, new, n_q, n_kv, page, window, sink
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
    ([1 + 37 * i for i in range(70)], [1] * 70, 24, 4, 64, 0, 0),    # more than 64, of many workgroups each
    ([1 + 37 * i for i in range(131)], [i % 3 for i in range(131)], 16, 2, 32, 500, 40),
    ([i % 71 for i in range(1100)], [int(i % 9 > 0) for i in range(1100)], 4, 2, 32, 0, 0),   # more than 1024
]


@pytest.mark.parametrize("i", range(len(DECODE)))
@pytest.mark.parametrize("out_bf16,gate", [(False, "f32"), (True, "bf16"), (False, "none")])
def test_decode(ctx, i, out_bf16, gate):
    lens, new, n_q, n_kv, page, window, sink = DECODE[i]
    say(f"decode {i} {lens[:6]} {new[:6]} heads {n_q}/{n_kv} page {page} window {window} sink {sink}")
    bt = Batch(lens, new, n_q, n_kv, page, window, sink, seed=i, lead=i % 3, tail=i % 2)
    at = Attn(ctx, bt, out_bf16, gate, acc=i % 2 == 0 or gate == "none")
    at.call()
    at.check(f"decode {i}")
    at.free()


TILES = [
    ([3], [3], 24, 4, 32, 0, 0),
    ([70, 1, 0, 33], [70, 1, 0, 9], 24, 4, 64, 0, 0),                # prompts, a decoding token, nothing
    ([200, 150], [11, 150], 24, 4, 64, 0, 0),                        # the end of a longer cache
    ([300], [300], 16, 1, 128, 0, 0),
    ([129, 65], [65, 65], 8, 8, 96, 0, 0),
    ([400, 90], [130, 90], 24, 4, 32, 50, 4),
    ([700, 31], [60, 31], 24, 4, 64, 33, 70),                        # sinks, a gap, the window
    ([300], [37], 10, 2, 256, 1, 0),
    ([260, 7], [260, 7], 24, 4, 64, 4096, 3),                        # a window longer than the cache
    ([2, 9], [5, 4], 24, 4, 64, 0, 0),                               # tokens without a row see nothing
    ([400] + [3 + i for i in range(69)], [400] + [i % 4 for i in range(69)], 24, 4, 64, 0, 0),   # more than 1024 places for row tiles
    ([1500] * 3, [700, 1, 260], 24, 4, 96, 300, 5),                  # more row tiles than CUs, pages no power of two
    ([9000], [3], 16, 2, 64, 0, 0),                                  # one row tile a KV head, cut into many parts
]


@pytest.mark.parametrize("i", range(len(TILES)))
@pytest.mark.parametrize("out_bf16,gate,inter", [(True, "bf16", True), (False, "f32", False), (True, "none", False)])
def test_tiles(ctx, i, out_bf16, gate, inter):
    lens, new, n_q, n_kv, page, window, sink = TILES[i]
    say(f"tiles {i} {lens} {new} heads {n_q}/{n_kv} page {page} window {window} sink {sink}")
    bt = Batch(lens, new, n_q, n_kv, page, window, sink, seed=100 + i, lead=i % 2, tail=i % 3)
    at = Attn(ctx, bt, out_bf16, gate, acc=gate != "bf16" or i % 2 == 1, interleaved=inter)
    at.call()
    at.check(f"tiles {i}")
    at.free()


@pytest.mark.parametrize("T,window,sink", [(1, 0, 0), (1, 2000, 5), (40, 0, 0), (40, 2000, 5)])
def test_every_tile_counts(ctx, T, window, sink):
    """One key of each tile in turn outweighs all others: a tile that is skipped or read twice changes its sequence's
    output by O(1)."""
    from vx27_amd import workloads as W
    lens = [3100 + 37 * b for b in range(12)]
    bt = Batch(lens, [T] * 12, 24, 4, 64, window, sink, seed=300 + T)
    for b in range(12):
        seen = bt.seen(b)
        everyone = np.nonzero(seen.all(0))[0]
        tiles = np.unique(everyone // 32)
        j = everyone[everyone // 32 == tiles[(b * 7919) % len(tiles)]][-1]
        k, v = bt.rows(b)
        q = f64(bt.q)[bt.start[b]:bt.start[b + 1]].reshape(T, 4, 6, HD).mean((0, 2))
        bt.put_row(b, j, W.bf16_bits((8 * q / np.abs(q).mean()).astype(np.float32)), W.bf16_bits(np.full((4, HD), b + 1, np.float32)))
    at = Attn(ctx, bt, out_bf16=T > 2, gate="none", acc=True)
    at.call()
    at.check(f"needles T={T} window={window}")
    at.free()


@pytest.mark.parametrize("lens,new,window,sink", [
    ([40, 9], [2, 2], 0, 0),                      # decode kernels, two tokens
    ([300, 70], [2, 1], 33, 4),
    ([90, 33], [60, 33], 0, 0),                   # tile kernel
    ([400, 90], [130, 90], 50, 4),
    ([3000, 10], [40, 3], 0, 0),                  # cut into parts
])
@pytest.mark.parametrize("value", [np.nan, np.inf])
def test_infinite_values_stay_with_the_rows_that_see_them(ctx, lens, new, window, sink, value):
    """An infinite or NaN value (or a whole NaN row) reaches the tokens that see its row and no other."""
    from vx27_amd import workloads as W
    say(f"value {value} {lens} {new} window {window}")
    bt = Batch(lens, new, 24, 4, 64, window, sink, seed=400 + len(lens) + new[0])
    bits = int(W.bf16_bits(np.array([value], np.float32))[0])
    some = {}
    for b in range(bt.B):
        seen = bt.seen(b)
        part = np.nonzero(seen.any(0) & ~seen.all(0))[0]
        picks = [part[0], part[len(part) // 2], part[-1]] if len(part) else []
        if seen.all(0).any():
            picks.append(np.nonzero(seen.all(0))[0][-1])
        for q, j in enumerate(dict.fromkeys(picks)):
            p, at = bt.table[b, j // bt.page], j % bt.page
            if q == 1 and np.isnan(value):
                bt.v[p, :, at // 32, :, at % 32] = bits
                some[b, j] = slice(None)
            else:
                bt.v[p, q % 4, at // 32, 17 * q + 3, at % 32] = bits
                some[b, j] = (q % 4, 17 * q + 3)
    at = Attn(ctx, bt, out_bf16=False, gate="none", lse=False)
    at.call()
    ctx.sync()
    out = at.out()
    # where a token sees such a value its output is not finite, and everywhere else it is as without them
    hit = np.zeros(out.shape, bool)
    clean = bt.v.copy()
    for (b, j), where in some.items():
        p, a_ = bt.table[b, j // bt.page], j % bt.page
        tokens = bt.start[b] + np.nonzero(bt.seen(b)[:, j])[0]
        if isinstance(where, slice):
            hit[tokens] = True
            clean[p, :, a_ // 32, :, a_ % 32] = 0
        else:
            h, d = where
            hit[np.ix_(tokens, range(6 * h, 6 * h + 6), [d])] = True
            clean[p, h, a_ // 32, d, a_ % 32] = 0
    bt.v = clean
    ref = bt.result(False)
    tol = out_tol(ref, max(lens), False, max(new) * 6 > 16)
    assert not np.isfinite(out[hit]).any()      # (the three parts of a weight may differ in sign: an infinity can end as NaN)
    assert np.all(np.abs(out[~hit] - ref["out"][~hit]) <= tol[~hit])
    at.free()


def test_matches_the_contiguous_decode(ctx):
    """Pages of a contiguous cache's size, one a sequence: vx27_hip_gqa_decode's own output within its bar, |d| <= 2e-2 +
    1e-2 |ref|, through append and attention."""
    from vx27_amd import lib as L, mixers as M, workloads as W
    d = W.gqa_decode(B=3, L=1000)
    lay = M.GatedGQALayer(ctx, 3, 1024, d["q_norm_w"], d["k_norm_w"])
    pg = M.PagedGQALayer(ctx, 3, 3, 1024, d["q_norm_w"], d["k_norm_w"], max_pages=1)
    for b in range(3):
        lay.write_kv(b, 0, W.bf16_to_f32(d["K"][b]), W.bf16_to_f32(d["V"][b]))
    L.check(L.lib().vx27_hip_d2d(ctx.h, pg.k_pages.ptr, lay.k_cache.ptr, lay.k_cache.nbytes))
    L.check(L.lib().vx27_hip_d2d(ctx.h, pg.v_pages.ptr, lay.v_cache.ptr, lay.v_cache.nbytes))
    pg.pages, pg.free, pg.rows, pg.pos = [[0], [1], [2]], [], [int(p) for p in d["pos"]], [int(p) for p in d["pos"]]
    want = lay.decode(d["pos"], d["qg"], d["k_new"], d["v_new"])
    got = pg.step([1, 1, 1], d["qg"], d["k_new"], d["v_new"])
    err = np.abs(got.astype(np.float64) - want)
    say(f"  paged against contiguous: max {err.max():.2e} of {np.abs(want).max():.2e}")
    assert np.all(err <= 2e-2 + 1e-2 * np.abs(want)) and err.max() <= 0.02 * np.abs(want).max()
    for b in range(3):      # the appended row has the same bits
        p = int(d["pos"][b])
        k0, v0 = lay.read_kv(b, p, 1)
        k1, v1 = pg.read_rows(b)
        assert np.array_equal(k0[0], k1[p]) and np.array_equal(v0[0], v1[p])


# ------------------------------------------------------------------ append
def ref_rope(x, w, pos, rope_dim, theta, yarn, direct):
    """x [..., 256] at positions pos (leading axis): norm and rotation in float64, the angle in fp32 as everywhere here."""
    x = x.astype(np.float64)
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + 1e-6) * (w if direct else 1.0 + w)
    h = rope_dim // 2
    if h:
        f = np.array([theta ** np.float64(np.float32(-2.0 * i) / np.float32(rope_dim)) for i in range(h)]).astype(np.float32)
        a = (pos.astype(np.float32)[:, None] / np.float32(yarn) * f).astype(np.float64)[:, None]
        c, s = np.cos(a), np.sin(a)
        u, v = y[..., :h].copy(), y[..., h:rope_dim].copy()
        y[..., :h], y[..., h:rope_dim] = u * c - v * s, u * s + v * c
    return y


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens,new,n_q,n_kv,page,rope,flags,pos,with_q", [
    ([1], [1], 24, 4, 64, 64, 0, False, True),
    ([500, 31, 32, 33, 64], [1] * 5, 24, 4, 32, 64, 0, False, True),
    ([70, 3, 0, 200], [70, 3, 0, 131], 24, 4, 64, 64, 0, True, True),
    ([100, 65], [35, 2], 8, 8, 96, 128, 1, False, True),
    ([100, 65], [34, 1], 16, 1, 64, 0, 0, False, True),
    ([90], [33], 10, 2, 128, 36, 0, True, True),
    ([257, 8], [40, 8], 24, 4, 256, 256, 0, False, False),
])
def test_append(ctx, dtype, lens, new, n_q, n_kv, page, rope, flags, pos, with_q):
    from vx27_amd import lib as L, workloads as W
    say(f"append {dtype} {lens} {new} heads {n_q}/{n_kv} page {page} rope {rope}")
    bt = Batch(lens, new, n_q, n_kv, page, seed=500 + len(lens) + page, lead=1, tail=2)
    r, N = bt.r, bt.N
    qg, kv = W.normal(r, (N, n_q, 2 * HD)), W.normal(r, (N, 2, n_kv, HD))
    if dtype == "bf16":
        qg, kv = W.bf16_to_f32(W.bf16_bits(qg)), W.bf16_to_f32(W.bf16_bits(kv))
    qn, kn = W.normal(r, HD, 0.1), W.normal(r, HD, 0.1)
    ps = r.integers(0, 200000, N).astype(np.int32)
    up = lambda x: ctx.put(W.bf16_bits(x) if dtype == "bf16" else x)   # noqa: E731
    bufs = dict(qg=up(qg), kv=up(kv), qn=ctx.put(qn), kn=ctx.put(kn), pos=ctx.put(ps), k=ctx.put(bt.k), v=ctx.put(bt.v),
                table=ctx.put(bt.table), len=ctx.put(np.asarray(lens, np.int32)), start=ctx.put(bt.start),
                out=ctx.put(np.full((N, n_q, HD), 0x7FA5, np.uint16)))
    d = L.PagedAppendDesc()
    d.B, d.n_q, d.n_kv, d.hd, d.rope_dim, d.rope_theta, d.rope_yarn, d.flags = bt.B, n_q, n_kv, HD, rope, 1e7, 2.0 if pos else 1.0, flags
    d.page_size, d.n_pages, d.max_pages, d.n_tok, d.max_T = page, bt.n_pages, bt.max_pages, N, max(new)
    d.table, d.len, d.q_start, d.pos = bufs["table"].ptr, bufs["len"].ptr, bufs["start"].ptr, bufs["pos"].ptr if pos else None
    e = 2 if dtype == "bf16" else 4
    d.in_dtype, d.k_new, d.v_new, d.kv_tok_stride = L.BF16 if dtype == "bf16" else L.F32, bufs["kv"].ptr, bufs["kv"].ptr + n_kv * HD * e, 2 * n_kv * HD
    if with_q:
        d.q, d.q_tok_stride, d.q_head_stride, d.q_norm_w, d.q_out = bufs["qg"].ptr, n_q * 2 * HD, 2 * HD, bufs["qn"].ptr, bufs["out"].ptr
    d.k_norm_w, d.k_pages, d.v_pages = bufs["kn"].ptr, bufs["k"].ptr, bufs["v"].ptr
    L.check(L.lib().vx27_hip_paged_append(ctx.h, C.byref(d)), "paged_append")
    ctx.sync()
    k, v = bufs["k"].download(bt.k.shape, np.uint16), bufs["v"].download(bt.v.shape, np.uint16)
    qo = bufs["out"].download((N, n_q, HD), np.uint16)
    row = np.concatenate([[0] * bt.lead, *[np.arange(n - t, n) for n, t in zip(lens, new)], [0, 0]]).astype(np.int32)
    where = ps if pos else row
    yarn = 2.0 if pos else 1.0
    lo, hi = bt.start[0], bt.start[-1]

    def close(bits, ref, scale):
        # one rounding to bf16, and before it fp32: a few operations on values up to `scale`
        err = np.abs(f64(bits) - ref)
        assert np.all(err <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -20 * scale), float((err / (2.0 ** -8 * np.abs(ref) + 2.0 ** -20 * scale)).max())
    kref = ref_rope(kv[:, 0], kn, where, rope, 1e7, yarn, flags & 1)
    want_k, want_v = bt.k.copy(), bt.v.copy()
    for b in range(bt.B):
        for t in range(new[b]):
            tok, j = bt.start[b] + t, lens[b] - new[b] + t
            p, at = bt.table[b, j // page], j % page
            close(k[p, :, at], kref[tok], np.abs(kref[tok]).max())
            want_k[p, :, at] = k[p, :, at]
            want_v[p, :, at // 32, :, at % 32] = W.bf16_bits(kv[tok, 1])
    assert np.array_equal(k, want_k) and np.array_equal(v, want_v)      # v exactly; every other row as it was
    if with_q:
        qref = ref_rope(qg[..., :HD], qn, where, rope, 1e7, yarn, flags & 1)
        close(qo[lo:hi], qref[lo:hi], np.abs(qref).max())
    keep = slice(lo, hi) if with_q else slice(0, 0)
    qo[keep] = 0x7FA5
    assert np.all(qo == 0x7FA5)
    for x in bufs.values():
        x.free()


# ---------------------------------------------------------------- eviction
def ref_evict(acc, n, budget, sink, recent):
    """Rows kept of n, by a stable sort of (weight, row); NaN heaviest."""
    if n <= budget:
        return np.arange(n)
    mid = np.arange(sink, n - recent)
    w = np.where(np.isnan(acc[mid]), np.inf, acc[mid])
    w2 = np.isnan(acc[mid])
    order = np.lexsort((mid, -w, ~w2))
    return np.sort(np.concatenate([np.arange(sink), mid[order[:budget - sink - recent]], np.arange(n - recent, n)]))


@pytest.mark.parametrize("lens,budget,sink,recent,page,n_kv,kind", [
    ([100], 40, 4, 8, 32, 4, "heavy"),
    ([100, 40, 41, 39, 1, 0], 40, 4, 8, 64, 4, "heavy"),
    ([2500, 1100, 3000], 1000, 16, 100, 64, 2, "ties"),
    ([2500, 1100], 1, 0, 0, 128, 4, "heavy"),
    ([700, 650], 600, 600, 0, 32, 1, "heavy"),          # sinks alone
    ([700, 650], 600, 0, 600, 96, 4, "zero"),           # recent rows alone
    ([5000, 4100], 4097, 1, 64, 256, 4, "zero"),        # every weight equal: the lowest rows
    ([900, 300], 250, 2, 3, 64, 4, "odd"),              # NaN, infinities, negative numbers, -0
    ([50, 20], 4000, 1, 1, 64, 4, "heavy"),             # a budget past the capacity
    ([40000, 33000, 32769], 9000, 4, 100, 128, 1, "ties"),   # more rows than a workgroup holds in registers
])
@pytest.mark.parametrize("optional", [True, False])
def test_evict(ctx, lens, budget, sink, recent, page, n_kv, kind, optional):
    from vx27_amd import lib as L
    say(f"evict {lens} to {budget} (sinks {sink}, recent {recent}) page {page} {kind}")
    r = np.random.default_rng([78, budget, page])
    B = len(lens)
    src = [max(0, -(-n // page)) for n in lens]
    mp = max(src) + 1
    cap = mp * page
    keep = [min(n, budget) for n in lens]
    dstc = [-(-n // page) for n in keep]
    n_pages = sum(src) + sum(dstc) + 3
    perm = r.permutation(n_pages)
    table = np.full((B, mp), -1, np.int32)
    dmp = max(1, -(-min(budget, cap) // page))
    dst = np.full((B, dmp), 10 ** 6, np.int32)
    at = 0
    for b in range(B):
        table[b, :src[b]] = perm[at:at + src[b]]
        at += src[b]
        dst[b, :dstc[b]] = perm[at:at + dstc[b]]
        at += dstc[b]
    k = r.integers(0, 65536, (n_pages, n_kv, page, HD)).astype(np.uint16)
    v = r.integers(0, 65536, (n_pages, n_kv, page // 32, HD, 32)).astype(np.uint16)
    acc = np.exp(2 * r.standard_normal((B, n_kv, cap + 3))).astype(np.float32)
    if kind == "ties":
        acc = np.round(acc * 2) / 2
    if kind == "zero":
        acc[:] = 0
    if kind == "odd":
        acc = r.choice(np.array([np.nan, np.inf, -np.inf, -1.5, -0.0, 0.0, 1e-40, 3.0], np.float32), acc.shape)
    acc = np.ascontiguousarray(acc, np.float32)
    ao = np.full((B, n_kv, budget + 2), -5, np.float32)
    bufs = dict(k=ctx.put(k), v=ctx.put(v), acc=ctx.put(acc), table=ctx.put(table), dst=ctx.put(dst), len=ctx.put(np.asarray(lens, np.int32)),
                ao=ctx.put(ao), kept=ctx.put(np.full((B, n_kv, budget), -9, np.int32)), dl=ctx.put(np.full(B, -1, np.int32)))
    d = L.PagedEvictDesc()
    d.B, d.n_kv, d.hd, d.page_size, d.n_pages, d.max_pages = B, n_kv, HD, page, n_pages, mp
    d.table, d.len, d.budget, d.n_sink, d.n_recent = bufs["table"].ptr, bufs["len"].ptr, budget, sink, recent
    d.acc, d.acc_stride, d.k_pages, d.v_pages = bufs["acc"].ptr, cap + 3, bufs["k"].ptr, bufs["v"].ptr
    d.dst_table, d.dst_max_pages, d.dst_len = bufs["dst"].ptr, dmp, bufs["dl"].ptr
    if optional:
        d.acc_out, d.acc_out_stride, d.kept = bufs["ao"].ptr, budget + 2, bufs["kept"].ptr
    L.check(L.lib().vx27_hip_paged_evict(ctx.h, C.byref(d)), "paged_evict")
    ctx.sync()
    assert np.array_equal(bufs["dl"].download((B,), np.int32), keep)
    wk, wv, wkept = k.copy(), v.copy(), np.full((B, n_kv, budget), -9, np.int32)
    for b in range(B):
        for h in range(n_kv):
            rows = ref_evict(acc[b, h], lens[b], budget, sink, recent)
            assert len(rows) == keep[b]
            to = np.arange(len(rows))
            wkept[b, h, :len(rows)] = rows
            ao[b, h, :len(rows)] = acc[b, h, rows]
            sp, dp = table[b][rows // page], dst[b][to // page]
            wk[dp, h, to % page] = k[sp, h, rows % page]
            wv[dp, h, to % page // 32, :, to % 32] = v[sp, h, rows % page // 32, :, rows % 32]
    assert np.array_equal(bufs["k"].download(k.shape, np.uint16), wk)
    assert np.array_equal(bufs["v"].download(v.shape, np.uint16), wv)
    if optional:
        assert np.array_equal(bufs["kept"].download(wkept.shape, np.int32), wkept)
        assert np.array_equal(bufs["ao"].download(ao.shape, np.float32), ao, equal_nan=True)
    for x in bufs.values():
        x.free()


# ------------------------------------------------------------ used together
@pytest.mark.parametrize("window,sink", [(0, 0), (150, 4)])
def test_a_conversation(ctx, window, sink):
    """Prompts of three conversations in chunks, decoding, eviction, more decoding: each step's output against float64 on
    the rows that the cache holds (read back), each new row against its inputs, each eviction against the weights added
    up on the host."""
    from vx27_amd import mixers as M, workloads as W
    r = np.random.default_rng(91 + window)
    qn, kn = W.normal(r, HD, 0.1), W.normal(r, HD, 0.1)
    lay = M.PagedGQALayer(ctx, 3, 60, 32, qn, kn, window=window, n_sink=sink, max_pages=24)
    acc = [np.zeros((4, 0)) for _ in range(3)]

    def step(new, weigh):
        N = sum(new)
        qg, k, v = W.normal(r, (N, 24, 2 * HD)), W.normal(r, (N, 4, HD)), W.normal(r, (N, 4, HD))
        pos = np.concatenate([np.arange(p, p + t) for p, t in zip(lay.pos, new)])
        out = lay.step(new, qg, k, v, weigh=weigh).astype(np.float64)
        # the rotated queries as the attention read them: bf16
        q = f64(W.bf16_bits(ref_rope(qg[..., :HD], qn, pos, 64, 1e7, 1.0, False).astype(np.float32)))
        at = 0
        for b, t in enumerate(new):
            kk, vv = lay.read_rows(b)
            bt = Batch.__new__(Batch)
            bt.lens, bt.new, bt.n_q, bt.n_kv, bt.qg, bt.window, bt.sink = [lay.rows[b]], [t], 24, 4, 6, window, sink
            bt.B, bt.N, bt.start, bt.gate = 1, t, np.array([0, t]), qg[at:at + t, :, HD:]
            bt.rows = lambda b, kk=kk, vv=vv: (W.bf16_bits(kk), W.bf16_bits(vv))
            res = bt.result(True, q=q[at:at + t])
            tol = out_tol(res, lay.rows[b], False, max(new) * 6 > 16)
            # a query element whose fp32 value lies next to a border may have been rounded the other way: one step of
            # 2^-7 in one of 256 products now and then; as much as 2^-7 of one product in 8 of them, S/32 * 2^-7
            tol += 2 * (2.0 ** -7 / 32 * res["S"])[..., None] * res["W"]
            err = np.abs(out[at:at + t] - res["out"])
            assert np.all(err <= tol), (b, float((err / tol).max()))
            kr = ref_rope(k[at:at + t], kn, pos[at:at + t], 64, 1e7, 1.0, False)
            assert np.all(np.abs(kk[lay.rows[b] - t:] - kr) <= 2.0 ** -8 * np.abs(kr) + 2.0 ** -18)
            assert np.array_equal(vv[lay.rows[b] - t:], W.bf16_to_f32(W.bf16_bits(v[at:at + t])))
            acc[b] = np.pad(acc[b], ((0, 0), (0, lay.rows[b] - acc[b].shape[1])))
            if weigh:
                acc[b] += res["acc"][0]
            at += t

    step([70, 200, 3], False)
    step([130, 1, 64], True)
    for _ in range(3):
        step([1, 1, 1], True)
    step([2, 0, 1], True)
    step([4, 3, 0], True)                     # drafted tokens
    before = [lay.read_rows(b) for b in range(3)]
    dev = lay.acc.download((3, 4, lay.acc_stride), np.float32)
    for b in range(3):
        assert np.all(np.abs(dev[b, :, :lay.rows[b]] - acc[b]) <= 2e-2 * acc[b] + 1e-5), b    # (the queries' roundings, as above)
    rows = list(lay.rows)
    kept = lay.evict(90, 4, 20)
    assert lay.rows == [min(x, 90) for x in rows]
    for b in range(3):
        k1, v1 = lay.read_rows(b)
        for h in range(4):
            want = ref_evict(dev[b, h], rows[b], 90, 4, 20)
            assert np.array_equal(kept[b, h, :lay.rows[b]], want) and np.all(kept[b, h, lay.rows[b]:] == -1)
            assert np.array_equal(k1[:, h], before[b][0][want, h]) and np.array_equal(v1[:, h], before[b][1][want, h])
        acc[b] = np.stack([dev[b, h][kept[b, h, :lay.rows[b]]].astype(np.float64) for h in range(4)])
    assert sum(len(p) for p in lay.pages) + len(lay.free) == 60
    for _ in range(2):
        step([1, 1, 1], True)
    step([5, 40, 1], True)
    lay.evict(64, 4, 60)
    acc = [np.zeros((4, 0)) for _ in range(3)]
    step([1, 0, 2], True)


def test_same_bits_every_time(ctx):
    """Nothing depends on the order in which workgroups end: three calls on the same inputs give the same bits."""
    for new in ([1] * 9, [40, 1, 1, 30, 1, 2, 9, 0, 1]):
        bt = Batch([2000, 300, 45, 1200, 64, 900, 9, 100, 2500], new, seed=7)
        at = Attn(ctx, bt, gate="f32", acc=True)
        got = []
        for _ in range(3):
            at.reset()
            at.call()
            ctx.sync()
            got.append(at.raw())
        assert all(np.array_equal(x, y) for g in got[1:] for x, y in zip(got[0], g))
        at.free()


def test_captured_and_replayed():
    """Two graphs on one context (their workspace is shared) replayed several times, with eager calls and a larger eager
    call between: every replay equals the eager result bit for bit."""
    from vx27_amd import lib as L
    with L.Ctx(0) as ctx:
        a = Attn(ctx, Batch([1500, 90, 700], [1, 1, 1], seed=21), acc=True)
        b = Attn(ctx, Batch([800, 64], [30, 64], seed=22), out_bf16=True, gate="bf16", acc=True)
        big = Attn(ctx, Batch([900] * 6, [2] * 6, seed=23), acc=True)
        want = []
        for x in (a, b):
            x.call()
            ctx.sync()
            want.append(x.raw())
        graphs = []
        for x in (a, b):
            ctx.graph_begin()
            x.call()
            graphs.append(ctx.graph_end())
        try:
            for rep in range(4):
                for x, g, w in zip((a, b), graphs, want):
                    x.reset()
                    ctx.graph_launch(g)
                    ctx.sync()
                    assert all(np.array_equal(p, q) for p, q in zip(x.raw(), w)), rep
                    if rep == 1:
                        big.reset()
                        big.call()
                        ctx.sync()
                    x.reset()
                    x.call()
                    ctx.sync()
                    assert all(np.array_equal(p, q) for p, q in zip(x.raw(), w)), rep
        finally:
            for g in graphs:
                L.check(L.lib().vx27_hip_graph_destroy(g), "graph_destroy")
        big.check("after replays")


def test_unsized_workspace_is_refused_in_a_capture():
    from vx27_amd import lib as L
    with L.Ctx(0) as ctx:
        a = Attn(ctx, Batch([4000] * 8, [1] * 8, seed=24), acc=True)
        ctx.graph_begin()
        rc = L.lib().vx27_hip_paged_attn(ctx.h, C.byref(a.d))
        msg = L.lib().vx27_hip_last_error().decode()
        g = ctx.graph_end()
        L.check(L.lib().vx27_hip_graph_destroy(g), "graph_destroy")
        assert rc == -1 and "before capturing" in msg
        a.call()
        a.check("eager afterwards")


def test_on_another_stream(ctx):
    """The calls go to the context's stream, whichever it is: work queued there before them is seen by them."""
    from vx27_amd import lib as L
    other = L.Ctx(0)
    bt = Batch([300, 20], [1, 1], seed=25)
    a = Attn(ctx, bt, acc=False)
    q = a.bufs["q"].download((bt.N, bt.n_q, HD), np.uint16)
    a.bufs["q"].zero()
    ctx.sync()
    keep = ctx.put(q)
    try:
        L.check(L.lib().vx27_hip_set_stream(ctx.h, L.lib().vx27_hip_get_stream(other.h)))
        L.check(L.lib().vx27_hip_d2d(ctx.h, a.bufs["q"].ptr, keep.ptr, q.nbytes))
        a.call()
        a.check("another stream")
    finally:
        L.check(L.lib().vx27_hip_set_stream(ctx.h, None))
        other.close()
    a.free()


@pytest.mark.parametrize("what", ["page", "negative page", "length", "start", "long", "append without rows"])
def test_bad_indices_are_reported(ctx, what):
    """Tables, lengths and token ranges outside their buffers: no access leaves them (host clamps, checked on the CPU in
    test_paged_host.py), the next sync reports it and the context goes on."""
    from vx27_amd import lib as L
    bt = Batch([200, 100], [1, 1], seed=26)
    good = bt.table.copy(), list(bt.lens), bt.start.copy()
    if what == "page":
        bt.table[1, 0] = bt.n_pages
    if what == "negative page":
        bt.table[1, 0] = -1
    if what == "length":
        bt.lens[0] = bt.max_pages * bt.page + 1
    if what == "start":
        bt.start[2] = bt.N + 1
    if what == "long":
        bt.start[:] = [0, 2, 2]
    a = Attn(ctx, bt, gate="none", lse=False)
    if what == "append without rows":
        d = L.PagedAppendDesc()
        d.B, d.n_kv, d.hd, d.page_size, d.n_pages, d.max_pages = 2, 4, HD, bt.page, bt.n_pages, bt.max_pages
        ln = ctx.put(np.array([200, 0], np.int32))
        kv = ctx.put(np.zeros((2, 4, HD), np.float32))
        kn = ctx.put(np.zeros(HD, np.float32))
        d.table, d.len, d.n_tok, d.max_T, d.k_new, d.v_new, d.k_norm_w = a.d.table, ln.ptr, 2, 1, kv.ptr, kv.ptr, kn.ptr
        d.k_pages, d.v_pages = a.d.k_pages, a.d.v_pages
        L.check(L.lib().vx27_hip_paged_append(ctx.h, C.byref(d)))
    else:
        a.call()
    with pytest.raises(L.HipError, match="paged cache"):
        ctx.sync()
    a.free()
    bt.table, bt.lens, bt.start = good
    a = Attn(ctx, bt, gate="none")
    a.call()
    a.check("after the report")
    a.free()


def test_no_tokens(ctx):
    from vx27_amd import lib as L
    bt = Batch([200, 100], [1, 1], seed=27)
    a = Attn(ctx, bt)
    a.d.n_tok = a.d.max_T = 0
    a.call()
    ctx.sync()
    assert np.array_equal(a.bufs["out"].download(a.sentinel.shape, np.float32), a.sentinel)
    a.free()


def test_a_step_captured_and_replayed():
    """Append, attention with weights and eviction in one graph, replayed over fresh pages and weights: each replay's
    bytes are the eager step's."""
    from vx27_amd import lib as L, workloads as W
    lens, P, n_kv, budget = [301, 90, 640], 64, 4, 128
    bt = Batch(lens, [1] * 3, page=P, seed=31)
    dst = 2
    pool = bt.n_pages + 3 * dst
    k = np.concatenate([bt.k, np.zeros((3 * dst,) + bt.k.shape[1:], np.uint16)])
    v = np.concatenate([bt.v, np.zeros((3 * dst,) + bt.v.shape[1:], np.uint16)])
    stride = bt.max_pages * P
    acc = bt.r.random((3, n_kv, stride)).astype(np.float32)
    with L.Ctx(0) as ctx:
        up = dict(k=k, v=v, acc=acc, table=bt.table, len=np.asarray(lens, np.int32), dst=np.arange(bt.n_pages, pool, dtype=np.int32),
                  q=W.normal(bt.r, (3, 24, HD)), kv=W.normal(bt.r, (2, 3, n_kv, HD)), w=W.normal(bt.r, HD, 0.1), rot=np.zeros((3, 24, HD), np.uint16),
                  out=np.zeros((3, 24, HD), np.float32), dl=np.zeros(3, np.int32), ao=np.zeros((3, n_kv, budget), np.float32))
        buf = {n: ctx.put(x) for n, x in up.items()}
        p, a, e = L.PagedAppendDesc(), L.PagedAttnDesc(), L.PagedEvictDesc()
        for d in (p, a, e):
            d.B, d.n_kv, d.hd, d.page_size, d.n_pages, d.max_pages = 3, n_kv, HD, P, pool, bt.max_pages
            d.table, d.len, d.k_pages, d.v_pages = buf["table"].ptr, buf["len"].ptr, buf["k"].ptr, buf["v"].ptr
        for d in (p, a):
            d.n_q, d.n_tok, d.max_T = 24, 3, 1
        p.rope_dim, p.rope_theta, p.rope_yarn, p.q, p.k_new, p.v_new = 64, 1e7, 1.0, buf["q"].ptr, buf["kv"].ptr, buf["kv"].ptr + 3 * n_kv * HD * 4
        p.q_norm_w, p.k_norm_w, p.q_out = buf["w"].ptr, buf["w"].ptr, buf["rot"].ptr
        a.q, a.out, a.acc, a.acc_stride = buf["rot"].ptr, buf["out"].ptr, buf["acc"].ptr, stride
        e.budget, e.n_sink, e.n_recent, e.acc, e.acc_stride = budget, 4, 16, buf["acc"].ptr, stride
        e.dst_table, e.dst_max_pages, e.dst_len, e.acc_out, e.acc_out_stride = buf["dst"].ptr, dst, buf["dl"].ptr, buf["ao"].ptr, budget
        lib = L.lib()

        def step():
            L.check(lib.vx27_hip_paged_append(ctx.h, C.byref(p)))
            L.check(lib.vx27_hip_paged_attn(ctx.h, C.byref(a)))
            L.check(lib.vx27_hip_paged_evict(ctx.h, C.byref(e)))

        def fresh():
            for n in ("k", "v", "acc", "rot", "out", "dl", "ao"):
                buf[n].upload(up[n])

        def raw():
            ctx.sync()
            return [buf[n].download((buf[n].nbytes,), np.uint8) for n in ("k", "v", "acc", "rot", "out", "dl", "ao")]
        step()
        want = raw()
        assert np.array_equal(buf["dl"].download((3,), np.int32), [128, 90, 128])
        fresh()
        ctx.graph_begin()
        step()
        g = ctx.graph_end()
        try:
            for rep in range(4):
                fresh()
                ctx.graph_launch(g)
                assert all(np.array_equal(x, y) for x, y in zip(raw(), want)), rep
                if rep % 2:
                    fresh()
                    step()
                    assert all(np.array_equal(x, y) for x, y in zip(raw(), want)), rep
        finally:
            L.check(lib.vx27_hip_graph_destroy(g), "graph_destroy")


def test_eviction_workspace_goes_by_the_rows(ctx):
    """Without `kept` the call's workspace is that of the rows there can be, whatever the budget."""
    from vx27_amd import lib as L
    before = ctx.mem_info()["scratch_bytes"]
    bt = Batch([70, 40], [1, 1], page=32, seed=33)
    n = bt.max_pages
    up = dict(k=bt.k, v=bt.v, table=np.zeros((2, n), np.int32), len=np.zeros(2, np.int32), dst=np.zeros((2, n), np.int32),
              dl=np.full(2, -1, np.int32), acc=np.zeros((2, 4, n * 32), np.float32))
    buf = {x: ctx.put(y) for x, y in up.items()}
    d = L.PagedEvictDesc()
    d.B, d.n_kv, d.hd, d.page_size, d.n_pages, d.max_pages, d.budget = 2, 4, HD, 32, bt.n_pages, n, 2 ** 31 - 1
    d.table, d.len, d.k_pages, d.v_pages = (buf[x].ptr for x in ("table", "len", "k", "v"))
    d.acc, d.acc_stride, d.dst_table, d.dst_max_pages, d.dst_len = buf["acc"].ptr, n * 32, buf["dst"].ptr, n, buf["dl"].ptr
    L.check(L.lib().vx27_hip_paged_evict(ctx.h, C.byref(d)), "paged_evict")
    ctx.sync()
    assert np.array_equal(buf["dl"].download((2,), np.int32), [0, 0])
    assert ctx.mem_info()["scratch_bytes"] <= max(before, 1 << 20)
    for x in buf.values():
        x.free()


def test_a_refused_step_changes_nothing(ctx):
    """A step that the pool or the library refuses leaves the layer's rows and positions, and the next one runs."""
    from vx27_amd import lib as L, mixers as M
    r = np.random.default_rng(34)
    lay = M.PagedGQALayer(ctx, 2, 3, 32, np.zeros(HD), np.zeros(HD))
    qg, k, v = (r.standard_normal((n, h, w)).astype(np.float32) for n, h, w in ((70, 24, 2 * HD), (70, 4, HD), (70, 4, HD)))
    with pytest.raises(L.HipError, match="pages"):
        lay.step([35, 35], qg, k, v)
    lay.rope_dim = 3
    with pytest.raises(L.HipError, match="rope_dim"):
        lay.step([5, 5], qg[:10], k[:10], v[:10])
    lay.rope_dim = 64
    assert lay.rows == [0, 0] and lay.pos == [0, 0]
    assert np.isfinite(lay.step([5, 5], qg[:10], k[:10], v[:10])).all()
    assert lay.rows == [5, 5] and lay.pos == [5, 5]
