"""The 4-bit paged cache's calls as a server uses them: planned, appended,
attended to and read over many steps, captured and replayed, on other streams,
from two threads, over large pools, with faulty tables, at the limits."""
import ctypes as C
import threading

import numpy as np
import pytest

from gpu_common import say
from paged_common import HD, f64
from plan_common import plan, pool
from q4_common import BLOCK, K_AT, V_AT, Batch4, get, norm_rope, out_tol, put, put_rows, quantise, values
from test_gpu_paged_q4 import SHAPES, Attn4, append_v, ctx  # noqa: F401

pytestmark = pytest.mark.gpu

SPLIT, TILES, FLAT = ([300, 95, 200], [1, 1, 1]), ([300, 95, 200], [30, 1, 9]), ([300, 95, 200], [130, 1, 9])
KINDS = [SPLIT, ([300, 95, 200], [2, 1, 2]), TILES, FLAT, ([40 + i for i in range(70)], [1] * 70)]


# ------------------------------------------------------------ used together
class Server:
    """A pool and its conversations on the device, driven by vx27_hip_paged_plan; on the host the keys and values that
    every conversation was given, quantised by the definition."""

    def __init__(self, ctx, B, n_pages, page, width, window, sink, room, seed, out_bf16=False):
        from vx27_amd import lib as L, workloads as W
        self.ctx, self.L, self.W, self.B, self.page, self.width, self.window, self.sink = ctx, L, W, B, page, width, window, sink
        self.room, self.out_bf16, self.r = room, out_bf16, np.random.default_rng(seed)
        self.state = dict(lens=np.zeros(B, int), table=np.full((B, width), -9, np.int32), nxt=np.zeros(B, int))
        _, free, n = pool(self.r, [], page, n_pages, 1)
        self.state.update(free=free, n_free=n)
        self.rows = [[] for _ in range(B)]
        self.qn, self.kn = W.normal(self.r, HD, 0.1), W.normal(self.r, HD, 0.1)
        i32 = lambda *s: np.zeros(s, np.int32)  # noqa: E731
        up = dict(new_tok=i32(B), ended=i32(B), len=i32(B), next_pos=i32(B), table=self.state["table"], free_pages=free,
                  n_free=np.array([n], np.int32), took=i32(B), q_start=i32(B + 1), slot=i32(room), pos=i32(room), seq=i32(room))
        self.buf = {n: ctx.put(x) for n, x in up.items()}
        b = self.buf
        self.sentinel = np.full((room, 24, HD), 0x7FA5, np.uint16) if out_bf16 else np.full((room, 24, HD), -777.25, np.float32)
        b.update(qg=ctx.buf(room * 24 * 2 * HD * 4), kv=ctx.buf(room * 2 * 4 * HD * 4), qn=ctx.put(self.qn), kn=ctx.put(self.kn),
                 k=ctx.put(self.r.integers(0, 256, n_pages * 4 * (page // 32) * BLOCK).astype(np.uint8)),
                 v=ctx.put(self.r.integers(0, 256, n_pages * 4 * (page // 32) * BLOCK).astype(np.uint8)),
                 q=ctx.buf(room * 24 * HD * 2), out=ctx.put(self.sentinel), ko=ctx.buf(room * 4 * HD * 4), vo=ctx.buf(room * 4 * HD * 4))
        p = self.plan_d = L.PagedPlanDesc(B=B, page_size=page, n_pages=n_pages, max_pages=width, n_tok=room)
        for n in up:
            setattr(p, n, b[n].ptr)
        p.len_out, p.next_pos_out, p.n_free_out = p.len, p.next_pos, p.n_free
        self.app, self.att = L.PagedAppendDesc(), L.PagedAttnDesc()
        for d in (self.app, self.att):
            d.B, d.n_q, d.n_kv, d.hd, d.page_size, d.n_pages, d.max_pages = B, 24, 4, HD, page, n_pages, width
            d.table, d.len, d.q_start, d.n_tok, d.max_T = p.table, p.len, p.q_start, room, room
            d.k_pages, d.v_pages = b["k"].ptr, b["v"].ptr
        a = self.app
        a.rope_dim, a.rope_theta, a.rope_yarn, a.pos = 64, 1e7, 1.0, p.pos
        a.q, a.q_tok_stride, a.q_head_stride = b["qg"].ptr, 24 * 2 * HD, 2 * HD
        a.k_new, a.v_new, a.kv_tok_stride = b["kv"].ptr, b["kv"].ptr + 4 * HD * 4, 2 * 4 * HD
        a.q_norm_w, a.k_norm_w, a.q_out = b["qn"].ptr, b["kn"].ptr, b["q"].ptr
        t = self.att
        t.q, t.window, t.n_sink, t.out, t.out_dtype = b["q"].ptr, window, sink, b["out"].ptr, L.BF16 if out_bf16 else L.F32
        t.gate, t.gate_tok_stride, t.gate_head_stride = b["qg"].ptr + HD * 4, 24 * 2 * HD, 2 * HD
        self.read = L.PagedReadDesc(n_kv=4, hd=HD, page_size=page, n_pages=n_pages, n_rows=room, slots=p.slot, k_pages=b["k"].ptr,
                                    v_pages=b["v"].ptr, k_out=b["ko"].ptr, v_out=b["vo"].ptr)

    def most(self, T):
        """The most tokens that a sequence brings."""
        self.app.max_T = self.att.max_T = T

    def give(self, new, ended):
        """The step's inputs onto the device, and what it is to lead to."""
        W, r = self.W, self.r
        s = self.state
        self.want = plan(s["lens"], new, s["table"], s["free"], s["n_free"], self.page, self.room, ended, s["nxt"])
        N = self.N = int(self.want["q_start"][-1])
        self.qg, self.kv = W.normal(r, (self.room, 24, 2 * HD)), W.normal(r, (self.room, 2, 4, HD))
        for n, x in (("new_tok", np.asarray(new, np.int32)), ("ended", np.asarray(ended, np.int32)), ("qg", self.qg), ("kv", self.kv),
                     ("out", self.sentinel)):
            self.buf[n].upload(x)
        pos = self.want["pos"][:N]
        k = norm_rope(self.kv[:N, 0], self.kn, pos, 64, 1e7)
        kq, vq = quantise(k), quantise(self.kv[:N, 1].astype(np.float64))
        for b in range(self.B):
            if ended[b]:
                self.rows[b] = []
        for i in range(N):
            self.rows[self.want["seq"][i]].append((*(x[i] for x in kq), *(x[i] for x in vq)))
        self.pos = pos

    def call(self):
        lib, h, check = self.L.lib(), self.ctx.h, self.L.check
        check(lib.vx27_hip_paged_plan(h, C.byref(self.plan_d)))
        check(lib.vx27_hip_paged_append_q4(h, C.byref(self.app)))
        check(lib.vx27_hip_paged_attn_q4(h, C.byref(self.att)))
        check(lib.vx27_hip_paged_read_q4(h, C.byref(self.read)))

    def check(self):
        self.ctx.sync()
        w, N = self.want, self.N
        get_i = lambda n, *s: self.buf[n].download(s, np.int32)  # noqa: E731
        for n, x in (("took", "took"), ("q_start", "q_start"), ("len", "len_out"), ("next_pos", "next_pos_out"), ("n_free", "n_free_out"),
                     ("slot", "slot"), ("pos", "pos"), ("seq", "seq")):
            assert np.array_equal(get_i(n, *w[x].shape), w[x]), n
        k = w["n_free_out"][0]
        table, free = get_i("table", self.B, self.width), get_i("free_pages", len(w["free_pages"]))
        assert np.array_equal(free[:k], w["free_pages"][:k])
        held = [x for b in range(self.B) for x in table[b, :-(-w["len_out"][b] // self.page)]]
        assert sorted([*held, *free[:k]]) == list(range(len(free)))
        self.state = dict(lens=w["len_out"], table=table, free=free, n_free=k, nxt=w["next_pos_out"])
        assert [len(x) for x in self.rows] == list(w["len_out"])
        if not N:
            assert np.array_equal(self.buf["out"].download(self.sentinel.shape, self.sentinel.dtype), self.sentinel)
            return
        # the rows of the step's tokens, read by slot
        for name, at, x in (("ko", 0, None), ("vo", 3, None)):
            got = self.buf[name].download((self.room, 4, HD), np.float32)[:N]
            want = np.stack([values(*self.rows[b][j][at:at + 3]) for b, j in zip(w["seq"][:N], self.row_of(N))])
            assert np.array_equal(got, want.astype(np.float32)), name
        bt = Batch4.__new__(Batch4)
        bt.lens, bt.new, bt.n_q, bt.n_kv, bt.qg, bt.window, bt.sink = list(w["len_out"]), list(w["took"]), 24, 4, 6, self.window, self.sink
        bt.B, bt.N, bt.start, bt.gate = self.B, N, w["q_start"], self.qg[:N, :, HD:]
        bt.held = lambda b: [[np.stack([r[at + i] for r in self.rows[b]]) for i in range(3)] for at in (0, 3)]
        # (the queries as the call rounded them; each within a bf16 rounding of the definition's, as the append's test has it)
        q = f64(self.buf["q"].download((self.room, 24, HD), np.uint16)[:N])
        qw = norm_rope(self.qg[:N, :, :HD], self.qn, self.pos, 64, 1e7)
        assert np.all(np.abs(q - qw) <= 2.0 ** -8 * np.abs(qw) + 2.0 ** -18 * np.abs(qw).max(-1, keepdims=True))
        ref = bt.result(True, q=q)
        rows = self.att.max_T * 6
        tiled = rows > (self.L.Q4_SPLIT_ROWS if self.out_bf16 else self.L.Q4_SPLIT_ROWS_F32)
        tol = out_tol(ref, max(bt.lens), self.out_bf16, 2.0 ** -8 if self.out_bf16 or tiled else 2.0 ** -16, tiled)
        got = self.buf["out"].download(self.sentinel.shape, self.sentinel.dtype)
        assert np.array_equal(got[N:], self.sentinel[N:])
        err = np.abs((f64(got[:N]) if self.out_bf16 else got[:N].astype(np.float64)) - ref["out"])
        assert np.all(err <= tol), float(np.nanmax(err / tol))

    def row_of(self, N):
        w = self.want
        b = w["seq"][:N]
        return (w["len_out"] - w["took"])[b] + np.arange(N) - w["q_start"][b]

    def free(self):
        for x in self.buf.values():
            x.free()


@pytest.mark.parametrize("out_bf16", [False, True])
@pytest.mark.parametrize("window,sink,page", [(0, 0, 64), (70, 4, 32)])
def test_a_server(ctx, window, sink, page, out_bf16):  # noqa: F811
    """Prompts, decoding, drafted tokens, conversations that end and others in their places, a pool that runs out: plan,
    append, attention and read of every step against the host's."""
    say(f"a server, window {window}, bf16 {out_bf16}")
    s = Server(ctx, 5, 1024 // page, page, 640 // page, window, sink, 400, 1300 + window, out_bf16)
    steps = [([130, 0, 5, 64, 33], 0), ([1] * 5, 0), ([1, 7, 1, 3, 1], 0), ([200, 1, 40, 1, 0], 0b00010), ([1] * 5, 0b11000),
             ([150, 90, 100, 120, 130], 0), ([0] * 5, 0), ([300, 300, 300, 1, 1], 0b00100), ([11, 1, 2, 1, 1], 0), ([1] * 5, 0b11111),
             ([9, 9, 9, 9, 9], 0)]
    for i, (new, over) in enumerate(steps):
        s.most(max(max(new), 1))
        s.give(new, [over >> b & 1 for b in range(5)])
        s.call()
        s.check()
    s.free()


@pytest.mark.parametrize("T", [1, 12])
def test_a_captured_server(T):
    """A step of all four calls captured once and replayed: the sequences go on, end and grow by pages without the host;
    an eager step now and then between the replays."""
    from vx27_amd import lib as L
    say(f"a captured server, up to {T} tokens")
    with L.Ctx(0) as c:
        s = Server(c, 6, 40, 32, 8, 100, 4, 6 * T, 1400 + T, out_bf16=T > 1)
        s.most(T)
        s.give([T] * 6, [0] * 6)
        s.call()
        s.check()
        c.graph_begin()
        s.call()
        g = c.graph_end()
        try:
            for step in range(14):
                new = s.r.integers(0, T + 1, 6) if T > 1 else s.r.random(6) < 0.9
                s.give(new.astype(int), (s.r.random(6) < 0.1).astype(int))
                if step % 5 == 3:
                    s.call()
                else:
                    c.graph_launch(g)
                s.check()
        finally:
            L.check(L.lib().vx27_hip_graph_destroy(g), "graph_destroy")


# ------------------------------------------------------------- every which way
def test_same_bits_every_time(ctx):  # noqa: F811
    for new in ([1] * 9, [40, 1, 1, 30, 1, 2, 9, 0, 1], [150, 1, 45, 30, 1, 2, 9, 0, 1]):
        say(f"same bits {new}")
        for out_bf16 in (False, True):
            at = Attn4(ctx, Batch4([2000, 300, 45, 1200, 64, 900, 9, 100, 2500], new, seed=7), out_bf16)
            got = []
            for _ in range(3):
                at.call()
                ctx.sync()
                got.append(at.raw())
            assert all(np.array_equal(x, y) for g in got[1:] for x, y in zip(got[0], g))
            at.free()


def test_captured_and_replayed():
    """Three graphs on one context (their workspace is shared: split kernel, tiles, tiles over values laid out in it),
    with eager calls between: every replay equals the eager result bit for bit."""
    from vx27_amd import lib as L
    say("three graphs, one workspace")
    with L.Ctx(0) as c:
        ats = [Attn4(c, Batch4([1500, 90, 700], [1, 1, 1], seed=21)), Attn4(c, Batch4([800, 64], [30, 64], seed=22), True),
               Attn4(c, Batch4([800, 64], [300, 64], seed=23), True)]
        want, graphs = [], []
        for x in ats:
            x.call()
            c.sync()
            want.append(x.raw())
        for x in ats:
            c.graph_begin()
            x.call()
            graphs.append(c.graph_end())
        try:
            for rep in range(4):
                for x, g, w in zip(ats, graphs, want):
                    c.graph_launch(g)
                    c.sync()
                    assert all(np.array_equal(p, q) for p, q in zip(x.raw(), w)), rep
                for x, w in zip(ats, want):
                    x.call()
                    c.sync()
                    assert all(np.array_equal(p, q) for p, q in zip(x.raw(), w)), rep
        finally:
            for g in graphs:
                L.check(L.lib().vx27_hip_graph_destroy(g), "graph_destroy")


@pytest.mark.parametrize("what", ["attn", "plan"])
def test_unsized_workspace_is_refused_in_a_capture(what):
    from vx27_amd import lib as L
    say(f"unsized workspace, {what}")
    with L.Ctx(0) as c:
        if what == "attn":
            a = Attn4(c, Batch4([4000] * 8, [1] * 8, seed=24))
            fn, d = L.lib().vx27_hip_paged_attn_q4, a.d
        else:
            from test_gpu_paged_plan import Plan
            B = 2000
            table, free, n = pool(np.random.default_rng(1), [5] * B, 32, 3, 2)
            a = Plan(c, [5] * B, [1] * B, table, free, n, 32, B)
            fn, d = L.lib().vx27_hip_paged_plan, a.d
        c.graph_begin()
        rc = fn(c.h, C.byref(d))
        msg = L.lib().vx27_hip_last_error().decode()
        g = c.graph_end()
        L.check(L.lib().vx27_hip_graph_destroy(g), "graph_destroy")
        assert rc == -1 and "before capturing" in msg
        a.call()
        if what == "attn":
            a.check("eager afterwards")
        c.sync()


class Step4:
    """Append, attention and read of a batch whose pages lie `off` pages into the pool."""

    def __init__(self, ctx, lens, new, off=0, out_bf16=True):
        from vx27_amd import lib as L, workloads as W
        self.ctx, self.L, self.off = ctx, L, off
        bt = self.bt = Batch4(lens, new, seed=700 + len(lens) + new[0])
        r, N = np.random.default_rng(77), bt.N
        self.up = dict(qg=W.normal(r, (N, 24, HD)), kv=W.normal(r, (2, N, 4, HD)), w=W.normal(r, HD, 0.1))
        self.page_bytes = 4 * (bt.page // 32) * BLOCK
        slots = np.concatenate([(bt.table[b, j // bt.page] + off) * bt.page + j % bt.page for b in range(bt.B) for j in [np.arange(bt.lens[b])]])
        n = self.n_rows = len(slots)
        up = dict(self.up, table=(bt.table + off).astype(np.int32), len=np.asarray(lens, np.int32), start=bt.start, slots=slots.astype(np.int32))
        self.buf = {k: ctx.put(x) for k, x in up.items()}
        self.out = dict(q=N * 24 * HD * 2, out=N * 24 * HD * (2 if out_bf16 else 4), ko=n * 4 * HD * 4, vo=n * 4 * HD * 4)
        self.buf.update({k: ctx.buf(x) for k, x in self.out.items()})
        pages = bt.n_pages + off
        self.buf.update(k=ctx.buf(pages * self.page_bytes), v=ctx.buf(pages * self.page_bytes))
        b = self.buf
        self.p, self.a = L.PagedAppendDesc(), L.PagedAttnDesc()
        for d in (self.p, self.a):
            d.B, d.n_q, d.n_kv, d.hd, d.page_size, d.n_pages, d.max_pages = bt.B, 24, 4, HD, bt.page, pages, bt.max_pages
            d.table, d.len, d.q_start, d.n_tok, d.max_T = b["table"].ptr, b["len"].ptr, b["start"].ptr, N, max(new)
            d.k_pages, d.v_pages = b["k"].ptr, b["v"].ptr
        p, a = self.p, self.a
        p.rope_dim, p.rope_theta, p.rope_yarn, p.q, p.k_new, p.v_new = 64, 1e7, 1.0, b["qg"].ptr, b["kv"].ptr, b["kv"].ptr + N * 4 * HD * 4
        p.q_norm_w, p.k_norm_w, p.q_out = b["w"].ptr, b["w"].ptr, b["q"].ptr
        a.q, a.out, a.out_dtype = b["q"].ptr, b["out"].ptr, L.BF16 if out_bf16 else L.F32
        self.rd = L.PagedReadDesc(n_kv=4, hd=HD, page_size=bt.page, n_pages=pages, n_rows=n, slots=b["slots"].ptr, k_pages=b["k"].ptr,
                                  v_pages=b["v"].ptr, k_out=b["ko"].ptr, v_out=b["vo"].ptr)

    def reset(self):
        for name, x in (("k", self.bt.kq), ("v", self.bt.vq)):
            y = np.ascontiguousarray(x)
            self.L.check(self.L.lib().vx27_hip_h2d(self.ctx.h, self.buf[name].ptr + self.off * self.page_bytes, y.ctypes.data, y.nbytes))
        for n, x in self.out.items():
            self.buf[n].upload(np.full(x, 0x5A, np.uint8))

    def call(self):
        lib, check = self.L.lib(), self.L.check
        check(lib.vx27_hip_paged_append_q4(self.ctx.h, C.byref(self.p)))
        check(lib.vx27_hip_paged_attn_q4(self.ctx.h, C.byref(self.a)))
        check(lib.vx27_hip_paged_read_q4(self.ctx.h, C.byref(self.rd)))

    def results(self):
        self.ctx.sync()
        return [self.buf[n].download((x,), np.uint8) for n, x in self.out.items()]

    def free(self):
        for x in self.buf.values():
            x.free()


@pytest.mark.parametrize("lens,new", KINDS)
def test_pages_past_2_to_32_bytes(ctx, lens, new):  # noqa: F811
    """A pool whose used pages begin past 2^32 bytes of K and of V: every output's bytes are those of the same batch at
    the pool's start."""
    say(f"far pages {lens[:3]} {new[:3]}")
    got = []
    for off in (0, (1 << 32) // (8 * BLOCK) + 3):
        s = Step4(ctx, lens, new, off)
        s.reset()
        s.call()
        got.append(s.results())
        s.free()
    assert all(np.array_equal(x, y) for x, y in zip(*got))


@pytest.mark.parametrize("lens,new", KINDS)
def test_inputs_that_are_late_on_the_callers_stream(ctx, lens, new):  # noqa: F811
    """Large copies are queued on the caller's stream, then one that delivers the inputs, then the calls: kernels on any
    other stream would be done with zeros long before."""
    from vx27_amd import lib as L
    say(f"late inputs {lens[:3]} {new[:3]}")
    lib, other = L.lib(), L.Ctx(0)
    s = Step4(ctx, lens, new)
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
        for _ in range(8):
            L.check(lib.vx27_hip_d2d(ctx.h, big[0].ptr, big[1].ptr, 4 << 30))
        for n, x in s.up.items():
            L.check(lib.vx27_hip_d2d(ctx.h, s.buf[n].ptr, keep[n].ptr, x.nbytes))
        s.call()
        assert all(np.array_equal(x, y) for x, y in zip(s.results(), want))
    finally:
        ctx.sync()
        L.check(lib.vx27_hip_set_stream(ctx.h, None))
        other.close()
        for x in (*big, *keep.values()):
            x.free()
        s.free()


def test_two_threads_at_once():
    """Two contexts, each with its own thread, stream, tables and workspace: every step gives its own bytes."""
    from vx27_amd import lib as L
    say("two threads")
    bad = []

    def work(s, want):
        for i in range(20):
            s.reset()
            s.call()
            if not all(np.array_equal(x, y) for x, y in zip(s.results(), want)):
                bad.append((s.bt.lens, i))

    ctxs = [L.Ctx(0) for _ in range(2)]
    try:
        jobs = []
        for c, x in zip(ctxs, (FLAT, ([700, 45], [1, 2]))):
            s = Step4(c, *x)
            s.reset()
            s.call()
            jobs.append((s, s.results()))
        threads = [threading.Thread(target=work, args=j) for j in jobs]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not bad
    finally:
        for c in ctxs:
            c.close()


# ------------------------------------------------------------------ lengths
@pytest.mark.parametrize("lens,new,window,sink", [
    ([20000, 9000], [1, 1], 0, 0), ([9000, 400], [6, 2], 0, 0), ([12000, 12001], [1, 1], 8000, 100), ([16000], [10], 0, 0)])
def test_long_sequences(ctx, lens, new, window, sink):  # noqa: F811
    say(f"long {lens} {new} window {window}")
    bt = Batch4(lens, new, 24, 4, 128, window, sink, seed=1500 + lens[0] + new[0])
    for out_bf16 in (False, True):
        at = Attn4(ctx, bt, out_bf16, gate="none")
        at.call()
        at.check(f"bf16 {out_bf16}")
        at.free()


@pytest.mark.parametrize("out_bf16", [False, True])
def test_every_part_of_millions_of_rows(ctx, out_bf16):  # noqa: F811
    """A sequence of 8.4 million rows (a table that repeats 40 pages): one key with half of all the weight, at places
    around the borders of a wave's tiles and look-ups. The rest is the 40 pages' rows by their numbers."""
    from vx27_amd import lib as L, workloads as W
    say(f"millions of rows, bf16 {out_bf16}")
    n_tile, P = 262144, 40
    r = np.random.default_rng(1600)
    bt = Batch4([32 * P], [1], 1, 1, 32, seed=1601)          # rows of N(0, 1) in P pages
    (kc, ks, km), (vc, vs, vm) = bt.held(0)
    order = bt.table[0, :P]
    q = r.standard_normal(HD) * 1.0
    qb = W.bf16_bits(q.astype(np.float32)[None, None])
    qf = f64(qb)[0, 0]
    s = values(kc, ks, km)[:, 0] @ qf / 16
    vals = values(vc, vs, vm)[:, 0]
    # the page of the heavy key: number P, one row along q, the others far from it
    alpha = 16 * (np.log(n_tile * 32 * np.exp(s).mean())) / (qf @ qf)
    heavy = np.stack([qf * alpha] + [-qf] * 31)[:, None]
    hv = r.standard_normal((32, 1, HD))
    kq, vq = np.concatenate([bt.kq, np.zeros((1, 1, 1, BLOCK), np.uint8)]), np.concatenate([bt.vq, np.zeros((1, 1, 1, BLOCK), np.uint8)])
    for j in range(32):
        for pages, x, at in ((kq, heavy, K_AT), (vq, hv, V_AT)):
            c, sc, m = quantise(x[j].astype(np.float64))
            put(pages[-1, 0, 0], at, j, c[0], sc[0], m[0])
    c, sc, m = quantise(heavy.astype(np.float64))
    s_heavy = (values(c, sc, m)[:, 0] @ qf / 16)
    v_heavy = values(*quantise(hv.astype(np.float64)))[:, 0]
    pick = r.integers(0, P, n_tile)
    chunk, places = n_tile // (2 * 256), []
    for wg in (0, 1, 511):
        places += [wg * chunk + x for x in (0, 3, 4, 7, 8, 4 * 61, 4 * 62 + 1, 4 * 63, 4 * 63 + 3, 4 * 64, 4 * 65 + 2, 4 * 66, 4 * 127, chunk - 1)]
    buf = dict(k=ctx.put(kq), v=ctx.put(vq), q=ctx.put(qb), len=ctx.put(np.array([32 * n_tile], np.int32)), table=ctx.buf(n_tile * 4),
               out=ctx.buf(HD * 4))
    d = L.PagedAttnDesc(B=1, n_q=1, n_kv=1, hd=HD, page_size=32, n_pages=len(kq), max_pages=n_tile, n_tok=1, max_T=1)
    d.table, d.len, d.q, d.k_pages, d.v_pages, d.out = (buf[x].ptr for x in ("table", "len", "q", "k", "v", "out"))
    d.out_dtype = L.BF16 if out_bf16 else L.F32
    e = np.exp(s).reshape(P, 32)
    page_l, page_o = e.sum(1), np.einsum("pr,prd->pd", e, vals.reshape(P, 32, HD))
    for at in places:
        p = pick.copy()
        p[at] = P
        table = np.where(p == P, len(kq) - 1, order[np.minimum(p, P - 1)]).astype(np.int32)
        buf["table"].upload(table[None])
        L.check(L.lib().vx27_hip_paged_attn_q4(ctx.h, C.byref(d)), "paged_attn_q4")
        ctx.sync()
        got = buf["out"].download((HD,), np.uint16 if out_bf16 else np.float32)
        got = f64(got) if out_bf16 else got
        n = np.bincount(p, minlength=P + 1)
        eh = np.exp(s_heavy)
        want = (n[:P] @ page_o + eh @ v_heavy) / (n[:P] @ page_l + eh.sum())
        # the heavy row has about half the weight: without it, or with it twice, the output moves by a quarter of its
        # values and more. (Sums of 8.4 million weights in fp32, in parts of at most 128 tiles a wave: 2^-13 at most.)
        assert np.all(np.abs(got - want) <= 0.01 * (1 + np.abs(want))), (at, np.abs(got - want).max())
    for x in buf.values():
        x.free()


@pytest.mark.parametrize("B,n_kv,qg", [(65535, 1, 1), (9000, 1, 16), (3, 1024, 1), (3, 1024, 16)])
@pytest.mark.parametrize("T", [1, 2, 32])
def test_most_sequences_and_heads(ctx, B, n_kv, qg, T):  # noqa: F811
    """As many sequences, or KV heads, as the calls take: a sequence of one row gives that row's value (its weight is 1);
    other tokens of a sequence come before its first row and see nothing."""
    from vx27_amd import lib as L
    say(f"B={B} n_kv={n_kv} group {qg} T={T}")
    r = np.random.default_rng([800, B, qg, T])
    P = 40 if n_kv == 1 else 4
    kq, vq = (r.integers(0, 256, (P, n_kv, 1, BLOCK)).astype(np.uint8) for _ in range(2))
    for x in (kq, vq):
        sm = r.integers(0x3F00, 0x4000, (P, n_kv, 1, 256)).astype(np.uint16)
        x[..., 4096::2], x[..., 4097::2] = sm & 255, sm >> 8
    new = np.ones(B, np.int32)
    new[:: max(3, B // 100)] = T
    N, n_q = int(new.sum()), n_kv * qg
    start = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
    table = r.integers(0, P, (B, 1)).astype(np.int32)
    q = r.integers(0x3F00, 0x4000, (N, n_q, HD)).astype(np.uint16)
    byte, shift, s_at, m_at = (x[0] for x in V_AT)
    blk = vq[:, :, 0]
    word = lambda at: f64(blk[..., at].astype(np.uint16) | (blk[..., at + 1].astype(np.uint16) << 8))  # noqa: E731
    row = word(m_at) + word(s_at) * ((blk[..., byte] >> shift.astype(np.uint8)) & 15)                    # [P][n_kv][256]
    for out_bf16 in (True, False):
        up = dict(k=kq, v=vq, table=table, len=np.ones(B, np.int32), start=start, q=q,
                  out=np.full((N, n_q, HD), 0x7FA5, np.uint16) if out_bf16 else np.full((N, n_q, HD), -777.25, np.float32))
        buf = {n: ctx.put(x) for n, x in up.items()}
        d = L.PagedAttnDesc(B=B, n_q=n_q, n_kv=n_kv, hd=HD, page_size=32, n_pages=P, max_pages=1, n_tok=N, max_T=T)
        d.table, d.len, d.q_start, d.q, d.k_pages, d.v_pages, d.out = (buf[x].ptr for x in ("table", "len", "start", "q", "k", "v", "out"))
        d.out_dtype = L.BF16 if out_bf16 else L.F32
        L.check(L.lib().vx27_hip_paged_attn_q4(ctx.h, C.byref(d)), "paged_attn_q4")
        ctx.sync()
        want = np.zeros((N, n_kv, HD))
        want[start[1:] - 1] = row[table[:, 0]]
        got = buf["out"].download(up["out"].shape, up["out"].dtype).reshape(N, n_kv, qg, HD)
        last = np.zeros(N, bool)
        last[start[1:] - 1] = True
        assert not got[~last].any()
        # one weight of 1: s and m rounded by it (2^-8, or two parts' 2^-16), and the output's rounding
        err = np.abs((f64(got) if out_bf16 else got.astype(np.float64))[last] - want[last][:, :, None])
        assert np.all(err <= (2.0 ** -7 if out_bf16 or T * qg > L.Q4_SPLIT_ROWS_F32 else 2.0 ** -15) * want[last][:, :, None])
        for x in buf.values():
            x.free()


def test_values_next_to_a_border(ctx):  # noqa: F811
    """Values a few last places of fp32 from where the code changes, where an fp32 quotient cannot tell, on both sides."""
    say("values next to a border")
    r = np.random.default_rng(1700)
    rows = []
    for scale, off in ((1.0, 0.0), (0.0390625, -3.0), (1.5e-3, 0.75), (3.0, 1e4), (2.0 ** -90, 0.0), (2.0 ** 100, 0.0), (7.0, -300.0)):
        for step in (0, 1, 2, 3, 8):
            x = (off + scale * (r.integers(0, 15, HD) + 0.5)).astype(np.float32)
            for _ in range(step):
                x = np.nextafter(x, np.where(r.random(HD) < 0.5, -np.inf, np.inf).astype(np.float32))
            x[::64], x[1::64] = np.float32(off), np.float32(off + 15 * scale)
            rows.append(x)
    rows = np.array(rows, np.float32)[:, None]
    got = append_v(ctx, rows)[1]
    c, s, m = quantise(rows[:, 0].astype(np.float64))
    for i in range(len(rows)):
        gc, gs, gm = get(got[i // 32], V_AT, i % 32)
        assert np.array_equal(gs, s[i]) and np.array_equal(gc, c[i]), i
        assert np.all((gm == m[i]) | ((gm | m[i]) & 0x7FFF == 0)), i


@pytest.mark.parametrize("out_bf16", [False, True])
@pytest.mark.parametrize("first,n", [(0, 64), (3, 61), (8, 17), (5, 8), (24, 300), (31, 9), (0, 7)])
def test_rows_in_order(ctx, first, n, out_bf16):  # noqa: F811
    """Rows of a sequence in order, from any row on: eight that share a block's units, and others, and one left out."""
    from vx27_amd import lib as L, workloads as W
    say(f"rows {first} .. {first + n - 1} in order")
    bt = Batch4([350], [350], 4, 4, 64, seed=1800 + first)
    rows = np.arange(first, first + n)
    slots = (bt.table[0, rows // 64] * 64 + rows % 64).astype(np.int32)
    slots[n // 2] = -1
    e = 2 if out_bf16 else 4
    buf = dict(k=ctx.put(bt.kq), v=ctx.put(bt.vq), slots=ctx.put(slots), ko=ctx.put(np.full((n + 1) * 4 * HD * e, 0x5A, np.uint8)),
               vo=ctx.put(np.full((n + 1) * 4 * HD * e, 0x5A, np.uint8)))
    d = L.PagedReadDesc(n_kv=4, hd=HD, page_size=64, n_pages=bt.n_pages, n_rows=n, slots=buf["slots"].ptr, k_pages=buf["k"].ptr,
                        v_pages=buf["v"].ptr, out_dtype=L.BF16 if out_bf16 else L.F32, k_out=buf["ko"].ptr, v_out=buf["vo"].ptr)
    L.check(L.lib().vx27_hip_paged_read_q4(ctx.h, C.byref(d)), "paged_read_q4")
    ctx.sync()
    for name, held in zip(("ko", "vo"), bt.held(0)):
        raw = buf[name].download((n + 1, 4, HD * e), np.uint8)
        assert np.all(raw[n // 2] == 0x5A) and np.all(raw[n] == 0x5A)
        got = np.frombuffer(raw.tobytes(), np.uint16 if out_bf16 else np.float32).reshape(n + 1, 4, HD)[:n]
        want = values(*(x[first:first + n] for x in held)).astype(np.float32)
        ok = slots >= 0
        assert np.array_equal(got[ok], (W.bf16_bits(want) if out_bf16 else want)[ok]), name
    for x in buf.values():
        x.free()


# ------------------------------------------------------------------- faults
def test_nothing_to_do(ctx):  # noqa: F811
    from vx27_amd import lib as L
    say("nothing to do")
    a = Attn4(ctx, Batch4([200, 100], [1, 1], seed=27))
    a.d.n_tok = a.d.max_T = 0
    a.call()
    P = a.bufs["out"].ptr
    L.check(L.lib().vx27_hip_paged_read_q4(ctx.h, C.byref(L.PagedReadDesc(n_kv=4, hd=HD, page_size=32, n_pages=1, slots=P, k_pages=P, v_pages=P,
                                                                           k_out=P, v_out=P))))
    ctx.sync()
    assert np.array_equal(a.bufs["out"].download(a.sentinel.shape, a.sentinel.dtype), a.sentinel)
    a.free()


@pytest.mark.parametrize("lens,new", [([200, 100], [1, 1]), ([200, 100], [40, 2]), ([200, 100], [150, 2])])
@pytest.mark.parametrize("what", ["page", "negative page", "length", "start", "long"])
def test_bad_indices_are_reported(ctx, lens, new, what):  # noqa: F811
    """Tables, lengths and token ranges outside their buffers: no access leaves them (the clamps are those of
    test_paged_host.py), the next sync reports it and the context goes on."""
    from vx27_amd import lib as L
    say(f"faulty {what} {new}")
    bt = Batch4(list(lens), new, seed=26)
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
        bt.start[:] = [0, bt.N, bt.N]
    for out_bf16 in (False, True):
        a = Attn4(ctx, bt, out_bf16, gate="none")
        a.call()
        with pytest.raises(L.HipError, match="paged cache"):
            ctx.sync()
        a.free()
    bt.table, bt.lens, bt.start = good
    a = Attn4(ctx, bt, gate="none")
    a.call()
    a.check("after the report")
    a.free()


@pytest.mark.parametrize("what", ["page", "length", "rows"])
def test_faulty_appends_are_reported(ctx, what):  # noqa: F811
    """Pages outside the pool, lengths past the table, tokens without a row: nothing outside the pages is written."""
    from vx27_amd import lib as L
    say(f"faulty append: {what}")
    r = np.random.default_rng(1900)
    guard = np.full(BLOCK, 0xA7, np.uint8)
    pages = r.integers(0, 256, (3, 1, 1, BLOCK)).astype(np.uint8)
    whole = np.concatenate([guard, pages.ravel(), guard])
    buf = dict(k=ctx.put(whole), v=ctx.put(whole), kn=ctx.put(np.ones((6, 1, HD), np.float32)), w=ctx.put(np.zeros(HD, np.float32)),
               t=ctx.put(np.array([[0, 3 if what == "page" else 1], [2, 2]], np.int32)),
               len=ctx.put(np.array([65 if what == "length" else 34, 1 if what == "rows" else 40], np.int32)), start=ctx.put(np.array([0, 3, 6], np.int32)))
    d = L.PagedAppendDesc(B=2, n_q=1, n_kv=1, hd=HD, rope_theta=1e7, rope_yarn=1.0, page_size=32, n_pages=3, max_pages=2, n_tok=6, max_T=3)
    d.table, d.len, d.q_start, d.k_new, d.v_new, d.k_norm_w = (buf[x].ptr for x in ("t", "len", "start", "kn", "kn", "w"))
    d.k_pages, d.v_pages = buf["k"].ptr + BLOCK, buf["v"].ptr + BLOCK
    L.check(L.lib().vx27_hip_paged_append_q4(ctx.h, C.byref(d)), "paged_append_q4")
    with pytest.raises(L.HipError, match="paged cache"):
        ctx.sync()
    for name in ("k", "v"):
        got = buf[name].download(whole.shape, np.uint8)
        assert np.array_equal(got[:BLOCK], guard) and np.array_equal(got[-BLOCK:], guard)
    for x in buf.values():
        x.free()


@pytest.mark.parametrize("bad", [-2, 3 * 64, 2 ** 31 - 1, -2 ** 31])
def test_faulty_slots_are_reported(ctx, bad):  # noqa: F811
    """A slot outside the pool leaves its row of the output as it was; the others are read."""
    from vx27_amd import lib as L
    say(f"faulty slot {bad}")
    bt = Batch4([150], [150], 2, 2, 64, seed=1950)
    assert bt.n_pages >= 3
    rows = np.arange(40)
    slots = (bt.table[0, rows // 64] * 64 + rows % 64).astype(np.int32)
    slots[[3, 17]] = bad
    buf = dict(k=ctx.put(bt.kq), v=ctx.put(bt.vq), slots=ctx.put(slots), ko=ctx.put(np.full((40, 2, HD), -7.5, np.float32)),
               vo=ctx.put(np.full((40, 2, HD), -7.5, np.float32)))
    d = L.PagedReadDesc(n_kv=2, hd=HD, page_size=64, n_pages=3, n_rows=40, slots=buf["slots"].ptr, k_pages=buf["k"].ptr, v_pages=buf["v"].ptr,
                        k_out=buf["ko"].ptr, v_out=buf["vo"].ptr)
    L.check(L.lib().vx27_hip_paged_read_q4(ctx.h, C.byref(d)), "paged_read_q4")
    with pytest.raises(L.HipError, match="paged cache"):
        ctx.sync()
    inside = slots // 64 < 3
    for name, held in zip(("ko", "vo"), bt.held(0)):
        got = buf[name].download((40, 2, HD), np.float32)
        want = values(*(x[:40] for x in held)).astype(np.float32)
        ok = (slots >= 0) & inside
        assert np.array_equal(got[ok], want[ok]) and np.all(got[~ok] == -7.5)
    for x in buf.values():
        x.free()


@pytest.mark.parametrize("B,few,ended", [(1500, 0.97, True), (4096, 0.99, True), (5000, 0.5, False), (65535, 0.9, True), (1025, 0.0, True)])
def test_plans_of_many_sequences(ctx, B, few, ended):  # noqa: F811
    """Long runs of sequences without tokens or pages between those that have some; more tokens than one launch takes."""
    from test_gpu_paged_plan import Plan
    say(f"plan of {B} sequences, {few} of them idle")
    r = np.random.default_rng([1960, B])
    page = 32
    idle = r.random(B) < few
    lens = np.where(r.random(B) < 0.3, 0, r.integers(0, 100, B))
    new = np.where(idle, 0, r.integers(0, 90, B))
    e = (r.random(B) < 0.3).astype(int) if ended else None
    need = int((-(-(lens + new) // page) - -(-lens // page)).sum())
    table, free, n_free = pool(r, lens, page, need // 2, 7)
    n_tok = int(new.sum()) + 5000
    want = plan(lens, new, table, free, n_free, page, n_tok, e, lens + 3)
    p = Plan(ctx, lens, new, table, free, n_free, page, n_tok, e, lens + 3)
    p.call()
    ctx.sync()
    p.check(want)
    p.free()


def widen(bt, pages=2100):
    """The batch with a page table of many more entries, behind the rows: the same rows, and a call that may see more."""
    bt.table = np.concatenate([bt.table, np.full((bt.B, pages), -7, np.int32)], axis=1)
    bt.max_pages += pages
    return bt


@pytest.mark.parametrize("out_bf16", [False, True])
@pytest.mark.parametrize("i", [i for i, s in enumerate(SHAPES) if max(s[1]) * s[2] // s[3] > 96])
def test_prompts_under_wide_tables(ctx, i, out_bf16):  # noqa: F811
    """Prompts of few rows whose tables have room for many: the tile kernel (small calls run the decode kernels)."""
    lens, new, n_q, n_kv, page, window, sink = SHAPES[i]
    say(f"wide tables {i} {lens} {new} bf16 {out_bf16}")
    at = Attn4(ctx, widen(Batch4(lens, new, n_q, n_kv, page, window, sink, seed=900 + i, lead=2, tail=3)), out_bf16, gate=("f32", "bf16", "none")[i % 3])
    at.call()
    at.check(f"{i}")
    at.free()


@pytest.mark.parametrize("lens,new,window,sink", [([90, 33], [60, 33], 0, 0), ([400, 90], [130, 90], 50, 4), ([1500, 10], [40, 3], 0, 0)])
@pytest.mark.parametrize("what", ["k", "v"])
def test_nan_groups_under_wide_tables(ctx, lens, new, window, sink, what):  # noqa: F811
    """A group held as NaN in the tile kernel: NaN where a token sees it, and nowhere else."""
    say(f"nan groups, wide tables {what} {lens} {new}")
    bt = widen(Batch4(lens, new, 24, 4, 64, window, sink, seed=650 + new[0]))
    seen, j = bt.seen(0), None
    part = np.nonzero(seen.any(0) & ~seen.all(0))[0]
    q, where = (bt.kq, K_AT) if what == "k" else (bt.vq, V_AT)
    clean, hit = q.copy(), np.zeros((bt.N, 24, HD), bool)
    for i, j in enumerate((part[0], part[len(part) // 2], part[-1])):
        p, at, g = bt.table[0, j // 64], j % 64, i % 4
        c, s, m = (x.copy() for x in get(q[p, 1, at // 32], where, at % 32))
        c[64 * g:64 * g + 64], s[g], m[g] = 0, 0, 0x7FC0
        put(q[p, 1, at // 32], where, at % 32, c, s, m)
        m[g] = 0
        put(clean[p, 1, at // 32], where, at % 32, c, s, m)
        hit[np.ix_(bt.start[0] + np.nonzero(seen[:, j])[0], range(6, 12), range(HD) if what == "k" else range(64 * g, 64 * g + 64))] = True
    at = Attn4(ctx, bt, True, gate="none")
    assert at.tiled()
    at.call()
    ctx.sync()
    out = at.out()
    if what == "k":
        bt.kq = clean
    else:
        bt.vq = clean
    ref = bt.result(False)
    assert np.isnan(out[hit]).all()
    assert np.all(np.abs(out[~hit] - ref["out"][~hit]) <= at.tol(ref, max(lens))[~hit])
    at.free()


@pytest.mark.parametrize("what", ["page", "negative page", "length", "start", "long"])
def test_bad_indices_under_wide_tables(ctx, what):  # noqa: F811
    """The tile kernel's faulty tables, as test_bad_indices_are_reported."""
    from vx27_amd import lib as L
    say(f"faulty {what}, wide tables")
    bt = widen(Batch4([200, 100], [150, 2], seed=26))
    if what == "page":
        bt.table[1, 0] = bt.n_pages
    if what == "negative page":
        bt.table[1, 0] = -1
    if what == "length":
        bt.lens[0] = bt.max_pages * bt.page + 1
    if what == "start":
        bt.start[2] = bt.N + 1
    if what == "long":
        bt.start[:] = [0, bt.N, bt.N]
    a = Attn4(ctx, bt, True, gate="none")
    a.call()
    with pytest.raises(L.HipError, match="paged cache"):
        ctx.sync()
    a.free()


def test_graphs_under_wide_tables():
    """Tiles, and tiles over values laid out in scratch, captured with a decode call on one workspace."""
    from vx27_amd import lib as L
    say("graphs, wide tables")
    with L.Ctx(0) as c:
        ats = [Attn4(c, widen(Batch4([800, 64], [30, 64], seed=22), 100), True), Attn4(c, widen(Batch4([800, 64], [300, 64], seed=23), 100), True),
               Attn4(c, Batch4([1500, 90, 700], [1, 1, 1], seed=21))]
        want, graphs = [], []
        for x in ats:
            x.call()
            c.sync()
            want.append(x.raw())
        for x in ats:
            c.graph_begin()
            x.call()
            graphs.append(c.graph_end())
        try:
            for rep in range(4):
                for x, g, w in zip(ats, graphs, want):
                    c.graph_launch(g)
                    c.sync()
                    assert all(np.array_equal(p, q) for p, q in zip(x.raw(), w)), rep
                for x, w in zip(ats, want):
                    x.call()
                    c.sync()
                    assert all(np.array_equal(p, q) for p, q in zip(x.raw(), w)), rep
        finally:
            for g in graphs:
                L.check(L.lib().vx27_hip_graph_destroy(g), "graph_destroy")
