"""The paged-cache operators at the numbers they allow, in graphs whose tables
change between replays, and in two threads at once."""
import ctypes as C
import threading

import numpy as np
import pytest

from gpu_common import say
from paged_common import HD
from test_gpu_paged import ctx  # noqa: F401
from test_gpu_paged_values import Step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,n_kv,qg", [(65535, 1, 1), (65535, 1, 16), (3, 1024, 1), (3, 1024, 16)])
@pytest.mark.parametrize("two", [False, True])
def test_most_sequences_and_heads(ctx, B, n_kv, qg, two):  # noqa: F811
    """As many sequences, or KV heads, as the calls take: a sequence of one row gives that row's value (its weight is 1);
    with `two` a 16-head group makes 32 rows of some sequences, which see nothing from their first token."""
    from vx27_amd import lib as L
    say(f"B={B} n_kv={n_kv} group {qg} two={two}")
    r = np.random.default_rng([800, B, qg, two])
    pool = 40 if n_kv == 1 else 4
    v = r.integers(0x3F00, 0x4000, (pool, n_kv, 1, HD, 32)).astype(np.uint16)
    k = r.integers(0x3F00, 0x4000, (pool, n_kv, 32, HD)).astype(np.uint16)
    new = np.ones(B, np.int32)
    if two:
        new[::3] = 2
    N, n_q = int(new.sum()), n_kv * qg
    start = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
    table = r.integers(0, pool - 1, (B, 1)).astype(np.int32)
    q = r.integers(0x3F00, 0x4000, (N, n_q, HD)).astype(np.uint16)
    up = dict(k=k, v=v, table=table, len=np.ones(B, np.int32), start=start, q=q, out=np.full((N, n_q, HD), 0x7FA5, np.uint16),
              acc=np.zeros((B, n_kv, 32), np.float32))
    buf = {n: ctx.put(x) for n, x in up.items()}
    d = L.PagedAttnDesc()
    d.B, d.n_q, d.n_kv, d.hd, d.page_size, d.n_pages, d.max_pages = B, n_q, n_kv, HD, 32, pool, 1
    d.table, d.len, d.q_start, d.n_tok, d.max_T = buf["table"].ptr, buf["len"].ptr, buf["start"].ptr, N, int(new.max())
    d.q, d.k_pages, d.v_pages, d.out, d.out_dtype = buf["q"].ptr, buf["k"].ptr, buf["v"].ptr, buf["out"].ptr, L.BF16
    d.acc, d.acc_stride = buf["acc"].ptr, 32
    L.check(L.lib().vx27_hip_paged_attn(ctx.h, C.byref(d)), "paged_attn")
    ctx.sync()
    want = np.zeros((N, n_kv, qg, HD), np.uint16)
    want[start[1:] - 1] = v[table[:, 0], :, 0, :, 0][:, :, None]
    assert np.array_equal(buf["out"].download((N, n_kv, qg, HD), np.uint16), want)
    acc = buf["acc"].download((B, n_kv, 32), np.float32)
    # (a weight and the division by their sum: 2^-20 as elsewhere)
    assert np.all(np.abs(acc[..., 0] - qg) <= qg * 2.0 ** -20) and not acc[..., 1:].any()
    if qg == 1 and not two:      # append and eviction: k is what is normed; v is copied
        ones = np.ones(HD, np.float32)
        vn = r.integers(0x3F00, 0x4000, (B, n_kv, HD)).astype(np.uint16)
        if B <= pool:
            table = np.arange(B, dtype=np.int32)[:, None]
            tb, vb, wb = ctx.put(table), ctx.put(vn), ctx.put(ones)
            p = L.PagedAppendDesc()
            p.B, p.n_q, p.n_kv, p.hd, p.page_size, p.n_pages, p.max_pages = B, n_q, n_kv, HD, 32, pool, 1
            p.table, p.len, p.n_tok, p.max_T, p.in_dtype = tb.ptr, buf["len"].ptr, B, 1, L.BF16
            p.k_new, p.v_new, p.k_norm_w, p.k_pages, p.v_pages = vb.ptr, vb.ptr, wb.ptr, buf["k"].ptr, buf["v"].ptr
            L.check(L.lib().vx27_hip_paged_append(ctx.h, C.byref(p)), "paged_append")
            ctx.sync()
            v[:B, :, 0, :, 0] = vn
            assert np.array_equal(buf["v"].download(v.shape, np.uint16), v)
            for x in (tb, vb, wb):
                x.free()
        e = L.PagedEvictDesc()
        fresh = ctx.put(np.full((B, 1), pool - 1, np.int32))
        dl, kept = ctx.put(np.full(B, -1, np.int32)), ctx.put(np.full((B, n_kv, 1), -1, np.int32))
        zero = ctx.put(np.where(np.arange(B) == B - 1, 1, 0).astype(np.int32))      # the last sequence has a row
        e.B, e.n_kv, e.hd, e.page_size, e.n_pages, e.max_pages = B, n_kv, HD, 32, pool, 1
        e.table, e.len, e.budget, e.acc, e.acc_stride = buf["table"].ptr, zero.ptr, 1, buf["acc"].ptr, 32
        e.k_pages, e.v_pages, e.dst_table, e.dst_max_pages, e.dst_len, e.kept = (buf["k"].ptr, buf["v"].ptr, fresh.ptr, 1, dl.ptr, kept.ptr)
        L.check(L.lib().vx27_hip_paged_evict(ctx.h, C.byref(e)), "paged_evict")
        ctx.sync()
        src = up["table"][B - 1, 0]
        v[pool - 1, :, 0, :, 0] = v[src, :, 0, :, 0]
        assert np.array_equal(buf["v"].download(v.shape, np.uint16), v)
        n, kp = dl.download((B,), np.int32), kept.download((B, n_kv), np.int32)
        assert not n[:-1].any() and n[-1] == 1 and np.all(kp[:-1] == -1) and np.all(kp[-1] == 0)
        for x in (fresh, dl, kept, zero):
            x.free()
    for x in buf.values():
        x.free()


@pytest.mark.parametrize("a,b", [
    (([300, 95, 200], [1, 1, 1]), ([95, 200, 300], [1, 1, 1])),
    (([300, 95, 200], [2, 0, 1]), ([200, 300, 95], [1, 2, 0])),
    (([300, 95, 200], [130, 1, 9]), ([200, 300, 95], [9, 130, 1])),
    (([40 + i for i in range(70)], [1] * 70), ([109 - i for i in range(70)], [1] * 70)),
])
def test_a_captured_step_follows_its_tables(a, b):
    """Append, attention with weights and eviction captured for one batch: after the tables, lengths and token ranges on
    the device become another batch's, a replay gives that batch's bytes; and the first one's once they are back."""
    from vx27_amd import lib as L
    say(f"tables change {a[0][:3]} {a[1][:3]}")
    with L.Ctx(0) as c:
        s, t = Step(c, *a), Step(c, *b)
        assert s.k.shape == t.k.shape and s.bt.table.shape == t.bt.table.shape and s.bt.N == t.bt.N
        want = []
        for x in (s, t):
            x.reset()
            x.call()
            want.append(x.results())
        names = ("table", "len", "start", "dst", "w")
        const = [{n: x.buf[n].download((x.buf[n].nbytes,), np.uint8) for n in names} for x in (s, t)]
        c.graph_begin()
        s.call()
        g = c.graph_end()
        try:
            for rep in range(4):
                x = (s, t)[rep % 2]
                for n, y in const[rep % 2].items():
                    s.buf[n].upload(y)
                s.h2d("k", x.k)
                s.h2d("v", x.v)
                for n, y in {**x.up, **x.outs}.items():
                    s.buf[n].upload(y)
                c.graph_launch(g)
                assert all(np.array_equal(p, q) for p, q in zip(s.results(), want[rep % 2])), rep
        finally:
            L.check(L.lib().vx27_hip_graph_destroy(g), "graph_destroy")


def test_two_threads_at_once():
    """Two contexts, each with its own thread, stream, tables and workspace: every step gives its own bytes."""
    from vx27_amd import lib as L
    shapes = [([300, 95, 200], [130, 1, 9]), ([700, 45], [1, 2])]
    bad = []

    def work(c, s, want):
        for i in range(20):
            s.reset()
            s.call()
            if not all(np.array_equal(x, y) for x, y in zip(s.results(), want)):
                bad.append((s.bt.lens, i))

    ctxs = [L.Ctx(0) for _ in shapes]
    try:
        jobs = []
        for c, x in zip(ctxs, shapes):
            s = Step(c, *x)
            s.reset()
            s.call()
            jobs.append((c, s, s.results()))
        threads = [threading.Thread(target=work, args=j) for j in jobs]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert not bad
    finally:
        for c in ctxs:
            c.close()
