"""The paged-cache operators where values and sizes are extreme."""
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
