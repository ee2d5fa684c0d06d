"""The 4-bit paged attention's outputs within what each of its kernels rounds:
every shape by the kernel that runs it (asked of the library's profiler), whole
servers, rows untouched by NaN, and pieces of many steps."""
import numpy as np
import pytest

import q4_bounds as Q
import test_gpu_paged_q4_use as U
from gpu_common import say
from paged_common import HD, f64
from q4_bounds import KERNELS, kernel_of, run, widen
from q4_common import K_AT, V_AT, Batch4, get, put
from test_gpu_paged_q4 import SHAPES, Attn4, ctx  # noqa: F401

pytestmark = pytest.mark.gpu


def within(at, res, kernel, tag):
    """The outputs and lse of the call's tokens."""
    at.ctx.sync()
    bt = at.bt
    lo, hi, keys = bt.start[0], bt.start[-1], max(max(bt.lens), 1)
    most, mean = Q.check(at.out()[lo:hi], Q.cut(res, lo, hi), kernel, keys, at.out_bf16)
    say(f"  {tag} {kernel}: err {most:.3f} of its bound, mean {mean:.3f}")
    assert most <= 1 and mean <= 1, tag
    lse, want, tol = (x[lo:hi] for x in (at.lse(), res["lse"], Q.lse_tol(res, keys)))
    f = np.isfinite(want)
    assert np.array_equal(np.isinf(lse), ~f) and np.all(np.abs(lse[f] - want[f]) <= tol[f]), tag


@pytest.mark.parametrize("i", range(len(SHAPES)))
def test_attention(ctx, i):  # noqa: F811
    lens, new, n_q, n_kv, page, window, sink = SHAPES[i]
    say(f"q4 attn bounds {i} {lens[:6]} {new[:6]} heads {n_q}/{n_kv} page {page} window {window} sink {sink}")
    refs, bt = {}, Batch4(lens, new, n_q, n_kv, page, window, sink, seed=900 + i, lead=2, tail=3)
    for wide in (False, True):
        if wide:
            widen(bt)
        for out_bf16 in (False, True):
            at = Attn4(ctx, bt, out_bf16, gate=("f32", "none")[i % 2])
            kernel = run(at)
            assert kernel == kernel_of(bt, out_bf16)
            if kernel not in refs:
                refs[kernel] = Q.result(bt, kernel, at.gated)
            within(at, refs[kernel], kernel, f"{i} wide {wide} bf16 {out_bf16}")
            at.free()


class Server(U.Server):
    """One whose outputs are held to the kernel's own bound."""

    def call(self):
        self.ctx.prof_enable(True)
        super().call()
        self.ran = [k for k in KERNELS if self.ctx.prof_read(k)[0]]
        self.ctx.prof_enable(False)

    def check(self):
        super().check()
        w, N, (kernel,) = self.want, self.N, self.ran
        if not N:
            return
        bt = Batch4.__new__(Batch4)
        bt.lens, bt.new, bt.n_q, bt.n_kv, bt.qg, bt.window, bt.sink = list(w["len_out"]), list(w["took"]), 24, 4, 6, self.window, self.sink
        bt.B, bt.N, bt.start, bt.gate = self.B, N, w["q_start"], self.qg[:N, :, HD:]
        bt.held = lambda b: [[np.stack([r[at + i] for r in self.rows[b]]) for i in range(3)] for at in (0, 3)]
        res = Q.result(bt, kernel, q=f64(self.buf["q"].download((self.room, 24, HD), np.uint16)[:N]))
        got = self.buf["out"].download(self.sentinel.shape, self.sentinel.dtype)[:N]
        most, mean = Q.check(f64(got) if self.out_bf16 else got.astype(np.float64), res, kernel, max(bt.lens), self.out_bf16)
        assert most <= 1 and mean <= 1, (kernel, most, mean)
        self.kernels = getattr(self, "kernels", set()) | {kernel}


@pytest.mark.parametrize("window,sink,page,width,kernels", [(0, 0, 64, 640, {"paged_rows_q4", "paged_rows_flat"}), (70, 4, 32, 640, {"paged_rows_q4", "paged_rows_flat"}),
                                                            (0, 0, 64, 64 * 1024, {"paged_rows_q4"})])
def test_a_server(ctx, window, sink, page, width, kernels):  # noqa: F811
    """Prompts, decoding and drafted tokens, under narrow tables and wide ones."""
    say(f"a server within its bounds, window {window}, room for {width} rows")
    s = Server(ctx, 5, 1024 // page, page, width // page, window, sink, 400, 1350 + window, True)
    for new, over in [([130, 0, 5, 64, 33], 0), ([1] * 5, 0), ([1, 7, 1, 3, 1], 0), ([90, 1, 40, 1, 0], 0b00010), ([1] * 5, 0b11000),
                      ([60, 40, 70, 80, 9], 0), ([11, 1, 2, 1, 1], 0)]:
        s.most(max(max(new), 1))
        s.give(new, [over >> b & 1 for b in range(5)])
        s.call()
        s.check()
    assert s.kernels == kernels | {"paged_q4_split"}
    s.free()


@pytest.mark.parametrize("kernel,lens,new,window,sink", [
    ("paged_q4_split", [300, 90], [7, 3], 0, 0), ("paged_q4_split", [300, 70], [2, 1], 33, 4), ("paged_rows_q4", [900, 400, 300], [100, 100, 100], 50, 4),
    ("paged_rows_q4", [3000, 10], [40, 3], 0, 0), ("paged_rows_flat", [400, 90], [130, 90], 50, 4), ("paged_rows_flat", [900, 90], [130, 90], 0, 0)])
@pytest.mark.parametrize("what", ["k", "v"])
def test_nan_groups_leave_other_rows_alone(ctx, kernel, lens, new, window, sink, what):  # noqa: F811
    """A group held as NaN at rows that some tokens see: NaN there, and every other output bit for bit as without it."""
    say(f"nan groups {what} {kernel} {lens} {new}")
    bt = Batch4(lens, new, 24, 4, 64, window, sink, seed=660 + new[0])
    seen = bt.seen(0)
    part = np.nonzero(seen.any(0) & ~seen.all(0))[0]
    clean = Attn4(ctx, bt, True, gate="none")
    assert run(clean) == kernel
    ctx.sync()
    want, hit = clean.out(), np.zeros((bt.N, 24, HD), bool)
    q, where = (bt.kq, K_AT) if what == "k" else (bt.vq, V_AT)
    for i, j in enumerate((part[0], part[len(part) // 2], part[-1])):
        p, at, g = bt.table[0, j // 64], j % 64, i % 4
        c, s, m = (x.copy() for x in get(q[p, 1, at // 32], where, at % 32))
        c[64 * g:64 * g + 64], s[g], m[g] = 0, 0, 0x7FC0
        put(q[p, 1, at // 32], where, at % 32, c, s, m)
        hit[np.ix_(bt.start[0] + np.nonzero(seen[:, j])[0], range(6, 12), range(HD) if what == "k" else range(64 * g, 64 * g + 64))] = True
    at = Attn4(ctx, bt, True, gate="none")
    assert run(at) == kernel
    ctx.sync()
    out = at.out()
    assert np.isnan(out[hit]).all() and np.array_equal(out[~hit], want[~hit])
    clean.free()
    at.free()
