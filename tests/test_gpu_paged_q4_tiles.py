"""The tile kernel over 4-bit pages where it decodes them itself, and both its
forms in pieces of many steps."""
import numpy as np
import pytest

import q4_bounds as Q
import test_gpu_paged_q4_use as U
from gpu_common import say
from paged_common import HD
from q4_bounds import kernel_of, run
from q4_common import Batch4
from test_gpu_paged_q4 import Attn4, ctx  # noqa: F401
from vx27_amd import workloads as W

pytestmark = pytest.mark.gpu

# prompts of few row tiles whose sequences have many tiles
TILES = ([3000, 95, 200], [60, 1, 9])


def ran(ctx):  # noqa: F811
    s = U.Step4(ctx, *TILES)
    s.reset()
    s.ctx.prof_enable(True)
    s.call()
    k = [k for k in Q.KERNELS if s.ctx.prof_read(k)[0]]
    s.ctx.prof_enable(False)
    s.results()
    s.free()
    return k


def test_pages_past_2_to_32_bytes(ctx):  # noqa: F811
    assert ran(ctx) == ["paged_rows_q4"]
    U.test_pages_past_2_to_32_bytes(ctx, *TILES)


def test_inputs_that_are_late_on_the_callers_stream(ctx):  # noqa: F811
    assert ran(ctx) == ["paged_rows_q4"]
    U.test_inputs_that_are_late_on_the_callers_stream(ctx, *TILES)


@pytest.mark.parametrize("kernel,lens,new", [("paged_rows_q4", [3000, 100], [40, 2]), ("paged_rows_flat", [900, 100], [150, 2]),
                                             ("paged_q4_split", [200, 100], [40, 2])])
@pytest.mark.parametrize("what", ["page", "negative page", "length", "start", "long"])
def test_bad_indices(ctx, kernel, lens, new, what):  # noqa: F811
    """As test_bad_indices_are_reported, by the kernels named."""
    from vx27_amd import lib as L
    bt = Batch4(lens, new, seed=26)
    assert kernel_of(bt, True) == kernel
    say(f"faulty {what}, {kernel}")
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
    a = Attn4(ctx, bt, True, gate="none")
    a.call()
    with pytest.raises(L.HipError, match="paged cache"):
        ctx.sync()
    a.free()
    bt.table, bt.lens, bt.start = good
    a = Attn4(ctx, bt, True, gate="none")
    assert run(a) == kernel
    ctx.sync()
    res = Q.result(bt, kernel, False)
    most, mean = Q.check(a.out(), res, kernel, max(lens), True)
    assert most <= 1 and mean <= 1
    a.free()


def pieces(steps, cus):
    """Steps of the longest piece that items of so many steps are cut into (paged_plan's rule)."""
    n = len(steps)
    room = (n + cus // 2 + cus - 1) // cus * cus - n
    limit = max(-(-sum(steps) // room), 4)
    parts = [-(-s // limit) for s in steps]
    return max(-(-s // p) for s, p in zip(steps, parts)), max(parts)


class Many(Attn4):
    """`seqs` sequences that all read one conversation's rows, the last T of each their own queries."""

    def __init__(self, ctx, rows, seqs, T, window, sink, seed, out_bf16=True):
        src = Batch4([rows], [rows], 16, 1, 256, seed=seed)
        bt = Batch4.__new__(Batch4)
        r = src.r
        bt.lens = [rows - 5 * (b % 7) for b in range(seqs)]
        bt.new, bt.n_q, bt.n_kv, bt.qg, bt.page, bt.window, bt.sink, bt.B = [T] * seqs, 16, 1, 16, 256, window, sink, seqs
        bt.start, bt.N = (T * np.arange(seqs + 1)).astype(np.int32), T * seqs
        bt.kq, bt.vq, bt.n_pages, bt.max_pages = src.kq, src.vq, src.n_pages, src.max_pages
        bt.table = np.repeat(src.table, seqs, axis=0)
        bt.q, bt.gate = W.bf16_bits(W.normal(r, (bt.N, 16, HD), 2.0)), None
        held = src.held(0)
        bt.held = lambda b: [[x[:bt.lens[b]] for x in part] for part in held]
        super().__init__(ctx, bt, out_bf16, gate="none")


@pytest.mark.parametrize("kernel,rows,seqs,T,window,sink", [
    ("paged_rows_q4", 6400, 128, 7, 0, 0),             # one row tile a sequence, 100 steps
    ("paged_rows_q4", 9000, 90, 8, 0, 0),              # 140 steps, cut in two
    ("paged_rows_q4", 9000, 128, 8, 4500, 40),         # a window's edge and sinks
    ("paged_rows_flat", 6400, 16, 64, 0, 0),           # eight row tiles a sequence
    ("paged_rows_flat", 5000, 16, 64, 4500, 70)])
def test_pieces_of_many_steps(ctx, kernel, rows, seqs, T, window, sink):  # noqa: F811
    """Pieces of more than 64 steps, whose blocks' addresses are looked up again and again: every token of some sequences
    against float64, the others (the same rows) by their own."""
    say(f"pieces of many steps: {kernel} {seqs} x {rows} rows, {T} tokens, window {window}")
    at = Many(ctx, rows, seqs, T, window, sink, 2000 + seqs)
    bt = at.bt
    assert kernel_of(bt, True) == kernel
    seen = min(rows, window + sink) if window else rows
    longest, parts = pieces([seen // 64] * (seqs * -(-T * 16 // 128)), 256)
    assert longest > 64, (longest, parts)
    assert run(at) == kernel
    ctx.sync()
    tokens = np.zeros(bt.N, bool)
    for b in range(0, seqs, 17 if T < 40 else 7):
        tokens[bt.start[b]:bt.start[b + 1]] = True
    res, out = Q.result(bt, kernel, False, tokens=tokens), at.out()
    most, mean = Q.check(out[tokens], {n: x[tokens] for n, x in res.items()}, kernel, rows, True)
    say(f"  err {most:.3f}, mean {mean:.3f}; pieces of {longest} steps, {parts} at most of an item")
    assert most <= 1 and mean <= 1
    # outputs of all sequences: means of many values of variance 1 (what is left out of one shows in its size)
    assert np.isfinite(out).all() and np.abs(out).max() < 4
    at.free()
