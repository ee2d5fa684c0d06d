"""The 4-bit paged attention where values and sizes are extreme."""
import numpy as np
import pytest

from gpu_common import say
from paged_common import HD, f64
from q4_common import BF16_MAX, Batch4, quantise, values
from test_gpu_paged_q4 import Attn4, ctx  # noqa: F401
from test_gpu_paged_q4_use import widen
from vx27_amd import workloads as W

pytestmark = pytest.mark.gpu

KERNELS = ("paged_q4_split", "paged_rows_q4", "paged_rows_flat")


def run(at):
    """The attention kernel that a call runs."""
    at.ctx.prof_enable(True)
    at.call()
    ran = [k for k in KERNELS if at.ctx.prof_read(k)[0]]
    at.ctx.prof_enable(False)
    assert len(ran) == 1
    return ran[0]


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
