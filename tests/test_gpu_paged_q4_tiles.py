"""The tile kernel over 4-bit pages where it decodes them itself."""
import pytest

import q4_bounds as Q
import test_gpu_paged_q4_use as U
from gpu_common import say
from q4_bounds import kernel_of, run
from q4_common import Batch4
from test_gpu_paged_q4 import Attn4, ctx  # noqa: F401

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
