"""The paged-cache operators where values and sizes are extreme."""
import numpy as np
import pytest

from gpu_common import say
from paged_common import HD, Batch, out_tol
from test_gpu_paged import Attn, ctx  # noqa: F401

pytestmark = pytest.mark.gpu

NAN = 0x7FC1


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
