"""PagedGQALayer on the GPU: places that end and are taken again, eviction in
a pool that is nearly full, and calls after one that was refused."""
import ctypes as C

import numpy as np
import pytest

from gpu_common import say
from paged_common import HD, Batch
from test_gpu_paged import Attn, ctx  # noqa: F401

pytestmark = pytest.mark.gpu


def tokens(r, n):
    return tuple(r.standard_normal(s).astype(np.float32) for s in ((n, 24, 2 * HD), (n, 4, HD), (n, 4, HD)))


def test_a_place_that_is_taken_again(ctx):  # noqa: F811
    """After end() a sequence's place gives the bytes of a fresh layer: outputs, rows and weights."""
    from vx27_amd import mixers as M
    r = np.random.default_rng(700)
    qn, kn = r.standard_normal(HD) / 10, r.standard_normal(HD) / 10
    old = M.PagedGQALayer(ctx, 2, 12, 32, qn, kn)
    old.step([150, 40], *tokens(r, 190), weigh=True)
    old.step([1, 3], *tokens(r, 4), weigh=True)
    old.end(0)
    fresh = M.PagedGQALayer(ctx, 2, 12, 32, qn, kn)
    for n in (100, 1, 1, 5):
        t = tokens(r, n)
        assert np.array_equal(old.step([n, 0], *t, weigh=True), fresh.step([n, 0], *t, weigh=True))
    for x, y in zip(old.read_rows(0), fresh.read_rows(0)):
        assert np.array_equal(x, y)
    a, b = (lay.acc.download((2, 4, lay.acc_stride), np.float32) for lay in (old, fresh))
    assert np.array_equal(a[0], b[0]) and a[1, :, :43].any()
    assert np.array_equal(old.evict(60, 4, 20)[0], fresh.evict(60, 4, 20)[0])


def test_eviction_in_a_nearly_full_pool(ctx):  # noqa: F811
    """Two free pages bring the one long sequence back to its budget; the others' rows, weights and next outputs are
    those of a layer that never evicted."""
    from vx27_amd import mixers as M
    r = np.random.default_rng(701)
    qn, kn = r.standard_normal(HD) / 10, r.standard_normal(HD) / 10
    lays = [M.PagedGQALayer(ctx, 3, n, 32, qn, kn, max_pages=6) for n in (9, 30)]
    first, nxt = tokens(r, 184), tokens(r, 2)
    for lay in lays:
        lay.step([64, 100, 20], *first, weigh=True)
    a = lays[0].acc.download((3, 4, lays[0].acc_stride), np.float32)
    rows = lays[0].read_rows(1)
    kept = lays[0].evict(64, 4, 20)
    b = lays[0].acc.download(a.shape, np.float32)
    assert lays[0].rows == [64, 64, 20] and len(lays[0].free) == 4
    assert np.array_equal(b[[0, 2]], a[[0, 2]]) and not b[1, :, 64:].any()
    for h in range(4):
        assert np.array_equal(b[1, h, :64], a[1, h, kept[1, h]])
        for x, y in zip(rows, lays[0].read_rows(1)):
            assert np.array_equal(y[:, h], x[kept[1, h], h])
    assert np.array_equal(lays[0].step([1, 0, 1], *nxt), lays[1].step([1, 0, 1], *nxt))


def test_a_workspace_that_cannot_be_had(ctx):  # noqa: F811
    """Weights of a capacity whose scores would take terabytes are refused when the workspace is asked for; the next call
    runs."""
    from vx27_amd import lib as L
    say("a workspace of terabytes")
    with L.Ctx(0) as c:
        a = Attn(c, Batch([70, 40], [1, 1], seed=702), acc=True)
        d = L.PagedAttnDesc()
        C.memmove(C.byref(d), C.byref(a.d), C.sizeof(d))
        d.B, d.n_tok, d.max_T, d.q_start = 64, 64, 1, None
        d.page_size, d.max_pages, d.acc_stride = 1 << 20, 1 << 10, 1 << 30
        with pytest.raises(L.HipError):
            L.check(L.lib().vx27_hip_paged_attn(c.h, C.byref(d)))
        a.call()
        a.check("after the refusal")
