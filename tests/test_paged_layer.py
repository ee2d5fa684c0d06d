"""The bookkeeping of PagedGQALayer without a GPU: pages, rows and device
buffers around steps and evictions that run or are refused.  "Device" memory
is host memory and the library's calls are stubs that record their
descriptors."""
import ctypes as C

import numpy as np
import pytest

from vx27_amd import lib as L, mixers as M

HD = 256


class FakeBuf:
    def __init__(self, ctx, nbytes):
        self.ctx, self.nbytes = ctx, int(nbytes)
        self.mem = np.zeros(self.nbytes, np.uint8)
        self.ptr = self.mem.ctypes.data
        ctx.live.append(self)

    def upload(self, arr):
        raw = np.frombuffer(np.ascontiguousarray(arr).tobytes(), np.uint8)
        assert raw.size <= self.nbytes
        self.mem[:raw.size] = raw
        return self

    def download(self, shape, dtype):
        return np.frombuffer(self.mem.tobytes(), dtype)[:int(np.prod(shape))].reshape(shape).copy()

    def zero(self):
        self.mem[:] = 0
        return self

    def free(self):
        if self.ptr:
            self.ctx.live.remove(self)
            self.ptr = None


class FakeCtx:
    h = None

    def __init__(self):
        self.live = []

    def buf(self, nbytes):
        return FakeBuf(self, nbytes)

    def put(self, arr):
        arr = np.ascontiguousarray(arr)
        return self.buf(max(arr.nbytes, 1)).upload(arr)

    def sync(self):
        L.check(L.lib().sync_rc(), "sync")


class FakeLib:
    """Calls succeed unless named in `refuse`; `seen` holds (name, len, new tokens or budget) of each."""

    def __init__(self):
        self.refuse, self.seen = set(), []

    def _call(self, name, d):
        n = np.ctypeslib.as_array(C.cast(d.len, C.POINTER(C.c_int)), (d.B,)).tolist()
        self.seen.append((name, n))
        return -1 if name in self.refuse else 0

    def vx27_hip_paged_append(self, h, d):
        return self._call("append", d._obj)

    def vx27_hip_paged_attn(self, h, d):
        return self._call("attn", d._obj)

    def vx27_hip_paged_evict(self, h, d):
        d = d._obj
        rc = self._call("evict", d)
        if rc == 0 and d.n_sink + d.n_recent > d.budget:
            return -1
        if rc == 0:
            n, out = (C.cast(x, C.POINTER(C.c_int)) for x in (d.len, d.dst_len))
            kept, acc, acc_out = (C.cast(x, C.POINTER(t)) for x, t in ((d.kept, C.c_int), (d.acc, C.c_float), (d.acc_out or d.acc, C.c_float)))
            for b in range(d.B):
                out[b] = min(n[b], d.budget)
                for h_ in range(d.n_kv):
                    s = b * d.n_kv + h_
                    for i in range(out[b]):      # (which rows stay does not matter here: the last ones)
                        r = n[b] - out[b] + i
                        kept[s * d.budget + i] = r
                        if d.acc_out:
                            acc_out[s * d.acc_out_stride + i] = acc[s * d.acc_stride + r]
        return rc

    def vx27_hip_memset(self, h, p, byte, n):
        C.memset(p, byte, n)
        return 0

    def vx27_hip_d2d(self, h, dst, src, n):
        C.memmove(dst, src, n)
        return 0

    def sync_rc(self):
        return -1 if "sync" in self.refuse else 0

    def vx27_hip_last_error(self):
        return b"refused"


@pytest.fixture
def fake(monkeypatch):
    f = FakeLib()
    monkeypatch.setattr(L, "lib", lambda: f)
    return f


def layer(n_seq=2, n_pages=3, page=32, **kw):
    return M.PagedGQALayer(FakeCtx(), n_seq, n_pages, page, np.zeros(HD), np.zeros(HD), **kw)


def tokens(n, n_q=24, n_kv=4):
    return np.zeros((n, n_q, 2 * HD), np.float32), np.zeros((n, n_kv, HD), np.float32), np.zeros((n, n_kv, HD), np.float32)


def held(lay):
    return [list(p) for p in lay.pages], list(lay.free), list(lay.rows), list(lay.pos)


@pytest.mark.parametrize("refuse", [None, "append", "attn", "sync"])
def test_a_refused_step_takes_no_pages(fake, refuse):
    """The pool is too small for the second sequence, or the library refuses: no sequence holds a page more, and a step
    that needs those pages runs."""
    lay = layer()
    lay.step([5, 0], *tokens(5))
    before = held(lay)
    if refuse:
        fake.refuse = {refuse}
    with pytest.raises(L.HipError):
        lay.step([40, 40] if refuse is None else [40, 1], *tokens(80 if refuse is None else 41))
    assert held(lay) == before
    fake.refuse = set()
    lay.step([0, 64], *tokens(64))
    assert lay.rows == [5, 64] and lay.free == [] and sorted(sum(lay.pages, [])) == [0, 1, 2]


@pytest.mark.parametrize("refuse", ["arguments", "evict", "sync"])
def test_a_refused_eviction_keeps_every_page(fake, refuse):
    """The library refuses the call or the sync reports one: the fresh pages are free again, the rows and their weights
    as they were, and the same eviction runs afterwards."""
    lay = layer(2, 8, max_pages=4)
    lay.step([70, 3], *tokens(73))
    lay.acc.upload(np.arange(lay.acc.nbytes // 4, dtype=np.float32))
    before, weights = held(lay), lay.acc.download((2, 4, lay.acc_stride), np.float32)
    if refuse != "arguments":
        fake.refuse = {refuse}
    with pytest.raises(L.HipError):
        lay.evict(40, 30 if refuse == "arguments" else 4, 20)
    assert held(lay) == before
    assert np.array_equal(lay.acc.download(weights.shape, np.float32), weights)
    fake.refuse = set()
    for _ in range(3):
        lay.evict(40, 4, 20)
    assert lay.rows == [40, 3] and len(lay.free) + sum(map(len, lay.pages)) == 8
    assert sorted(lay.free + sum(lay.pages, [])) == list(range(8))


@pytest.mark.parametrize("refuse", ["append", "attn", "evict", "sync"])
def test_no_buffers_stay_behind(fake, refuse):
    """A call that runs and a call that is refused leave no device buffer of their own."""
    lay = layer(2, 8, max_pages=4)
    lay.step([70, 3], *tokens(73), weigh=True)
    live = len(lay.ctx.live)
    fake.refuse = {refuse}
    with pytest.raises(L.HipError):
        lay.evict(40, 4, 20) if refuse == "evict" else lay.step([1, 1], *tokens(2))
    assert len(lay.ctx.live) == live
    fake.refuse = set()
    lay.step([1, 1], *tokens(2))
    lay.evict(40, 4, 20)
    assert len(lay.ctx.live) == live


def test_eviction_touches_only_sequences_past_the_budget(fake):
    """In a pool with two free pages one long sequence is brought back to its budget: the others keep their pages, rows
    and weights, and where none is past the budget nothing is needed."""
    lay = layer(3, 9, max_pages=6)
    lay.step([64, 100, 20], *tokens(184), weigh=True)
    assert len(lay.free) == 2
    pages = [list(p) for p in lay.pages]
    w = np.random.default_rng(1).random((3, 4, lay.acc_stride)).astype(np.float32)
    lay.acc.upload(w)
    kept = lay.evict(64, 4, 60)
    assert fake.seen[-1] == ("evict", [0, 100, 0])
    assert lay.rows == [64, 64, 20] and lay.pages[0] == pages[0] and lay.pages[2] == pages[2]
    assert sorted(lay.free + sum(lay.pages, [])) == list(range(9)) and len(lay.free) == 4
    for b, n, old in ((0, 64, range(64)), (1, 64, range(36, 100)), (2, 20, range(20))):
        assert np.array_equal(kept[b], np.broadcast_to(list(old) + [-1] * (64 - n), (4, 64)))
    want = w.copy()
    want[1] = 0
    want[1, :, :64] = w[1, :, 36:100]
    assert np.array_equal(lay.acc.download(w.shape, np.float32), want)
    before = held(lay)
    lay.free = []
    kept = lay.evict(64, 4, 60)
    assert (lay.pages, lay.rows, lay.pos) == (before[0], before[2], before[3])
    assert np.array_equal(kept[2, 0], list(range(20)) + [-1] * 44)
    assert np.array_equal(lay.acc.download(w.shape, np.float32), want)
    with pytest.raises(L.HipError):
        lay.evict(64, 60, 60)          # refused whatever the rows


def test_an_ended_sequence_gives_everything_back(fake):
    """end() returns a sequence's pages and clears its rows, position and weights, so that another conversation may take
    its place."""
    lay = layer(2, 4)
    lay.step([70, 30], *tokens(100), weigh=True)
    lay.acc.upload(np.ones(lay.acc.nbytes // 4, np.float32))
    with pytest.raises(L.HipError):
        lay.step([0, 40], *tokens(40))
    lay.end(0)
    assert lay.rows == [0, 30] and lay.pos == [0, 30] and lay.pages[0] == []
    acc = lay.acc.download((2, 4 * lay.acc_stride), np.float32)
    assert not acc[0].any() and acc[1].all()
    lay.step([1, 60], *tokens(61))
    assert lay.rows == [1, 90] and lay.pos == [1, 90]
    with pytest.raises(L.HipError):
        lay.step([40, 0], *tokens(40))     # the pool is full again
    lay.end(0)
    lay.end(0)
    assert sorted(lay.free + sum(lay.pages, [])) == list(range(4))
    for b in (-1, 2):
        with pytest.raises(L.HipError, match="sequence"):
            lay.end(b)


@pytest.mark.parametrize("new,n,what", [
    ([3], 3, "new"), ([1, 1, 1], 3, "new"), ([3, -1], 2, "new"), ([2, 1], 2, "qg"), ([2, 1], (3, 2, 3), "k_new"),
    ([2, 1], (3, 3, 2), "v_new")])
def test_arguments_that_hold_too_little_are_refused(fake, new, n, what):
    """The calls read sum(new) tokens of each array: an array that holds fewer, or counts that are not one a sequence, do
    not reach the library."""
    lay = layer(2, 4)
    n = (n, n, n) if isinstance(n, int) else n
    args = [tokens(k)[i] for i, k in enumerate(n)]
    before = held(lay)
    with pytest.raises(L.HipError, match=what):
        lay.step(new, *args)
    assert fake.seen == [] and held(lay) == before


@pytest.mark.parametrize("which", [0, 1])
def test_short_norm_weights_are_refused(fake, which):
    w = [np.zeros(HD), np.zeros(HD)]
    w[which] = np.zeros(HD - 1)
    with pytest.raises(L.HipError, match="norm_w"):
        M.PagedGQALayer(FakeCtx(), 1, 1, 32, *w)
