"""The device-side plan of a step's rows and pages against its definition, one
sequence after the other on the host."""
import ctypes as C

import numpy as np
import pytest

from gpu_common import say
from plan_common import NAMES, plan, pool
from test_gpu_paged_q4 import ctx  # noqa: F401

pytestmark = pytest.mark.gpu


class Plan:
    """A pool's state on the device and its plan call.  Written-to arrays stand between guard words."""

    def __init__(self, ctx, lens, new, table, free, n_free, page, n_tok, ended=None, next_pos=None, in_place=False, drop=()):
        from vx27_amd import lib as L
        self.ctx, self.L, B = ctx, L, len(lens)
        i32 = lambda x: np.asarray(x, np.int32)  # noqa: E731
        self.up = dict(len=i32(lens), new_tok=i32(new), n_free=i32([n_free]), table=table, free_pages=free)
        if ended is not None:
            self.up["ended"] = i32(ended)
        if next_pos is not None:
            self.up["next_pos"] = i32(next_pos)
        size = dict(took=B, q_start=B + 1, len_out=B, next_pos_out=B, n_free_out=1, slot=n_tok, pos=n_tok, seq=n_tok)
        if next_pos is None:
            del size["next_pos_out"]
        for n in drop:
            del size[n]
        same = {"len_out": "len", "next_pos_out": "next_pos", "n_free_out": "n_free"} if in_place else {}
        for n, k in size.items():
            if n not in same:
                self.up[n] = np.full(k, -55, np.int32)
        self.shape = {n: x.shape for n, x in self.up.items()}
        self.buf = {n: ctx.buf(x.nbytes + 64) for n, x in self.up.items()}
        self.upload()
        d = self.d = L.PagedPlanDesc()
        d.B, d.page_size, d.n_pages, d.max_pages, d.n_tok = B, page, len(free), table.shape[1], n_tok
        for n, b in self.buf.items():
            setattr(d, n, b.ptr + 32)
        for n, x in same.items():
            if x in self.buf:
                setattr(d, n, self.buf[x].ptr + 32)
                self.shape[n] = self.shape[x]
                self.buf[n] = self.buf[x]

    def upload(self):
        for n, x in self.up.items():
            guard = np.full(8, 0x13579BDF, np.int32)
            self.buf[n].upload(np.concatenate([guard, x.ravel(), guard]))

    def call(self):
        self.L.check(self.L.lib().vx27_hip_paged_plan(self.ctx.h, C.byref(self.d)), "paged_plan")

    def get(self, n):
        k = int(np.prod(self.shape[n]))
        x = self.buf[n].download((k + 16,), np.int32)
        assert np.all(x[:8] == 0x13579BDF) and np.all(x[8 + k:] == 0x13579BDF), f"{n}: written outside"
        return x[8:8 + k].reshape(self.shape[n])

    def check(self, want):
        for n in NAMES:
            if n in self.buf:
                got = self.get(n)
                assert np.array_equal(got, want[n]), (n, got, want[n])

    def free(self):
        for b in set(self.buf.values()):
            b.free()


def draw(r, B, page, long, most):
    """Rows and tokens: nothing, part of a page, whole pages, one more, many."""
    lens = np.where(r.random(B) < 0.5, r.integers(0, 3 * page, B), r.integers(0, 4, B) * page + r.integers(-1, 2, B)).clip(0)
    new = np.where(r.random(B) < 0.6, r.integers(0, 3, B), r.integers(0, most + 1, B))
    if long:
        new[r.integers(0, B)] = 20 * page + 1
    return lens, new


CASES = [(B, page, long, ended, pos, short, room) for B, page in ((1, 32), (2, 96), (7, 64), (64, 32), (300, 128))
         for long, ended, pos, short, room in ((False, False, False, 0, 0), (True, True, True, 0, 0), (False, True, False, 3, 0),
                                               (True, False, True, 2, 1), (False, True, True, 0, 2))]
CASES += [(1023, 32, True, True, True, 2, 0), (1024, 64, False, True, False, 0, 0), (1025, 64, True, True, True, 3, 1),
          (3000, 32, False, True, True, 0, 2), (9000, 64, False, False, True, 2, 0)]


@pytest.mark.parametrize("B,page,long,ended,pos,short,room", CASES)
def test_plan(ctx, B, page, long, ended, pos, short, room):  # noqa: F811
    """short: a part of the pages that are needed are free; room: a part of the tokens fits."""
    say(f"plan B={B} page={page} long={long} ended={ended} pos={pos} short={short} room={room}")
    r = np.random.default_rng([1000, B, page, long, ended, pos, short, room])
    lens, new = draw(r, B, page, long, 2 * page)
    need = int((-(-(lens + new) // page) - -(-lens // page)).sum())
    max_pages = int((-(-lens // page)).max()) + (4 if long else 3)        # (a long request is past it)
    table, free, n_free = pool(r, lens, page, need // short if short else need + 2, max_pages, spare=3)
    e = (r.random(B) < 0.2).astype(np.int32) * r.integers(1, 5, B) if ended else None
    nxt = lens + r.integers(0, 1000, B) if pos else None
    n_tok = int(new.sum()) // 2 if room == 1 else 0 if room == 2 and B < 5 else int(new.sum()) + 3
    want = plan(lens, new, table, free, n_free, page, n_tok, e, nxt)
    if nxt is None:
        want["pos"] = np.where(want["seq"] >= 0, want["pos"], -1)
    for in_place in (False, True):
        p = Plan(ctx, lens, new, table, free, n_free, page, n_tok, e, nxt, in_place, drop=("pos",) if B == 7 else ())
        p.call()
        ctx.sync()
        p.check(want)
        p.free()


def test_steps_go_on_in_place(ctx):  # noqa: F811
    """A captured plan, replayed: lengths, positions and free pages go on from step to step; sequences end and others
    take their places; every page is somewhere exactly once."""
    from vx27_amd import lib as L
    say("captured plans in place")
    r = np.random.default_rng(1100)
    for B, big in ((5, 0), (40, 0), (40, 5000)):
        page, width = 32, 9
        lens = r.integers(0, 100, B)
        table, free, n_free = pool(r, lens, page, 30, width, spare=0)
        n_tok = 3 * B + big
        nxt = lens + 7
        p = Plan(ctx, lens, np.ones(B, int), table, free, n_free, page, n_tok, np.zeros(B, int), nxt, in_place=True)
        p.call()
        ctx.sync()
        p.upload()
        ctx.graph_begin()
        p.call()
        g = ctx.graph_end()
        state = dict(lens=lens, table=table, free=free, n_free=n_free, nxt=nxt)
        for step in range(12):
            new = r.integers(0, 4, B)
            e = (r.random(B) < 0.15).astype(np.int32)
            for n, x in (("new_tok", new), ("ended", e)):
                g8 = np.full(8, 0x13579BDF, np.int32)
                p.buf[n].upload(np.concatenate([g8, x.astype(np.int32), g8]))
            want = plan(state["lens"], new, state["table"], state["free"], state["n_free"], page, n_tok, e, state["nxt"])
            ctx.graph_launch(g)
            ctx.sync()
            got = {n: p.get(n) for n in NAMES}
            k = want["n_free_out"][0]
            assert np.array_equal(got["free_pages"][:k], want["free_pages"][:k])
            want["free_pages"] = got["free_pages"]
            for n in NAMES:
                assert np.array_equal(got[n], want[n]), (step, n)
            held = [x for b in range(B) for x in got["table"][b, :-(-got["len_out"][b] // page)]]
            assert sorted([*held, *got["free_pages"][:k]]) == list(range(len(free)))
            state = dict(lens=want["len_out"], table=want["table"], free=want["free_pages"], n_free=k, nxt=want["next_pos_out"])
        L.check(L.lib().vx27_hip_graph_destroy(g))
        p.free()


@pytest.mark.parametrize("B", [3, 2000])
@pytest.mark.parametrize("what", ["len", "new", "n_free", "page", "free page", "twice"])
def test_faulty_tables_are_reported(ctx, B, what):  # noqa: F811
    """Values outside their ranges are clamped: nothing is written outside its array, and sync reports it; the next call
    is as before."""
    from vx27_amd import lib as L
    say(f"faulty {what}, B={B}")
    r = np.random.default_rng([1200, B])
    page, width = 32, 6
    lens = r.integers(1, 100, B)
    new = r.integers(20, 60, B)
    table, free, n_free = pool(r, lens, page, 3 * B, width)
    n_tok = int(new.sum())
    e = np.zeros(B, int)
    e[B - 1] = what != "free page"                 # (released pages would be taken before the free ones)
    args = dict(lens=lens.copy(), new=new.copy(), table=table.copy(), free=free.copy(), n_free=n_free)
    if what == "len":
        args["lens"][:3] = [-5, 2 ** 31 - 1, width * page + 1]
    if what == "new":
        args["new"][:2] = [-1, -2 ** 31]
    if what == "n_free":
        args["n_free"] = len(free) + 1
    if what == "page":
        args["table"][0, 0], args["table"][1, :], args["table"][B - 1, 0] = 10 ** 9, -7, len(free)
    if what == "free page":
        args["free"][:n_free] = -1
        args["free"][0] = 2 ** 31 - 1
    if what == "twice":
        args["n_free"] = len(free)                  # (all pages free, and one sequence gives some back)
        args["free"][:] = np.arange(len(free))
    p = Plan(ctx, args["lens"], args["new"], args["table"], args["free"], args["n_free"], page, n_tok, e, np.arange(B))
    p.call()
    with pytest.raises(L.HipError, match="outside its paged cache"):
        ctx.sync()
    for n in p.buf:
        p.get(n)                                    # (guards)
    p.free()
    p = Plan(ctx, lens, new, table, free, n_free, page, n_tok, e, np.arange(B))
    p.call()
    ctx.sync()
    p.check(plan(lens, new, table, free, n_free, page, n_tok, e, np.arange(B)))
    p.free()
