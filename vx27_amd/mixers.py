"""Host-side mirror of the reference's mixer interface over the C ABI.

Two levels, both calling libvx27_hip (no host compute):
  * the reference's own per-head functions (deltanet_step_exact, conv1d_step,
    rmsnorm, attn_1q, rope_*), host arrays in / out, exactly the reference's
    arguments (src/vx27_deltanet.h:10-59, src/vx27_gqa.h:8-13,
    src/vx27_rope.h:11-17);
  * device-resident layer objects (DeltaNetLayer, GatedGQALayer) holding the
    state / KV cache of B sequences and running the batched decode kernels,
    the form vx27_qlayer's mixer sections (src/vx27_qfwd.c:92-215) take here.
"""
from __future__ import annotations

import contextlib
import ctypes as C

import numpy as np

from . import lib as L
from .lib import check, hptr


def _f32(a):
    return np.ascontiguousarray(a, np.float32)


# ----------------------------------------------- the reference's own calls
def deltanet_step_exact(S, q, k, v, beta, g_log):
    """vx27_deltanet_step_exact: S (float32 [hd][hd]) updated in place; returns o."""
    assert S.dtype == np.float32 and S.flags["C_CONTIGUOUS"]
    q, k, v = _f32(q), _f32(k), _f32(v)
    o = np.empty(q.size, np.float32)
    L.lib().vx27_deltanet_step_exact(hptr(S), hptr(q), hptr(k), hptr(v), float(beta), float(g_log),
                                     hptr(o), q.size)
    return o


def deltanet_gate_params(a, A_log, b, dt_bias):
    be, g = C.c_double(), C.c_double()
    L.lib().vx27_deltanet_gate_params(float(a), float(A_log), float(b), float(dt_bias),
                                      C.byref(be), C.byref(g))
    return be.value, g.value


def deltanet_l2norm(x):
    x = _f32(x)
    y = np.empty_like(x)
    L.lib().vx27_deltanet_l2norm(hptr(x), hptr(y), x.size)
    return y


def conv1d_step(state, x, w, apply_silu=True):
    """vx27_conv1d_step: state float32 [C][3] updated in place; returns y."""
    assert state.dtype == np.float32 and state.flags["C_CONTIGUOUS"]
    x, w = _f32(x), _f32(w)
    y = np.empty(x.size, np.float32)
    L.lib().vx27_conv1d_step(hptr(state), hptr(x), hptr(w), hptr(y), x.size, int(bool(apply_silu)))
    return y


def rmsnorm(x, w, eps):
    x, w = _f32(x), _f32(w)
    y = np.empty_like(x)
    L.lib().vx27_rmsnorm(hptr(x), hptr(w), hptr(y), x.size, float(eps))
    return y


def attn_1q(q, kcache, vcache, n_pos):
    q, kc, vc = _f32(q), _f32(kcache), _f32(vcache)
    out = np.empty(24 * 256, np.float32)
    L.lib().vx27_attn_1q(hptr(q), hptr(kc), hptr(vc), int(n_pos), hptr(out))
    return out


def rope_cos_sin(pos, rope_dim=64, theta=1e7, yarn=1.0):
    c = np.empty(rope_dim // 2, np.float32)
    s = np.empty(rope_dim // 2, np.float32)
    L.lib().vx27_rope_cos_sin(int(pos), hptr(c), hptr(s), rope_dim, float(theta), float(yarn))
    return c, s


def rope_apply(v, n_heads, head_dim, rope_dim, cosv, sinv):
    """vx27_rope_apply in place on float32 v."""
    assert v.dtype == np.float32 and v.flags["C_CONTIGUOUS"]
    cosv, sinv = _f32(cosv), _f32(sinv)
    L.lib().vx27_rope_apply(hptr(v), n_heads, head_dim, rope_dim, hptr(cosv), hptr(sinv))


# ------------------------------------------------- device-resident layers
class DeltaNetLayer:
    """One Gated DeltaNet layer's mixer core for B sequences, state on device.

    S [B][nv][128][128] fp32 (row = key dim), conv state [B][C][3] fp32.
    decode() runs `steps` tokens per sequence through vx27_hip_dn_decode.
    """

    def __init__(self, ctx, B, nqk, nv, A_log, dt_bias, norm_w=None, conv_w=None,
                 conv_w_dtype=L.F32, S0=None, conv0=None, hd=128):
        self.ctx, self.B, self.nqk, self.nv, self.hd = ctx, B, nqk, nv, hd
        self.C = 2 * nqk * hd + nv * hd
        nS = B * nv * hd * hd
        self.S = ctx.buf(nS * 4)
        if S0 is None:
            self.S.zero()
        else:
            self.S.upload(_f32(S0).reshape(-1))
        self.conv_state = ctx.buf(B * self.C * 3 * 4)
        if conv0 is None:
            self.conv_state.zero()
        else:
            self.conv_state.upload(_f32(conv0).reshape(-1))
        self.A_log = ctx.put(_f32(A_log))
        self.dt_bias = ctx.put(_f32(dt_bias))
        self.norm_w = ctx.put(_f32(norm_w)) if norm_w is not None else None
        self.conv_w_dtype = conv_w_dtype
        if conv_w is not None:
            cw = np.ascontiguousarray(conv_w, np.uint16 if conv_w_dtype == L.BF16 else np.float32)
            self.conv_w = ctx.put(cw)
        else:
            self.conv_w = None

    def desc(self, steps, flags, out, a, b, x=None, q=None, k=None, v=None, z=None):
        """Descriptor over device pointers (ints)."""
        d = L.DnDesc()
        d.B, d.nqk, d.nv, d.hd, d.steps, d.flags = self.B, self.nqk, self.nv, self.hd, steps, flags
        d.S = self.S.ptr
        d.conv_state = self.conv_state.ptr
        d.conv_w = self.conv_w.ptr if self.conv_w else None
        d.conv_w_dtype = self.conv_w_dtype
        d.x, d.q, d.k, d.v, d.a, d.b, d.z, d.out = x, q, k, v, a, b, z, out
        d.A_log, d.dt_bias = self.A_log.ptr, self.dt_bias.ptr
        d.norm_w = self.norm_w.ptr if self.norm_w else None
        return d

    def decode(self, steps, flags, a, b, x=None, q=None, k=None, v=None, z=None):
        """Host arrays in, host output [steps][B][nv][hd] back."""
        ctx = self.ctx
        bufs = {n: ctx.put(_f32(arr)) for n, arr in
                (("a", a), ("b", b), ("x", x), ("q", q), ("k", k), ("v", v), ("z", z))
                if arr is not None}
        out = ctx.buf(steps * self.B * self.nv * self.hd * 4)
        p = {n: bb.ptr for n, bb in bufs.items()}
        d = self.desc(steps, flags, out.ptr, p["a"], p["b"], p.get("x"), p.get("q"), p.get("k"),
                      p.get("v"), p.get("z"))
        check(L.lib().vx27_hip_dn_decode(ctx.h, C.byref(d)), "dn_decode")
        res = out.download((steps, self.B, self.nv, self.hd), np.float32)
        for bb in list(bufs.values()) + [out]:
            bb.free()
        return res

    def state(self):
        return self.S.download((self.B, self.nv, self.hd, self.hd), np.float32)

    def conv(self):
        return self.conv_state.download((self.B, self.C, 3), np.float32)


class GatedGQALayer:
    """One gated GQA layer's mixer core for B sequences over a bf16 KV cache
    of capacity L positions (format of vx27_hip.h)."""

    def __init__(self, ctx, B, Lcap, q_norm_w, k_norm_w, n_q=24, n_kv=4, hd=256, rope_dim=64,
                 theta=1e7, yarn=1.0, flags=0):
        assert Lcap % 64 == 0
        self.ctx, self.B, self.L, self.n_q, self.n_kv, self.hd = ctx, B, Lcap, n_q, n_kv, hd
        self.rope_dim, self.theta, self.yarn, self.flags = rope_dim, theta, yarn, flags
        n = B * n_kv * Lcap * hd
        self.k_cache = ctx.buf(n * 2).zero()
        self.v_cache = ctx.buf(n * 2).zero()
        self.q_norm_w = ctx.put(_f32(q_norm_w))
        self.k_norm_w = ctx.put(_f32(k_norm_w))

    def write_kv(self, b, p0, k_rows, v_rows):
        """Rows [n][n_kv][hd] (fp32, rounded to bf16) at positions p0.. of sequence b."""
        k_rows, v_rows = _f32(k_rows), _f32(v_rows)
        n = k_rows.shape[0]
        kb, vb = self.ctx.put(k_rows), self.ctx.put(v_rows)
        check(L.lib().vx27_hip_kv_write(self.ctx.h, self.k_cache.ptr, self.v_cache.ptr, self.B,
                                        self.n_kv, self.hd, self.L, b, p0, n, kb.ptr, vb.ptr),
              "kv_write")
        self.ctx.sync()
        kb.free(); vb.free()

    def read_kv(self, b, p0, n):
        kb = self.ctx.buf(max(n, 1) * self.n_kv * self.hd * 4)
        vb = self.ctx.buf(max(n, 1) * self.n_kv * self.hd * 4)
        check(L.lib().vx27_hip_kv_read(self.ctx.h, self.k_cache.ptr, self.v_cache.ptr, self.B,
                                       self.n_kv, self.hd, self.L, b, p0, n, kb.ptr, vb.ptr),
              "kv_read")
        k = kb.download((n, self.n_kv, self.hd), np.float32)
        v = vb.download((n, self.n_kv, self.hd), np.float32)
        kb.free(); vb.free()
        return k, v

    def desc(self, pos, q, q_strides, gate, g_strides, k_new, v_new, out, n_split=0):
        d = L.GqaDesc()
        d.B, d.n_q, d.n_kv, d.hd = self.B, self.n_q, self.n_kv, self.hd
        d.rope_dim, d.rope_theta, d.rope_yarn, d.L, d.flags = (self.rope_dim, self.theta,
                                                              self.yarn, self.L, self.flags)
        d.pos, d.q, d.gate, d.k_new, d.v_new, d.out = pos, q, gate, k_new, v_new, out
        d.q_seq_stride, d.q_head_stride = q_strides
        d.gate_seq_stride, d.gate_head_stride = g_strides
        d.q_norm_w, d.k_norm_w = self.q_norm_w.ptr, self.k_norm_w.ptr
        d.k_cache, d.v_cache = self.k_cache.ptr, self.v_cache.ptr
        d.n_split = n_split
        return d

    def decode(self, pos, qg, k_new, v_new, n_split=0):
        """qg [B][n_q][2*hd] interleaved q|gate (vx27_qfwd.c:160-167); k_new, v_new
        [B][n_kv][hd]; pos [B].  Returns out [B][n_q][hd]."""
        ctx = self.ctx
        hd = self.hd
        qb = ctx.put(_f32(qg))
        kb, vb = ctx.put(_f32(k_new)), ctx.put(_f32(v_new))
        pb = ctx.put(np.ascontiguousarray(pos, np.int32))
        ob = ctx.buf(self.B * self.n_q * hd * 4)
        d = self.desc(pb.ptr, qb.ptr, (self.n_q * 2 * hd, 2 * hd), qb.ptr + hd * 4,
                      (self.n_q * 2 * hd, 2 * hd), kb.ptr, vb.ptr, ob.ptr, n_split)
        check(L.lib().vx27_hip_gqa_decode(ctx.h, C.byref(d)), "gqa_decode")
        out = ob.download((self.B, self.n_q, hd), np.float32)
        for bb in (qb, kb, vb, pb, ob):
            bb.free()
        return out


class PagedGQALayer:
    """One gated GQA layer's mixer core for sequences of any length over a
    paged bf16 KV cache (format of vx27_hip.h): a pool of n_pages pages, a
    page list per sequence kept here on the host, and each row's accumulated
    attention weight once a step asked for it.

    step() appends the sequences' new tokens and attends from them; evict()
    brings sequences past a budget back to it; end() frees a sequence's place
    for another.  max_pages: the most pages a sequence may have (n_pages by
    default); the weights, and the workspace of steps that add them up, go by
    n_seq * max_pages.
    """

    def __init__(self, ctx, n_seq, n_pages, page_size, q_norm_w, k_norm_w, n_q=24, n_kv=4, hd=256, rope_dim=64,
                 theta=1e7, yarn=1.0, flags=0, window=0, n_sink=0, max_pages=None):
        self.ctx, self.n_seq, self.n_pages, self.page = ctx, n_seq, n_pages, page_size
        self.n_q, self.n_kv, self.hd, self.rope_dim, self.theta, self.yarn = n_q, n_kv, hd, rope_dim, theta, yarn
        self.flags, self.window, self.n_sink = flags, window, n_sink
        self.max_pages = max_pages or n_pages
        if np.size(q_norm_w) < hd or np.size(k_norm_w) < hd:
            raise L.HipError(f"paged cache: q_norm_w and k_norm_w need {hd} numbers (got {np.size(q_norm_w)}, {np.size(k_norm_w)})")
        n = n_pages * n_kv * page_size * hd
        self.k_pages = ctx.buf(n * 2).zero()
        self.v_pages = ctx.buf(n * 2).zero()
        self.q_norm_w, self.k_norm_w = ctx.put(_f32(q_norm_w)), ctx.put(_f32(k_norm_w))
        self.acc_stride = self.max_pages * page_size
        self.acc = ctx.buf(n_seq * n_kv * self.acc_stride * 4).zero()
        self.free = list(range(n_pages))[::-1]
        self.pages = [[] for _ in range(n_seq)]
        self.rows = [0] * n_seq          # cached rows
        self.pos = [0] * n_seq           # positions seen (rows that were evicted included)

    @contextlib.contextmanager
    def _grown(self, rows):
        """Pages for `rows` rows of every sequence: all of them, or none where there are too few; given back if the
        call within fails."""
        need = [max(-(-n // self.page), len(p)) for n, p in zip(rows, self.pages)]
        more = sum(need) - sum(map(len, self.pages))
        if max(need) > self.max_pages or more > len(self.free):
            raise L.HipError(f"paged cache: {more} more pages needed ({len(self.free)} free), {max(need)} for one "
                             f"sequence ({self.max_pages} at most)")
        before = [len(p) for p in self.pages], list(self.free)
        for p, n in zip(self.pages, need):
            while len(p) < n:
                p.append(self.free.pop())
        try:
            yield
        except BaseException:
            for p, n in zip(self.pages, before[0]):
                del p[n:]
            self.free = before[1]
            raise

    @contextlib.contextmanager
    def _buffers(self):
        """buf and put of the context for the time of one call: freed at its end, whichever it is."""
        with contextlib.ExitStack() as stack:
            def buf(nbytes):
                b = self.ctx.buf(nbytes)
                stack.callback(b.free)
                return b
            yield buf, lambda arr: buf(max(arr.nbytes, 1)).upload(arr)

    def _table(self, pages):
        t = np.zeros((self.n_seq, self.max_pages), np.int32)
        for b, p in enumerate(pages):
            t[b, :len(p)] = p
        return t

    def step(self, new, qg, k_new, v_new, weigh=False, out_dtype=L.F32):
        """new [n_seq] tokens of each sequence; qg [N][n_q][2*hd] interleaved q|gate, k_new, v_new [N][n_kv][hd],
        the sequences' tokens one after the other.  weigh adds the rows' weights up.  Returns out [N][n_q][hd]
        (float32)."""
        N = int(np.sum(new))
        if len(new) != self.n_seq or min(new) < 0:
            raise L.HipError(f"paged cache: new must hold a count for each of {self.n_seq} sequences (got {list(new)})")
        for name, x, each in (("qg", qg, self.n_q * 2), ("k_new", k_new, self.n_kv), ("v_new", v_new, self.n_kv)):
            if np.size(x) < N * each * self.hd:
                raise L.HipError(f"paged cache: {name} holds {np.size(x)} numbers, {N} tokens need {N * each * self.hd}")
        if N == 0:
            return np.empty((0, self.n_q, self.hd), np.float32)
        rows = [n + int(t) for n, t in zip(self.rows, new)]
        with self._grown(rows), self._buffers() as (buf, put):
            out = self._step(buf, put, new, rows, qg, k_new, v_new, weigh, out_dtype)
        self.rows = rows
        self.pos = [p + int(t) for p, t in zip(self.pos, new)]
        return out

    def _step(self, buf, put, new, rows, qg, k_new, v_new, weigh, out_dtype):
        ctx, N, hd = self.ctx, int(np.sum(new)), self.hd
        start = np.concatenate(([0], np.cumsum(new))).astype(np.int32)
        pos = np.concatenate([np.arange(p, p + t) for p, t in zip(self.pos, new)]).astype(np.int32)
        qb, kb, vb, tb, lb, sb, pb = (put(x) for x in (_f32(qg), _f32(k_new), _f32(v_new), self._table(self.pages),
                                                       np.asarray(rows, np.int32), start, pos))
        rot, out = buf(N * self.n_q * hd * 2), buf(N * self.n_q * hd * 4)
        d = L.PagedAppendDesc()
        a = L.PagedAttnDesc()
        for x in (d, a):
            x.B, x.n_q, x.n_kv, x.hd, x.page_size, x.n_pages = self.n_seq, self.n_q, self.n_kv, hd, self.page, self.n_pages
            x.max_pages, x.table, x.len, x.q_start, x.n_tok, x.max_T = self.max_pages, tb.ptr, lb.ptr, sb.ptr, N, int(max(new))
            x.k_pages, x.v_pages = self.k_pages.ptr, self.v_pages.ptr
        d.rope_dim, d.rope_theta, d.rope_yarn, d.flags, d.pos = self.rope_dim, self.theta, self.yarn, self.flags, pb.ptr
        d.q, d.q_tok_stride, d.q_head_stride, d.k_new, d.v_new = qb.ptr, self.n_q * 2 * hd, 2 * hd, kb.ptr, vb.ptr
        d.q_norm_w, d.k_norm_w, d.q_out = self.q_norm_w.ptr, self.k_norm_w.ptr, rot.ptr
        a.q, a.window, a.n_sink, a.out, a.out_dtype = rot.ptr, self.window, self.n_sink, out.ptr, out_dtype
        if not self.flags & L.GQA_NO_GATE:
            a.gate, a.gate_tok_stride, a.gate_head_stride = qb.ptr + hd * 4, self.n_q * 2 * hd, 2 * hd
        if weigh:
            a.acc, a.acc_stride = self.acc.ptr, self.acc_stride
        check(L.lib().vx27_hip_paged_append(ctx.h, C.byref(d)), "paged_append")
        check(L.lib().vx27_hip_paged_attn(ctx.h, C.byref(a)), "paged_attn")
        ctx.sync()
        if out_dtype == L.BF16:
            return (out.download((N, self.n_q, hd), np.uint16).astype(np.uint32) << 16).view(np.float32)
        return out.download((N, self.n_q, hd), np.float32)

    def evict(self, budget, n_sink, n_recent):
        """Every sequence past `budget` rows keeps that many, in fresh pages; the others stay as they are.  Returns kept
        [n_seq][n_kv][budget], the old rows (-1 behind a sequence's last)."""
        with self._buffers() as (buf, put):
            return self._evict(buf, put, budget, n_sink, n_recent)

    def _evict(self, buf, put, budget, n_sink, n_recent):
        ctx, past = self.ctx, [n > budget for n in self.rows]
        need = [-(-budget // self.page) if p else 0 for p in past]
        if sum(need) > len(self.free):
            raise L.HipError(f"paged cache: eviction needs {sum(need)} fresh pages, {len(self.free)} are free")
        left = list(self.free)           # (the free pages are these only once the call has run)
        fresh = [[left.pop() for _ in range(k)] for k in need]
        width = max(1, min(self.max_pages, -(-budget // self.page)))
        dst = self._table(fresh)[:, :width]
        # sequences within the budget take part with no rows
        tb, lb, db, kb = (put(x) for x in (self._table(self.pages), np.where(past, self.rows, 0).astype(np.int32), dst,
                                           np.full((self.n_seq, self.n_kv, budget), -1, np.int32)))
        len2 = buf(self.n_seq * 4)
        d = L.PagedEvictDesc()
        d.B, d.n_kv, d.hd, d.page_size, d.n_pages, d.max_pages = self.n_seq, self.n_kv, self.hd, self.page, self.n_pages, self.max_pages
        d.table, d.len, d.budget, d.n_sink, d.n_recent = tb.ptr, lb.ptr, budget, n_sink, n_recent
        d.acc, d.acc_stride, d.k_pages, d.v_pages = self.acc.ptr, self.acc_stride, self.k_pages.ptr, self.v_pages.ptr
        d.dst_table, d.dst_max_pages, d.dst_len, d.kept = db.ptr, width, len2.ptr, kb.ptr
        if any(past):                    # (then the budget is below acc_stride)
            acc2 = buf(self.acc.nbytes).zero()
            d.acc_out, d.acc_out_stride = acc2.ptr, self.acc_stride
        check(L.lib().vx27_hip_paged_evict(ctx.h, C.byref(d)), "paged_evict")
        ctx.sync()
        kept = kb.download((self.n_seq, self.n_kv, budget), np.int32)
        each = self.n_kv * self.acc_stride * 4
        for b, p in enumerate(past):
            if p:
                check(L.lib().vx27_hip_d2d(ctx.h, self.acc.ptr + b * each, acc2.ptr + b * each, each), "d2d")
                left += self.pages[b]
                self.pages[b], self.rows[b] = fresh[b], budget
            else:
                kept[b, :, :self.rows[b]] = np.arange(self.rows[b])
        self.free = left
        return kept

    def end(self, b):
        """Sequence b ends: its pages are free, and its place, rows, position and weights as at the start."""
        if not 0 <= b < self.n_seq:
            raise L.HipError(f"paged cache: no sequence {b} (n_seq {self.n_seq})")
        each = self.n_kv * self.acc_stride * 4
        check(L.lib().vx27_hip_memset(self.ctx.h, self.acc.ptr + b * each, 0, each), "memset")
        self.free += self.pages[b]
        self.pages[b], self.rows[b], self.pos[b] = [], 0, 0

    def read_rows(self, b):
        """The cached rows of sequence b: K and V [rows][n_kv][hd] as float32."""
        n, P = self.rows[b], self.page
        k = self.k_pages.download((self.n_pages, self.n_kv, P, self.hd), np.uint16)[self.pages[b]]
        v = self.v_pages.download((self.n_pages, self.n_kv, P // 32, self.hd, 32), np.uint16)[self.pages[b]]
        k = k.transpose(0, 2, 1, 3).reshape(-1, self.n_kv, self.hd)[:n]
        v = v.transpose(0, 2, 4, 1, 3).reshape(-1, self.n_kv, self.hd)[:n]
        return tuple((x.astype(np.uint32) << 16).view(np.float32) for x in (k, v))
