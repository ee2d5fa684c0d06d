"""Ragged batches over a paged cache and their float64 results, for the paged
operators' tests.  Rows that no token of a case sees hold NaN, as stale pages
may: one that gets in shows."""
from __future__ import annotations

import numpy as np

from vx27_amd import workloads as W

HD = 256
NAN_BITS = 0x7FC1


def f64(bits):
    with np.errstate(invalid="ignore"):     # (the NaN of stale rows)
        return W.bf16_to_f32(bits).astype(np.float64)


class Batch:
    """Sequences of `lens` rows whose last `new` are the call's tokens."""

    def __init__(self, lens, new, n_q=24, n_kv=4, page=64, window=0, sink=0, seed=0, q_std=2.0, lead=0, tail=0):
        r = np.random.default_rng([77, seed])
        self.r, self.lens, self.new = r, list(lens), list(new)
        self.n_q, self.n_kv, self.page, self.window, self.sink = n_q, n_kv, page, window, sink
        self.B, self.qg = len(lens), n_q // n_kv
        self.max_pages = max(1, max(-(-n // page) for n in lens)) + 1
        self.lead, self.N = lead, lead + sum(new) + tail
        self.start = np.concatenate(([lead], lead + np.cumsum(new))).astype(np.int32)
        counts = [-(-n // page) for n in lens]
        self.n_pages = sum(counts) + 2
        order = r.permutation(self.n_pages)
        self.table = np.full((self.B, self.max_pages), -7, np.int32)     # entries behind the last page hold anything
        self.k = np.full((self.n_pages, n_kv, page, HD), NAN_BITS, np.uint16)
        self.v = np.full((self.n_pages, n_kv, page // 32, HD, 32), NAN_BITS, np.uint16)
        at = 0
        for b, n in enumerate(lens):
            self.table[b, :counts[b]] = order[at:at + counts[b]]
            at += counts[b]
            for j in np.nonzero(self.seen(b).any(0))[0]:
                self.put_row(b, j, W.bf16_bits(W.normal(r, (n_kv, HD))), W.bf16_bits(W.normal(r, (n_kv, HD))))
        self.q = W.bf16_bits(W.normal(r, (self.N, n_q, HD), q_std))
        self.gate = W.normal(r, (self.N, n_q, HD))

    def seen(self, b):
        """[tokens][rows] of sequence b: what each token sees."""
        n, t = self.lens[b], self.new[b]
        i = (n - t + np.arange(t))[:, None]
        j = np.arange(n)[None]
        s = j <= i
        if self.window:
            s &= (j > i - self.window) | (j < self.sink)
        return s

    def put_row(self, b, j, k, v):
        p, at = self.table[b, j // self.page], j % self.page
        self.k[p, :, at] = k
        self.v[p, :, at // 32, :, at % 32] = v

    def rows(self, b):
        """K and V bits of sequence b, [rows][n_kv][hd]."""
        n = self.lens[b]
        pg = self.table[b, :-(-n // self.page)] if n else self.table[b, :0]
        k = self.k[pg].transpose(0, 2, 1, 3).reshape(-1, self.n_kv, HD)[:n]
        v = self.v[pg].transpose(0, 2, 4, 1, 3).reshape(-1, self.n_kv, HD)[:n]
        return k, v

    def result(self, gate=True, q=None):
        """dict of float64 results: out, lse [N][n_q], acc increments (list of [n_kv][rows]), and for tolerances W (the
        weighted sum of |v|) and S (the largest sum of |q||k| / 16 of a token's scores)."""
        q = f64(self.q) if q is None else q
        out, Wt = np.zeros((self.N, self.n_q, HD)), np.zeros((self.N, self.n_q, HD))
        lse, S, acc = np.full((self.N, self.n_q), -np.inf), np.zeros((self.N, self.n_q)), []
        for b in range(self.B):
            k, v = self.rows(b)
            seen, t0 = self.seen(b), self.start[b]
            ok = seen.any(0)
            k, v = f64(k), f64(v)
            k[~ok] = 0
            v[~ok] = 0
            inc = np.zeros((self.n_kv, self.lens[b]))
            for h in range(self.n_q):
                qq, kk, vv = q[t0:t0 + self.new[b], h], k[:, h // self.qg], v[:, h // self.qg]
                if not len(qq) or not len(kk):
                    continue
                with np.errstate(all="ignore"):
                    s = np.where(seen, qq @ kk.T / 16.0, -np.inf)
                    m = s.max(1, keepdims=True)
                    p = np.where(seen, np.exp(s - np.where(np.isfinite(m), m, 0)), 0.0)
                    l = p.sum(1, keepdims=True)
                    w = np.where(l > 0, p / l, 0.0)
                    lse[t0:t0 + self.new[b], h] = (m + np.log(l))[:, 0]
                out[t0:t0 + self.new[b], h] = w @ vv
                Wt[t0:t0 + self.new[b], h] = w @ np.abs(vv)
                S[t0:t0 + self.new[b], h] = (np.where(seen, np.abs(qq) @ np.abs(kk).T, 0) / 16.0).max(1)
                inc[h // self.qg] += w.sum(0)
            acc.append(inc)
        if gate:
            g = 1.0 / (1.0 + np.exp(-self.gate.astype(np.float64)))
            out *= g
            Wt *= g
        return {"out": out, "lse": lse, "acc": acc, "W": Wt, "S": S}


def score_err(S):
    """Bound of a score's error: 256 products summed in fp32 in any order, 256 * 2^-24 of the sum of their magnitudes."""
    return 256 * 2.0 ** -24 * S


def out_tol(res, keys, out_bf16, one_part):
    """Elementwise bound of the attention output's error.  A weight's relative error is at most that of its score (and
    the row's maximum and sum: twice), plus 2^-20 for exp2 and its argument, plus 2^-8 where it is rounded to bf16 once
    (one_part); sums over up to `keys` rows in fp32, in 3 parts each, add 3 * keys * 2^-24; rounding the output to bf16
    2^-8 of it.  All relative to the weighted sum of |v|."""
    rel = 2 * score_err(res["S"])[..., None] + 2.0 ** -20 + 3 * keys * 2.0 ** -24 + (2.0 ** -8 if one_part else 0.0)
    return 1.01 * rel * res["W"] + (2.0 ** -8 * np.abs(res["out"]) if out_bf16 else 0.0) + 1e-30
