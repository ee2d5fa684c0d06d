"""Results of the 4-bit paged attention as each of its kernels rounds, and
bounds that go no further than these roundings.

The decode kernels (paged_q4_split) take codes and queries as they are, sum
s (q c) and m (sum of q) in fp32, and weigh by two bf16 parts. The tile kernels
(paged_rows_q4, paged_rows_flat) round every value to bf16 first, which the
result here does too, so that the bound holds only what follows: scores, sums
and statistics in fp32, and each weight rounded to bf16 once."""
from __future__ import annotations

import numpy as np

from paged_common import HD, f64, score_err
from q4_common import values
from vx27_amd import workloads as W

PART = {"paged_q4_split": 2.0 ** -16, "paged_rows_q4": 2.0 ** -8, "paged_rows_flat": 2.0 ** -8}


def rounded(x):
    """As the tile kernels hold values: an fp32 number (one rounding of m + s c), to bf16."""
    with np.errstate(over="ignore", invalid="ignore"):
        return f64(W.bf16_bits(np.asarray(x, np.float32)))


def result(bt, kernel, gate=True, q=None, seen=None, tokens=None):
    """float64 out [N][n_q][256], lse [N][n_q]; W, the weighted sum of the magnitudes of the kernel's terms (values; of the
    decode kernels s c + |m|); V, the root of the sum of their weighted squares; S [N][n_q], the largest sum of magnitudes
    of a token's scores, and R the largest root of the sum of their squares. seen(b): what tokens see, if not bt.seen; tokens: only these rows of the call (a mask)."""
    q = f64(bt.q) if q is None else q
    out, Wt, V = (np.zeros((bt.N, bt.n_q, HD)) for _ in range(3))
    lse, S, R = np.full((bt.N, bt.n_q), -np.inf), np.zeros((bt.N, bt.n_q)), np.zeros((bt.N, bt.n_q))
    for b in range(bt.B):
        if not bt.lens[b] or not bt.new[b]:
            continue
        see, t0 = (seen or bt.seen)(b), bt.start[b]
        pick = np.arange(bt.new[b]) if tokens is None else np.nonzero(tokens[t0:t0 + bt.new[b]])[0]
        if not len(pick):
            continue
        see, at = see[pick], t0 + pick
        (kc, ks, km), (vc, vs, vm) = bt.held(b)
        k, v = values(kc, ks, km), values(vc, vs, vm)
        if kernel == "paged_q4_split":
            ka, va = (values(c, s, (m & 0x7FFF).astype(np.uint16)) for c, s, m in ((kc, ks, km), (vc, vs, vm)))
        else:
            k, v = rounded(k), rounded(v)
            ka, va = np.abs(k), np.abs(v)
        for x in (k, v, ka, va):
            x[~see.any(0)] = 0
        for h in range(bt.n_q):
            g, qq = h // bt.qg, q[at, h]
            with np.errstate(all="ignore"):
                s = np.where(see, qq @ k[:, g].T / 16.0, -np.inf)
                m = s.max(1, keepdims=True)
                p = np.where(see, np.exp(s - np.where(np.isfinite(m), m, 0)), 0.0)
                l = p.sum(1, keepdims=True)
                w = np.where(l > 0, p / l, 0.0)
                lse[at, h] = (m + np.log(l))[:, 0]
            out[at, h], Wt[at, h] = w @ v[:, g], w @ va[:, g]
            V[at, h] = np.sqrt((w * w) @ (va[:, g] ** 2))
            S[at, h] = (np.where(see, np.abs(qq) @ ka[:, g].T, 0) / 16.0).max(1)
            R[at, h] = np.sqrt(np.where(see, (qq * qq) @ (ka[:, g] ** 2).T, 0).max(1)) / 16.0
    if gate:
        x = 1.0 / (1.0 + np.exp(-bt.gate.astype(np.float64)))
        out, Wt, V = out * x, Wt * x, V * x
    return {"out": out, "lse": lse, "W": Wt, "V": V, "S": S, "R": R}


def elementwise(res, kernel, keys, out_bf16):
    """Every roundings' worst case: a weight's score twice (its own, and its row's sum), 2^-20 for exp2, its argument and
    the gate, 3 * keys * 2^-24 for the fp32 sums, the weight's parts; the output's own rounding."""
    rel = 2 * score_err(res["S"])[..., None] + 2.0 ** -20 + 3 * keys * 2.0 ** -24 + PART[kernel]
    return 1.01 * rel * res["W"] + (2.0 ** -8 * np.abs(res["out"]) if out_bf16 else 0.0) + 1e-30


def together(res, kernel, keys, out_bf16):
    """Bound of the root of the mean square error over a call's outputs, where roundings do not all point one way: of n of
    them, sqrt(n) times one. A score's 256 sums go by the root of its terms' squares (R); every row's weight has its own
    errors (its score's, twice, and its parts', each all that it can be), so they weigh the terms' squares (V). A rounding
    to bf16 is spread evenly over half a step, whose root mean square is at most 2^-8 / sqrt(3) of the value; a tenth
    more for how the values of a call happen to lie."""
    rms = lambda x: float(np.sqrt(np.mean(np.square(x))))  # noqa: E731
    fp32 = rms(2 * 16 * 2.0 ** -24 * res["R"][..., None] * res["V"]) + rms((2.0 ** -20 + 3 * np.sqrt(keys) * 2.0 ** -24) * res["W"])
    own = 1.1 * 2.0 ** -8 / np.sqrt(3) * rms(res["out"]) if out_bf16 else 0.0
    return float(np.hypot(PART[kernel] * rms(res["V"]), own)) + fp32 + 1e-30


def check(out, res, kernel, keys, out_bf16):
    """(largest error by its elementwise bound, root mean square error by its bound) of outputs [tokens][n_q][256]; both
    are at most 1 (and a NaN is not)."""
    err = np.abs(out - res["out"])
    if not err.size:
        return 0.0, 0.0
    return float(np.max(err / elementwise(res, kernel, keys, out_bf16))), float(np.sqrt(np.mean(err * err)) / together(res, kernel, keys, out_bf16))


def lse_tol(res, keys):
    return score_err(res["S"]) + 2.0 ** -20 * (1 + np.abs(np.where(np.isfinite(res["lse"]), res["lse"], 0))) + keys * 2.0 ** -24


def cut(res, lo, hi):
    return {n: x[lo:hi] for n, x in res.items()}


FLAT_ROWS, FLAT_TILES = 6, 8192      # (as in vx_paged_rows.h)


def tile_cap(max_pages, page, max_T, window, sink):
    cap = max_pages * page // 32
    return min(cap, (window + max_T) // 32 + 2 + -(-sink // 32)) if window else cap


def kernel_of(bt, out_bf16):
    """The attention kernel of a batch's call, by the rule that the header gives."""
    from vx27_amd import lib as L
    T = max(bt.new)
    rows, tiles = T * bt.qg, tile_cap(bt.max_pages, bt.page, T, bt.window, bt.sink)
    if rows <= (L.Q4_SPLIT_ROWS if out_bf16 else L.Q4_SPLIT_ROWS_F32) or (bt.N * bt.qg // 16 + bt.B) * bt.n_kv * tiles <= L.Q4_SPLIT_TILES:
        return "paged_q4_split"
    flat = -(-rows // 128) >= FLAT_ROWS and bt.B * bt.n_kv * tiles <= FLAT_TILES
    return "paged_rows_flat" if flat else "paged_rows_q4"


KERNELS = tuple(PART)


def run(at):
    """The attention kernel that a call ran."""
    at.ctx.prof_enable(True)
    at.call()
    ran = [k for k in KERNELS if at.ctx.prof_read(k)[0]]
    at.ctx.prof_enable(False)
    assert len(ran) == 1, ran
    return ran[0]


def widen(bt, pages=2100):
    """The batch with a page table of many more entries, behind the rows: the same rows, and a call that may see more."""
    bt.table = np.concatenate([bt.table, np.full((bt.B, pages), -7, np.int32)], axis=1)
    bt.max_pages += pages
    return bt
