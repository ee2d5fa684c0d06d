// Attention over a paged bf16 KV cache on gfx950: ragged batches of new
// tokens, causal, with an optional sliding window whose first rows (sinks)
// stay visible, an optional output gate, and optionally each row's softmax
// weights added up for eviction.
//
// Token at row i sees row j <= i if j > i - window (or no window) or
// j < n_sink:  s_ij = q_i.k_j / 16,  out_i = sum_j exp(s_ij - m_i) v_j / l_i.
//
// The query rows of one KV head are its group's heads of every token: row r
// is head r % qg of token r / qg.  All kernels work on tiles of 32 keys (a V
// block, so a tile lies in one page) and 16 query rows:
//   S^T[key][row] = K . Q^T     v_mfma_f32_16x16x32_bf16, two 16-key blocks.
//                               Row m of block r loads key 8(m/4) + 4r + m%4,
//                               so lane (g,n) ends with keys 8g..8g+7 of row n
//   O^T[dim][row] += V^T . P^T  16 MFMAs; lane (g,n)'s B operand is its own 8
//                               weights, the A operand 16 contiguous bytes of
//                               the dim-major V block.
#include "vx_paged_rows.h"

namespace {

__device__ __forceinline__ bf16x8_t load8_nt(const uint16_t *p) { return __builtin_nontemporal_load((const bf16x8_t *)p); }

// One wave's state for 16 query rows.
struct Rows {
    bf16x8_t q[8];
    floatx4_t o[16];
    float m, l;
};
__device__ __forceinline__ void rows_begin(const Args &a, const vx_pseq &s, int kvh, int r0, Rows &w) {
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15, r = r0 + n, t = row_tok(a, r);
    const bool live = t < s.T;
    const uint16_t *qp = a.q + (size_t)(s.start + (live ? t : 0)) * a.q_ts + (size_t)(live ? row_head(a, kvh, r, t) : 0) * a.q_hs + 8 * g;
#pragma unroll
    for (int k = 0; k < 8; k++) w.q[k] = load8(qp + 32 * k);
    if (!live) {
#pragma unroll
        for (int k = 0; k < 8; k++)
#pragma unroll
            for (int e = 0; e < 8; e++) w.q[k][e] = (__bf16)0.0f;
    }
#pragma unroll
    for (int d = 0; d < 16; d++) w.o[d] = (floatx4_t){0.f, 0.f, 0.f, 0.f};
    w.m = -INFINITY;
    w.l = 0.0f;
}

// Scores of 32 keys against 16 rows: lane (g,n) gets keys 8g + 0..7 of row n.
__device__ __forceinline__ void score_tile(const bf16x8_t (&ka)[8], const bf16x8_t (&kb)[8], const bf16x8_t (&q)[8], float (&s)[8]) {
    floatx4_t s0 = {0.f, 0.f, 0.f, 0.f}, s1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 8; k++) {
        s0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka[k], q[k], s0, 0, 0, 0);
        s1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kb[k], q[k], s1, 0, 0, 0);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        s[e] = s0[e];
        s[4 + e] = s1[e];
    }
}

// Online softmax and P V of one tile for R rows.  NP bf16 parts of each
// weight: three hold all 24 bits of it.  V of keys that no row sees is zeroed,
// so that what stale rows hold cannot get in.  `one`: the rows are of one token,
// so that all see the same keys.
template <int NP>
__device__ __forceinline__ void attend_tile(Rows &w, int R, bool one, const float (&s)[8], const vx_sight &v, int key0, bf16x8_t (&va)[16]) {
    const int g = (threadIdx.x & 63) >> 4;
    float x[8];
    float mt = -INFINITY;
    bool all = true;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        const bool see = v.sees(key0 + 8 * g + e);
        all &= see;
        x[e] = see ? s[e] : -INFINITY;
        mt = fmaxf(mt, x[e]);
    }
    mt = fmaxf(mt, __shfl_xor(mt, 16, 64));
    mt = fmaxf(mt, __shfl_xor(mt, 32, 64));
    // (nothing seen yet, or NaN scores alone: the reference is 0, so that those stay NaN)
    const float m_new = fmaxf(w.m, mt * SC2);
    const bool none = m_new == -INFINITY;
    const float ref = none ? 0.0f : m_new;
    const float alpha = none ? 1.0f : __builtin_amdgcn_exp2f(w.m - m_new);
    bf16x8_t p[NP];
    float ls = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        float pe = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], SC2, -ref));
        ls += pe;
#pragma unroll
        for (int k = 0; k < NP; k++) {
            p[k][e] = (__bf16)pe;
            pe -= (float)p[k][e];
        }
    }
    w.l = w.l * alpha + ls;
    w.m = m_new;
    if (__any(alpha != 1.0f)) {
#pragma unroll
        for (int d = 0; d < 16; d++) w.o[d] *= alpha;
    }
    if (!__all(all)) {
        const int lane = threadIdx.x & 63;
        const uint32_t group = (1u << R) - 1;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            // which of a lane group's rows see its key 8g + e
            const bool see = v.sees(key0 + 8 * g + e);
            const uint64_t seen = __ballot(see);
            const uint32_t mine = (uint32_t)(seen >> (16 * g)) & group;
            if (mine == 0) {
#pragma unroll
                for (int d = 0; d < 16; d++) va[d][e] = (__bf16)0.0f;
            }
            if (one || !__any(mine != 0 && mine != group)) continue;
            // A key that some rows see and others do not, with an infinite or
            // NaN value: 0 times that would reach the others.  Its values go
            // to the rows that see it by addition (any weight times an
            // infinity is one) and out of the product.
            bool odd = false;
#pragma unroll
            for (int d = 0; d < 16; d++) odd |= !is_finite(va[d][e]);
            uint64_t bad = __ballot(odd && mine);
            while (bad) {
                const int gk = __builtin_ctzll(bad) >> 4;
                bad &= ~(0xffffull << (16 * gk));
                const bool own = v.sees(key0 + 8 * gk + e);
#pragma unroll
                for (int d = 0; d < 16; d++)
#pragma unroll
                    for (int i = 0; i < 4; i++) {   // dim 16d + 4g + i is lane 4g + i's of the key's group
                        const float x = __shfl((float)va[d][e], 16 * gk + 4 * (lane >> 4) + i, 64);
                        if (own && !is_finite(x)) w.o[d][i] += x;
                    }
            }
#pragma unroll
            for (int d = 0; d < 16; d++)
                if (odd && !is_finite(va[d][e])) va[d][e] = (__bf16)0.0f;
        }
    }
#pragma unroll
    for (int k = 0; k < NP; k++)
#pragma unroll
        for (int d = 0; d < 16; d++) w.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va[d], p[k], w.o[d], 0, 0, 0);
}

// ---------------------------------------------------------------- decode
// At most 16 query rows a KV head.  The tiles of every (sequence, KV head)
// pair form one list; workgroup w of G takes tiles [w c, (w+1) c) of it, so
// a ragged batch is as even as an equal one.  A pair wholly inside one
// workgroup is finished there; the first and the last piece of a
// workgroup's range may be parts of a pair and go to its two partial slots,
// which paged_join merges in order.
//
// Bound by the stream of K and V, 1 KiB a row and KV head, which two
// workgroups a CU (8 waves with 24 KiB of loads in flight each) take at 6.6
// TB/s: 4 x 131072 rows, 2.15 GB, in 325 us (one workgroup a CU: 327), a
// plain read of as much 298.  Short calls are two launches and the latencies
// of the table, the tiles and the join: 12 us for one sequence of 1000 rows.
// (253 VGPRs, of the 256 that two workgroups a CU leave; some 90 scalars do not
// fit the SGPRs and are kept in lanes of them.)
//
__global__ __launch_bounds__(256, 2) void paged_split(Args a) {
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, n = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    __shared__ __attribute__((aligned(16))) float s_o[4][16 * HDG];
    __shared__ float s_m[4][16], s_l[4][16];
    const Units un = units_of<false>(a, gridDim.x);
    const int u0 = blockIdx.x * un.chunk, u1 = min(u0 + un.chunk, un.total);
    if (u0 >= u1) return;
    int b = units_find(a, un, u0);
    const int krow0 = 8 * (n >> 2) + (n & 3);
    vx_pseq s;
    vx_tiles tl;
    int before = units_before<false>(a, un, b, s, tl);
    for (int u = u0; u < u1;) {
        if (u >= before + tl.nt * a.p.n_kv) {
            before += tl.nt * a.p.n_kv;
            b++;
            if (a.p.B <= 64) units_before<false>(a, un, b, s, tl);
            else seq_units<false>(a, b, s, tl);
            continue;
        }
        const int kvh = (u - before) / tl.nt, i0 = (u - before) - kvh * tl.nt;
        const int cnt = min(tl.nt - i0, u1 - u);
        const int R = s.T * a.qg;
        Rows w;
        rows_begin(a, s, kvh, 0, w);
        const vx_sight v = sight_of(a, s, n);
        for (int i = i0 + wave; i < i0 + cnt; i += 4) {
            const int tile = tl.at(i), key0 = tile * TILE;
            const int page = vx_paged_page(a.p, b, key0), at = key0 - vx_page_slot(a.p, key0) * a.p.page_size;
            const uint16_t *kr0 = a.k_pages + vx_k_index(a.p.n_kv, a.p.page_size, page, kvh, at + krow0, 8 * g);
            const uint16_t *vt = a.v_pages + vx_v_index(a.p.n_kv, a.p.page_size, page, kvh, at, n) + 8 * g;
            bf16x8_t ka[8], kb[8], va[16];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                ka[k] = load8_nt(kr0 + 32 * k);
                kb[k] = load8_nt(kr0 + 4 * HDG + 32 * k);
            }
#pragma unroll
            for (int d = 0; d < 16; d++) va[d] = load8_nt(vt + (size_t)d * 16 * TILE);
            float sc[8];
            score_tile(ka, kb, w.q, sc);
            if (a.stash && n < R) {
                float *st = a.stash + (((size_t)b * a.p.n_kv + kvh) * a.part_rows + n) * ((size_t)a.tile_cap * TILE) + (size_t)i * TILE + 8 * g;
                *(float4 *)st = make_float4(sc[0], sc[1], sc[2], sc[3]);
                *(float4 *)(st + 4) = make_float4(sc[4], sc[5], sc[6], sc[7]);
            }
            attend_tile<3>(w, R, s.T == 1, sc, v, key0, va);
        }
        w.l += __shfl_xor(w.l, 16, 64);
        w.l += __shfl_xor(w.l, 32, 64);
        // the four waves' results through LDS (16-byte units swizzled by the row)
        if (n < R) {
#pragma unroll
            for (int d = 0; d < 16; d++) *(floatx4_t *)&s_o[wave][n * HDG + (((4 * d + g) ^ n) << 2)] = w.o[d];
            if (g == 0) {
                s_m[wave][n] = w.m;
                s_l[wave][n] = w.l;
            }
        }
        __syncthreads();
        // wave w merges rows w, w + 4, ..., lane L dims 4L .. 4L + 3
        const bool whole = cnt == tl.nt;
        const int slot = 2 * blockIdx.x + (u == u0 ? 0 : 1);
        for (int r = wave; r < R; r += 4) {
            const int t = row_tok(a, r), tok = s.start + t, h = row_head(a, kvh, r, t);
            float4 gt = make_float4(0.f, 0.f, 0.f, 0.f);
            if (whole && a.gate) gt = gate_row(a, tok, h);
            float m[4], l[4];
            float4 o[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                m[k] = s_m[k][r];
                l[k] = s_l[k][r];
                o[k] = *(const float4 *)&s_o[k][r * HDG + ((lane ^ r) << 2)];
            }
            const float M = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
            float L = 0.0f;
            float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < 4; k++) add_part(O, L, o[k], l[k], m[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[k] - M));
            if (whole) {
                row_finish(a, tok, h, O, M, L, gt);
            } else {
                *(float4 *)(a.part_o + ((size_t)slot * a.part_rows + r) * HDG + 4 * lane) = O;
                if (lane == 0) a.part_ml[(size_t)slot * a.part_rows + r] = make_float2(M, L);
            }
        }
        __syncthreads();
        u += cnt;
    }
}

// grid (tile_cap / 8, n_kv, B), block 256: one thread per key; the stashed
// scores become weights, summed over the rows that see the key.  (The scores
// are kept, 4 bytes a row of queries and keys against the 512 of K that a
// second pass would read: 8 us of the 63 for 16 ragged sequences of 8190 rows.)
__global__ __launch_bounds__(256) void paged_weigh(Args a) {
    const int kvh = blockIdx.y, b = blockIdx.z;
    const int i = blockIdx.x * 8 + (threadIdx.x >> 5);
    const vx_pseq s = vx_paged_seq(a.p, b);
    const vx_tiles tl = tiles_of(a, s, 0, s.T - 1);
    if (i >= tl.nt) return;
    const int j = tl.at(i) * TILE + (threadIdx.x & 31);
    const size_t stride = (size_t)a.tile_cap * TILE;
    const float *st = a.stash + ((size_t)b * a.p.n_kv + kvh) * a.part_rows * stride + (size_t)i * TILE + (threadIdx.x & 31);
    float sum = 0.0f;
    bool any = false;
    for (int r = 0; r < s.T * a.qg; r++) {
        if (!sight_of(a, s, r).sees(j)) continue;
        const int t = row_tok(a, r);
        const float2 ml = a.stat[(size_t)(s.start + t) * a.n_q + row_head(a, kvh, r, t)];
        sum += __builtin_amdgcn_exp2f(__builtin_fmaf(st[r * stride], SC2, -ml.x)) * ml.y;
        any = true;
    }
    if (any) a.acc[((size_t)b * a.p.n_kv + kvh) * a.acc_stride + j] += sum;
}

// Every row's weights of the tile kernel's tokens, the scores formed again
// (the tile kernel has a row's maximum and sum only at its end).  grid
// (tile_cap / 8, n_kv, B), block 256: wave w keeps two key blocks of the tile
// list in registers as K operands, and the 32-row tiles of queries that see
// any of the workgroup's keys pass through LDS, one ahead.  A lane's sums are
// over its row of each tile; at the end the 32 lanes of a key are added up.
// One workgroup owns a key, so the order of the sums is fixed.
// 54 us for 4 x 64 tokens over 9000 rows, 28 GFLOP; 576 workgroups for 512
// places.  (One key block a wave, four workgroups a CU: 85 us, as the queries
// are then read from LDS twice as often.)
constexpr int QT = 32, QBUF = QT * HDG * 2;
__global__ __launch_bounds__(256, 2) void paged_rows_weigh(Args a) {
    __shared__ __attribute__((aligned(16))) char sq[2][QBUF];
    const int kvh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63, g = lane >> 5, n = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const vx_pseq s = vx_paged_seq(a.p, b);
    const vx_tiles tl = tiles_of(a, s, 0, s.T - 1);
    const int first = blockIdx.x * 8;
    if (first >= tl.nt) return;
    // the tokens that see any of the workgroup's keys lo .. hi
    const int lo = tl.at(first) * TILE, hi = tl.at(min(first + 8, tl.nt) - 1) * TILE + TILE - 1;
    const int t0 = max(lo - s.row0, 0);
    const int t1 = a.window && lo >= a.n_sink ? (int)min((int64_t)s.T - 1, (int64_t)hi + a.window - 1 - s.row0) : s.T - 1;
    const int ra = t0 * a.qg, rz = (t1 + 1) * a.qg, R = s.T * a.qg;   // query rows ra .. rz - 1

    int key0[2];
    bf16x8_t kf[2][16];
#pragma unroll
    for (int kb = 0; kb < 2; kb++) {
        const int i = first + 2 * wave + kb, key = tl.at(min(i, tl.nt - 1)) * TILE;
        key0[kb] = i < tl.nt ? key : -1;
        const int page = vx_paged_page(a.p, b, key), krow = 16 * (n >> 4) + 8 * ((n >> 2) & 1) + 4 * ((n >> 3) & 1) + (n & 3);
        const uint16_t *kp = a.k_pages + vx_k_index(a.p.n_kv, a.p.page_size, page, kvh, key - vx_page_slot(a.p, key) * a.p.page_size + krow, 8 * g);
#pragma unroll
        for (int k = 0; k < 16; k++) kf[kb][k] = load8(kp + 16 * k);
    }
    float sum[32];
#pragma unroll
    for (int i = 0; i < 32; i++) sum[i] = 0.0f;

    // Queries r .. r + 31 into a buffer: 2 rows a load, 16-byte unit u of row
    // q at slot u ^ (q & 7) (rows past the last: the last again)
    auto stage = [&](int r, int buf) {
        const int tb = row_tok(a, min(r, R - 1));
        const uint16_t *base = vx_uniform_ptr(a.q + (size_t)(s.start + tb) * a.q_ts + (size_t)kvh * a.qg * a.q_hs);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int q = wave * 8 + 2 * j + (lane >> 5), row = min(r + q, R - 1), t = row_tok(a, row);
            const uint32_t off = (uint32_t)(((size_t)(t - tb) * a.q_ts + (size_t)(row - t * a.qg) * a.q_hs) * 2) + (((lane & 31) ^ (q & 7)) << 4);
            vx_dma16(base, off, vx_lds_addr(sq[buf]) + (wave * 8 + 2 * j) * 512);
        }
    };
    auto stat_of = [&](int r) {
        const int row = min(r + n, R - 1), t = row_tok(a, row);
        return a.stat[(size_t)(s.start + t) * a.n_q + row_head(a, kvh, row, t)];
    };
    if (ra < rz) {
        float2 st = stat_of(ra);
        stage(ra, 0);
        int buf = 0;
        for (int r = ra; r < rz; r += QT, buf ^= 1) {
            __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
            vx_lds_barrier();
            const float2 ml = st;
            st = stat_of(min(r + QT, rz - 1));
            if (r + QT < rz) stage(r + QT, buf ^ 1);
            const int row = r + n;
            vx_sight v = vx_paged_sight(s, row_tok(a, min(row, R - 1)), a.window, a.n_sink);
            if (row >= rz) v.i = -1;
            floatx16_t S[2];
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int i = 0; i < 16; i++) S[kb][i] = 0.0f;
            const char *qrow = sq[buf] + n * 512;
#pragma unroll
            for (int k = 0; k < 16; k++) {
                const bf16x8_t qf = lds8(qrow + (((2 * k + g) ^ (n & 7)) << 4));
#pragma unroll
                for (int kb = 0; kb < 2; kb++) S[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[kb][k], qf, S[kb], 0, 0, 0);
            }
#pragma unroll
            for (int kb = 0; kb < 2; kb++) {
                const uint32_t bits = key0[kb] < 0 ? 0u : v.block(key0[kb]);
                if (__all(bits == 0xffffffffu)) {
#pragma unroll
                    for (int i = 0; i < 16; i++) sum[16 * kb + i] += __builtin_amdgcn_exp2f(__builtin_fmaf(S[kb][i], SC2, -ml.x)) * ml.y;
                } else {
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(S[kb][i], SC2, -ml.x)) * ml.y;
                        sum[16 * kb + i] += (bits >> (8 * g)) & (1u << (16 * (i >> 3) + (i & 7))) ? p : 0.0f;
                    }
                }
            }
        }
    }
    // over the 32 lanes: halves of the values change sides until lane n has value n
#pragma unroll
    for (int off = 16, half = 16; off >= 1; off >>= 1, half >>= 1)
#pragma unroll
        for (int i = 0; i < half; i++) {
            const bool up = n & off;
            const float keep = up ? sum[i + half] : sum[i], send = up ? sum[i] : sum[i + half];
            sum[i] = keep + __shfl_xor(send, off, 64);
        }
    vx_sight any = vx_paged_sight(s, 0, a.window, a.n_sink);
    if (any.i < 0) any.lo = 0;
    any.i = s.len - 1;
    const int kb = n >> 4, i = n & 15, key = (kb ? key0[1] : key0[0]) + 16 * (i >> 3) + 8 * g + (i & 7);
    if ((kb ? key0[1] : key0[0]) >= 0 && any.sees(key)) a.acc[((size_t)b * a.p.n_kv + kvh) * a.acc_stride + key] += sum[0];
}

}  // namespace

extern "C" int vx27_hip_paged_attn(vx27_hip_ctx *ctx, const vx27_paged_attn_desc *d) {
    static const char who[] = "vx27_hip_paged_attn";
    VX_REQUIRE(d != nullptr, "%s: null descriptor", who);
    Args a = {};
    const int todo = attn_fill(who, ctx, d, a);
    if (todo <= 0) return todo;
    const int64_t tile_cap = a.tile_cap;
    const int rows = d->max_T * a.qg;
    const size_t stat_bytes = d->acc ? ((size_t)d->n_tok * d->n_q * sizeof(float2) + 255) / 256 * 256 : 0;
    if (rows <= 16) {
        VX_REQUIRE((int64_t)d->B * d->n_kv * tile_cap < MOST_UNITS, "%s: more than 2^31 key tiles (B=%d n_kv=%d, %lld tiles each)", who,
                   d->B, d->n_kv, (long long)tile_cap);
        // (one sequence of 1000 rows: 13.1 us with 4, 12.1 with 2, 11.9 with 1; of 3000: 16.4, 13.6, 15.8; of 8000: 18.8, 19.5, 19.5)
        a.min_tiles = 2;
        const int64_t most = ((int64_t)d->B * d->n_kv * tile_cap + a.min_tiles - 1) / a.min_tiles;
        const int grid = (int)std::min<int64_t>(most, 2 * ctx->n_cu);
        a.part_rows = rows;
        const size_t n_part = (size_t)2 * grid * rows;
        const size_t o_bytes = n_part * HDG * 4, ml_bytes = (n_part * sizeof(float2) + 255) / 256 * 256;
        const size_t st_bytes = d->acc ? (size_t)d->B * d->n_kv * rows * tile_cap * TILE * 4 : 0;
        const size_t before_bytes = d->B > 64 ? ((size_t)d->B + 1) * sizeof(int) : 0;
        void *scr;
        if (vx_ctx_scratch(ctx, o_bytes + ml_bytes + stat_bytes + st_bytes + before_bytes, &scr)) return -1;
        a.part_o = (float *)scr;
        a.part_ml = (float2 *)((char *)scr + o_bytes);
        a.stat = d->acc ? (float2 *)((char *)scr + o_bytes + ml_bytes) : nullptr;
        a.stash = d->acc ? (float *)((char *)scr + o_bytes + ml_bytes + stat_bytes) : nullptr;
        a.before = d->B > 64 ? (int *)((char *)scr + o_bytes + ml_bytes + stat_bytes + st_bytes) : nullptr;
        if (a.before) VX_LAUNCH_NAMED(ctx, "paged_units", (paged_units<false, false>), dim3(1), dim3(1024), a);
        VX_LAUNCH(ctx, paged_split, dim3(grid), dim3(256), a);
        VX_LAUNCH_NAMED(ctx, "paged_join", (paged_join<false>), dim3(rows, d->n_kv, d->B), dim3(256), a, grid);
        if (d->acc) VX_LAUNCH(ctx, paged_weigh, dim3((a.tile_cap + 7) / 8, d->n_kv, d->B), dim3(256), a);
        return 0;
    }
    // (a 32-row tile's queries are addressed by 32-bit offsets from its first)
    VX_REQUIRE(!d->acc || (a.q_ts < (1u << 26) && a.q_hs < (1u << 26)), "%s: q strides past 2^26 elements with acc (got %zu, %zu)", who, a.q_ts, a.q_hs);
    if (rows_launch<false>(who, ctx, d, a, rows, stat_bytes)) return -1;
    if (d->acc) VX_LAUNCH(ctx, paged_rows_weigh, dim3((a.tile_cap + 7) / 8, d->n_kv, d->B), dim3(256), a);
    return 0;
}
