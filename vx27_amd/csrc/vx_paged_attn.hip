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
#include <math.h>

#include <algorithm>

#include "vx_lds.h"
#include "vx_paged.h"

namespace {

constexpr int HDG = VX_GQA_HD, TILE = VX_PG_TILE;
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx4_t __attribute__((ext_vector_type(4)));
constexpr float SC2 = 0.0625f * 1.4426950408889634f;   // 1/sqrt(256) * log2(e): scores in the exp2 domain

struct RowPlan;
struct RowPiece;
struct RowJoin;
struct Args {
    vx_paged p;
    int n_q, qg, window, n_sink;
    uint32_t qg_magic;           // floor(2^32 / qg) + 1: row / qg as a high product (rows < 2^28), 0 for qg = 1
    const uint16_t *q;
    size_t q_ts, q_hs;
    const uint16_t *k_pages, *v_pages;
    const void *gate;            // NULL: no output gate
    int gate_bf16;
    size_t g_ts, g_hs;
    void *out;
    int out_bf16;
    float *lse;                  // optional
    float *acc;                  // optional
    size_t acc_stride;
    float2 *stat;                // with acc: [n_tok][n_q] (max in the exp2 domain, 1 / sum)
    // decode
    int min_tiles;               // tiles a workgroup takes at least
    int tile_cap;                // most tiles any sequence can have
    float *part_o;               // [2 grid][max rows][256]
    float2 *part_ml;             // [2 grid][max rows]
    int part_rows;
    int *before;                 // B > 64: [B + 1] units before each sequence
    // tiles (scratch)
    int cus;
    RowPlan *plan;
    RowPiece *pieces;
    RowJoin *joins;
    float *stash;                // with acc: raw scores [B][n_kv][max rows][tile_cap * 32]
};

// The token, and the query head, of query row r of KV head kvh.
__device__ __forceinline__ int row_tok(const Args &a, int r) { return a.qg_magic ? (int)__umulhi((uint32_t)r, a.qg_magic) : r; }
__device__ __forceinline__ int row_head(const Args &a, int kvh, int r, int t) { return kvh * a.qg + r - t * a.qg; }

__device__ __forceinline__ vx_tiles tiles_of(const Args &a, const vx_pseq &s, int t0, int t1) {
    return vx_paged_tiles(s, t0, t1, a.window, a.n_sink);
}
// What query row r of a sequence sees (rows past the last see nothing).
__device__ __forceinline__ vx_sight sight_of(const Args &a, const vx_pseq &s, int r) {
    return vx_paged_sight(s, row_tok(a, r), a.window, a.n_sink);
}

__device__ __forceinline__ bf16x8_t load8(const uint16_t *p) { return *(const bf16x8_t *)p; }
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

__device__ __forceinline__ bool is_finite(float x) { return __builtin_fabsf(x) < INFINITY; }

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

// A row's lse, and its reference and 1 / sum for the weights' pass.  SHIFT: the
// reference lies that far above a maximum; the weights' pass takes the maximum,
// so that its arguments are small (the difference as it was rounded: exact
// below 2^24, and none where a last place is larger).
template <int SHIFT>
__device__ __forceinline__ void stat_store(const Args &a, int tok, int h, float m, float L) {
    const size_t at = (size_t)tok * a.n_q + h;
    if (a.lse) a.lse[at] = L > 0.0f || L != L ? (m + log2f(L)) * 0.6931471805599453f : -INFINITY;
    // (a row that weighs nothing: from 0, so that scores of -inf become weights of 0 and not NaN)
    const float ref = m - SHIFT;
    if (a.stat) a.stat[at] = L > 0.0f || L != L ? make_float2(ref, (SHIFT ? __builtin_amdgcn_exp2f(ref - m) : 1.0f) / L) : make_float2(0.0f, 0.0f);
}

// hardware round-to-nearest-even pack (v_cvt_pk_bf16_f32)
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    const bf16x2_t v = (bf16x2_t){(__bf16)x, (__bf16)y};
    return __builtin_bit_cast(uint32_t, v);
}
// A query row's gate logits across a wave (lane L: dims 4L..4L+3).
__device__ __forceinline__ float4 gate_row(const Args &a, int tok, int h) {
    const size_t at = (size_t)tok * a.g_ts + (size_t)h * a.g_hs + 4 * (threadIdx.x & 63);
    if (!a.gate_bf16) return *(const float4 *)((const float *)a.gate + at);
    const uint2 u = *(const uint2 *)((const uint16_t *)a.gate + at);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ void row_write(const Args &a, int tok, int h, float4 r) {
    const size_t at = ((size_t)tok * a.n_q + h) * HDG + 4 * (threadIdx.x & 63);
    if (a.out_bf16) *(uint2 *)((uint16_t *)a.out + at) = make_uint2(pack2(r.x, r.y), pack2(r.z, r.w));
    else *(float4 *)((float *)a.out + at) = r;
}
// (hardware exp2 and reciprocal: one part in 2^22, below the rounding of the
// tile kernel's weights)
__device__ __forceinline__ float fast_sigmoid(float y) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(y * -1.4426950408889634f)); }
// A finished query row of the tile kernel across a wave, gated by logits x.
__device__ __forceinline__ void row_store(const Args &a, int tok, int h, float4 r, float4 x) {
    if (a.gate) {
        r.x *= fast_sigmoid(x.x); r.y *= fast_sigmoid(x.y); r.z *= fast_sigmoid(x.z); r.w *= fast_sigmoid(x.w);
    }
    row_write(a, tok, h, r);
}
// The same from a decode row's sums (fp32 accuracy), with its statistics.
__device__ __forceinline__ void row_finish(const Args &a, int tok, int h, float4 O, float M, float L, float4 x) {
    const bool some = L > 0.0f || L != L;   // (0 where nothing was seen)
    float4 r = some ? make_float4(O.x / L, O.y / L, O.z / L, O.w / L) : make_float4(0.f, 0.f, 0.f, 0.f);
    if (a.gate) {
        auto sg = [](float y) { return 1.0f / (1.0f + expf(-y)); };
        r.x *= sg(x.x); r.y *= sg(x.y); r.z *= sg(x.z); r.w *= sg(x.w);
    }
    row_write(a, tok, h, r);
    if ((threadIdx.x & 63) == 0) stat_store<0>(a, tok, h, M, L);
}
__device__ __forceinline__ void add_part(float4 &O, float &L, float4 o, float l, float w) {
    L += l * w;
    O.x += o.x * w; O.y += o.y * w; O.z += o.z * w; O.w += o.w * w;
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
// 16 rows are what one MFMA tile holds, so this form ends there: a third token
// of 6 heads goes to the tiles below (4 x 131072 rows: 328 us for two tokens
// a sequence, 377 for three there; one of 1000 rows: 14 and 26).
// The list of a call's tiles: up to 64 sequences are held one a lane and read
// once; of more, paged_units adds up the units before each first (each
// workgroup doing so for itself took 3.2 ms for 4096 sequences of 100 rows).
struct Units {
    vx_pseq s;          // of sequence `lane` (B <= 64)
    vx_tiles t;
    int upto;           // units of sequences 0 .. lane
    int total, chunk;
};
__device__ __forceinline__ int seq_units(const Args &a, int b, vx_pseq &s, vx_tiles &t) {
    s = vx_paged_seq(a.p, b);
    t = tiles_of(a, s, 0, s.T - 1);
    return t.nt * a.p.n_kv;
}
__device__ __forceinline__ Units units_of(const Args &a, int grid) {
    const int lane = threadIdx.x & 63;
    Units u;
    if (a.p.B <= 64) {
        const int n = seq_units(a, min(lane, a.p.B - 1), u.s, u.t);
        u.upto = vx_wave_scan(lane < a.p.B ? n : 0);
        u.total = __builtin_amdgcn_readlane(u.upto, 63);
    } else {
        u.total = a.before[a.p.B];
    }
    u.chunk = max((u.total + grid - 1) / grid, a.min_tiles);
    return u;
}
// Sequence b: itself, its tiles, and the units before it.
__device__ __forceinline__ int units_before(const Args &a, const Units &u, int b, vx_pseq &s, vx_tiles &t) {
    if (a.p.B <= 64) {
        auto get = [&](int x) { return __builtin_amdgcn_readlane(x, b); };
        s = {get(u.s.start), get(u.s.T), get(u.s.len), get(u.s.row0)};
        t = {get(u.t.st), get(u.t.fm), get(u.t.nt)};
        return get(u.upto) - t.nt * a.p.n_kv;
    }
    seq_units(a, b, s, t);
    return a.before[b];
}
// The sequence of unit x < total: the last with at most x units before it,
// among 64 of them at a time.
__device__ __forceinline__ int units_find(const Args &a, const Units &u, int x) {
    const int lane = threadIdx.x & 63;
    if (a.p.B <= 64) return __builtin_ctzll(__ballot(u.upto > x));
    int b = 0;
    for (int n = a.p.B; n > 1;) {
        const int step = (n + 63) / 64, at = lane * step;
        const uint64_t le = __ballot(at < n && a.before[b + min(at, n - 1)] <= x);
        const int k = le ? 63 - __builtin_clzll(le) : 0;
        b += k * step;
        n = min(step, n - k * step);
    }
    return b;
}

// grid 1, block 1024: the units before each sequence, and in all.
__global__ __launch_bounds__(1024) void paged_units(Args a) {
    __shared__ int s_sum[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (a.p.B + 1023) / 1024, b0 = min(tid * per, a.p.B), b1 = min(b0 + per, a.p.B);
    vx_pseq s;
    vx_tiles t;
    int sum = 0;
    for (int b = b0; b < b1; b++) sum += seq_units(a, b, s, t);
    int at = vx_wave_scan(sum);
    if (lane == 63) s_sum[wave] = at;
    __syncthreads();
    for (int w = 0; w < wave; w++) at += s_sum[w];
    if (tid == 1023) a.before[a.p.B] = at;
    at -= sum;
    for (int b = b0; b < b1; b++) {
        a.before[b] = at;
        at += seq_units(a, b, s, t);
    }
}

__global__ __launch_bounds__(256, 2) void paged_split(Args a) {
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, n = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    __shared__ __attribute__((aligned(16))) float s_o[4][16 * HDG];
    __shared__ float s_m[4][16], s_l[4][16];
    const Units un = units_of(a, gridDim.x);
    const int u0 = blockIdx.x * un.chunk, u1 = min(u0 + un.chunk, un.total);
    if (u0 >= u1) return;
    int b = units_find(a, un, u0);
    const int krow0 = 8 * (n >> 2) + (n & 3);
    vx_pseq s;
    vx_tiles tl;
    int before = units_before(a, un, b, s, tl);
    for (int u = u0; u < u1;) {
        if (u >= before + tl.nt * a.p.n_kv) {
            before += tl.nt * a.p.n_kv;
            b++;
            if (a.p.B <= 64) units_before(a, un, b, s, tl);
            else seq_units(a, b, s, tl);
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

// grid (most rows, n_kv, B), block 256 (4-7 us): merges the parts of one query row, in
// their order: wave w takes parts w, w + 4, ..., eight in flight; a row of a
// sequence without rows gets 0.
__global__ __launch_bounds__(256) void paged_join(Args a, int grid) {
    const int r = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Units un = units_of(a, grid);
    vx_pseq s;
    vx_tiles tl;
    const int p0 = units_before(a, un, b, s, tl) + kvh * tl.nt, p1 = p0 + tl.nt;
    if (r >= s.T * a.qg) return;
    const int t = row_tok(a, r), tok = s.start + t, h = row_head(a, kvh, r, t);
    const int g0 = p0 / un.chunk, g1 = (p1 - 1) / un.chunk;
    if (tl.nt > 0 && g0 == g1) return;
    float4 gt = make_float4(0.f, 0.f, 0.f, 0.f);
    if (wave == 0 && a.gate) gt = gate_row(a, tok, h);
    __shared__ float4 s_o[4][64];
    __shared__ float s_m[4], s_l[4];
    float M = -INFINITY, L = 0.0f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int NP = 8;
    for (int w0 = g0 + wave; w0 <= g1 && tl.nt > 0; w0 += 4 * NP) {
        float2 ml[NP];
        float4 o[NP];
#pragma unroll
        for (int k = 0; k < NP; k++) {   // (past the last part: the last again, weighed 0)
            const int w = min(w0 + 4 * k, g1);
            const size_t pi = (size_t)(2 * w + (w == g0 && p0 != w * un.chunk ? 1 : 0)) * a.part_rows + r;
            ml[k] = a.part_ml[pi];
            o[k] = ((const float4 *)(a.part_o + pi * HDG))[lane];
        }
        float mn = M;
#pragma unroll
        for (int k = 0; k < NP; k++) {
            if (w0 + 4 * k > g1) ml[k].x = -INFINITY;
            mn = fmaxf(mn, ml[k].x);
        }
        const float ref = mn == -INFINITY ? 0.0f : mn;   // (parts of NaN scores alone stay NaN)
        const float sa = __builtin_amdgcn_exp2f(M - ref);
        L *= sa;
        O.x *= sa; O.y *= sa; O.z *= sa; O.w *= sa;
#pragma unroll
        for (int k = 0; k < NP; k++) add_part(O, L, o[k], ml[k].y, __builtin_amdgcn_exp2f(ml[k].x - ref));
        M = mn;
    }
    s_o[wave][lane] = O;
    if (lane == 0) {
        s_m[wave] = M;
        s_l[wave] = L;
    }
    __syncthreads();
    if (wave) return;
    const float Mt = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    L = 0.0f;
    O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < 4; k++) add_part(O, L, s_o[k][lane], s_l[k], s_m[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_m[k] - Mt));
    row_finish(a, tok, h, O, Mt, L, gt);
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

// ------------------------------------------------------------------ tiles
// More than 16 query rows a KV head: 128 rows (tokens x the group's heads,
// packed) against 64 keys a step, in 4 waves, one per SIMD, of 32 rows each
// (v_mfma_f32_32x32x16_bf16): S^T[key][row] = K . Q^T, O^T[dim][row] += V^T .
// P^T.
//
// Row m of a K operand holds key 16 (m/16) + 8 (m/4 % 2) + 4 (m/8 % 2) + m%4
// of its 32-key block, so that the C layout of S^T leaves lane (g,n) with
// keys 16 s + 8 g + 0..7 of row n in registers 8 s .. 8 s + 7: the B operand
// of O^T += V^T P^T as it stands.  Row maxima, rescales and sums are then one
// value a lane.
//
// A step's two key blocks are consecutive entries of the tile list, so a
// sink block and the window's first block make a step without a gap.
//
// Bound by the MFMAs' issue beside the softmax: a step of 64 MFMAs a wave takes
// about 2.15 us (3900 cycles at the 1.8 GHz that the chip then holds; the MFMAs
// alone are 2050), and a piece another 13 us for its first loads, its first
// scores and its output, which nothing overlaps.  8192 tokens of 24 heads under
// a window of 1024: 300 us, 0.65 PFLOP/s of what the rows see.  (Neither is the
// card's limit: gqp_attn_pp, of the same tile, takes 1.75 us a step.)
// Weights are one bf16 part, as there: three would triple the second half of
// the step's MFMAs.
//
// (Measured against it: waves of 64 rows x one key block, and 128 dims of O,
// which read half as much from LDS but exchange weights and maxima through it
// and meet twice a step: 315 us; a persistent loop over the pieces spilled.)
constexpr int TR = 128;                      // query rows of a workgroup
constexpr int HALF = TILE * HDG * 2;         // bytes of one key block of K or of V
typedef float floatx16_t __attribute__((ext_vector_type(16)));
// A row's reference lies 2^16 above its first block's maximum and moves once a
// later one is past it: weights then start at 2^-16 and stay below 1, so that
// sums and O are bounded as without a reference that stays behind (rows times
// |v|), and a rescale of O (400 instructions a wave) hardly ever runs.  (2^8
// takes the windowed prompt from 298 to 326 us: of a first step of sinks and
// the window's edge a row sees few keys.)
constexpr int LAZY = 16;

struct TileSmem {
    char k[2][2 * HALF], v[2][2 * HALF];     // [buffer][key block]
    int piece;
    int odd;                                 // some value was infinite or NaN where not every row sees it
};

// vx_dma16 with a constant offset, which counts in memory and in LDS.
template <int OFF>
__device__ __forceinline__ void dma16(const void *base, uint32_t off, uint32_t lds) {
    uint32_t saved;
    __asm__ volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %3\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %1, %2 offset:%4\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "v"(off), "s"(base), "s"(lds), "n"(OFF)
        : "memory");
}
__device__ __forceinline__ int kswz(int r) { return (r & 3) | ((r >> 1) & 12); }
__device__ __forceinline__ bf16x8_t lds8(const char *p) { return *(const bf16x8_t *)p; }

// An item is a row tile of a sequence and KV head.  One workgroup of
// paged_plan lists the items (by KV head, sequence, last rows first), cut
// into pieces of at most `limit` steps where there are too few items for the
// CUs; paged_rows runs one workgroup a piece, and the parts of a cut item go
// to slots that paged_rows_join adds up in order.
struct RowPiece {
    int b, kvh, r0, c0, c1, slot;             // steps c0 .. c1 - 1 of its list; slot -1: the whole item
    vx_pseq s;                                // its sequence
    int pad[2];
};
struct RowJoin {
    int b, kvh, r0, slot, parts, pad[3];
};
struct RowPlan {
    int pieces, joins;
    int heads[8];                             // pieces taken of each XCD's run
};
__device__ __forceinline__ int row_tiles(const Args &a, const vx_pseq &s) { return (s.T * a.qg + TR - 1) / TR; }
// Steps of entry e = b * n_rt + k of one KV head, row tile k from the end of
// sequence b (rows that see nothing: one, for their output); 0 past its rows.
__device__ __forceinline__ int entry_steps(const Args &a, int n_rt, int e, int &b, int &r0, vx_pseq &s) {
    b = e / n_rt;
    s = vx_paged_seq(a.p, b);
    const int rt = row_tiles(a, s) - 1 - (e - b * n_rt);
    if (rt < 0) return 0;
    r0 = rt * TR;
    const vx_tiles tl = tiles_of(a, s, row_tok(a, r0), row_tok(a, min(r0 + TR, s.T * a.qg) - 1));
    return max(1, (tl.nt + 1) / 2);
}

// grid 1, block 1024 (6 us; 9 for the 1536 items of an 8192-token prompt).  It
// goes by B * n_rt entries, n_rt of the longest token range: 256 decoding
// sequences beside a chunk of 8192 tokens 105 us, 4096 beside 4096 1.8 ms.
constexpr int PLAN = 1024;
__global__ __launch_bounds__(PLAN) void paged_plan(Args a, int n_rt, int n_cu, int max_pieces) {
    __shared__ int64_t s_steps[PLAN / 64];
    __shared__ int s_sum[3][PLAN / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int E = a.p.B * n_rt, per = (E + PLAN - 1) / PLAN, e0 = min(tid * per, E);
    int e1 = min(e0 + per, E);
    int b = 0, r0 = 0, items = 0, n0 = 0;
    vx_pseq s = {};
    int64_t steps = 0;
    for (int e = e0; e < e1; e++) {
        n0 = entry_steps(a, n_rt, e, b, r0, s);
        steps += n0;
        items += n0 > 0;
    }
    // (a thread's only entry is not looked up again)
    auto steps_of = [&](int e) { return per == 1 ? n0 : entry_steps(a, n_rt, e, b, r0, s); };
    items = vx_wave_scan(items);
    for (int off = 32; off >= 1; off >>= 1) steps += __shfl_xor(steps, off, 64);
    if (lane == 63) {
        s_steps[wave] = steps;
        s_sum[0][wave] = items;
    }
    __syncthreads();
    steps = items = 0;
#pragma unroll
    for (int w = 0; w < PLAN / 64; w++) {
        steps += s_steps[w];
        items += s_sum[0][w];
    }
    // As many rounds of the CUs as leave at least half a round for cuts, and
    // pieces short enough to fill them: at most 3/2 n_cu cuts.
    const int64_t I = (int64_t)items * a.p.n_kv, room = ((I + n_cu / 2 + n_cu - 1) / n_cu) * n_cu - I;
    const int limit = (int)max((steps * a.p.n_kv + room - 1) / room, (int64_t)4);
    __syncthreads();
    // (pieces, slots, joins) of this thread's entries, then their places
    int cnt[3] = {0, 0, 0};
    for (int e = e0; e < e1; e++) {
        const int n = steps_of(e), parts = (n + limit - 1) / limit;
        cnt[0] += parts;
        cnt[1] += parts > 1 ? parts : 0;
        cnt[2] += parts > 1;
    }
    int at[3], tot[3];
#pragma unroll
    for (int c = 0; c < 3; c++) {
        const int x = vx_wave_scan(cnt[c]);
        if (lane == 63) s_sum[c][wave] = x;
        at[c] = x - cnt[c];
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < 3; c++) {
        tot[c] = 0;
#pragma unroll
        for (int w = 0; w < PLAN / 64; w++) {
            const int x = s_sum[c][w];
            at[c] += w < wave ? x : 0;
            tot[c] += x;
        }
    }
    // (token ranges that overlap, an error that vx_paged_seq has flagged, may
    // make more pieces than there is room for: then nothing runs)
    if ((int64_t)tot[0] * a.p.n_kv > max_pieces) e1 = e0, tot[0] = tot[2] = 0, *a.p.err_flag = 1;
    for (int e = e0; e < e1; e++) {
        const int n = steps_of(e), parts = (n + limit - 1) / limit;
        if (parts == 0) continue;
        const int len = n / parts, more = n - len * parts;   // the first `more` parts have one step more
        for (int h = 0; h < a.p.n_kv; h++) {
            const int slot = h * tot[1] + at[1];
            RowPiece *pc = a.pieces + h * tot[0] + at[0];
            for (int k = 0; k < parts; k++) {
                const int c0 = k * len + min(k, more);
                pc[k] = {b, h, r0, c0, c0 + len + (k < more), parts > 1 ? slot + k : -1, s};
            }
            if (parts > 1) {
                const RowJoin j = {b, h, r0, slot, parts};
                a.joins[h * tot[2] + at[2]] = j;
            }
        }
        at[0] += parts;
        at[1] += parts > 1 ? parts : 0;
        at[2] += parts > 1;
    }
    if (tid == 0) {
        a.plan->pieces = tot[0] * a.p.n_kv;
        a.plan->joins = tot[2] * a.p.n_kv;
    }
    if (tid < 8) a.plan->heads[tid] = 0;
}

// grid the most pieces there can be, block 256.
__global__ __launch_bounds__(256, 1) void paged_rows(Args a) {
    __shared__ __attribute__((aligned(16))) TileSmem sm;
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 5, n = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // The dispatcher deals workgroups round-robin over the 8 XCDs.  Each takes
    // the next piece of its own eighth of the list, so that the row tiles in
    // flight on an XCD are neighbours, whose keys its L2 then holds once; one
    // whose eighth is all taken helps another, beyond the pieces that the
    // other's CUs start with.  (The first workgroups of an XCD, as many as its
    // eighth has pieces, see that all of it is taken.  More would only help,
    // and only where pieces are left over: 208 more at the counters than the
    // 240 pieces of a call took it from 73 to 77 us.)
    const int pieces = a.plan->pieces, at_once = a.cus / 8;
    const int helper = (int)(blockIdx.x / 8) - pieces / 8 - ((int)(blockIdx.x & 7) < pieces % 8);
    if (helper >= 0 && (pieces / 8 < at_once || helper >= at_once)) return;
    if (wave == 0) {
        const int x = (blockIdx.x + lane) & 7, lo = x * (pieces / 8) + min(x, pieces % 8), n = pieces / 8 + (x < pieces % 8);
        int i = n;
        if (lane == 0) i = atomicAdd(&a.plan->heads[x], 1);
        uint32_t got = (uint32_t)__ballot(lane == 0 && i < n);
        if (!got) {   // lane k: the eighth k further on
            const int taken = __hip_atomic_load(&a.plan->heads[x], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            for (uint32_t left = (uint32_t)__ballot(taken >= at_once && taken < n) & 255; left && !got; left &= left - 1) {
                const int k = __builtin_ctz(left);
                if (lane == k) i = atomicAdd(&a.plan->heads[x], 1);
                got = (uint32_t)__ballot(lane == k && i < n);
            }
        }
        const int piece = __builtin_amdgcn_readlane(lo + i, __builtin_ctz(got | 1u << 31) & 7);
        if (lane == 0) {
            sm.piece = got ? piece : -1;
            sm.odd = 0;
        }
    }
    __syncthreads();
    const int piece = __builtin_amdgcn_readfirstlane(sm.piece);
    if (piece < 0) return;
    const RowPiece *pc = a.pieces + piece;
    const int b = __builtin_amdgcn_readfirstlane(pc->b), kvh = __builtin_amdgcn_readfirstlane(pc->kvh), r0 = __builtin_amdgcn_readfirstlane(pc->r0);
    const int c0 = __builtin_amdgcn_readfirstlane(pc->c0), c1 = __builtin_amdgcn_readfirstlane(pc->c1), slot = __builtin_amdgcn_readfirstlane(pc->slot);
    vx_pseq s;
    s.start = __builtin_amdgcn_readfirstlane(pc->s.start);
    s.T = __builtin_amdgcn_readfirstlane(pc->s.T);
    s.len = __builtin_amdgcn_readfirstlane(pc->s.len);
    s.row0 = s.len - s.T;
    const int R = s.T * a.qg;
    const int t0 = row_tok(a, r0), t1 = row_tok(a, min(r0 + TR - 1, R - 1));
    const vx_tiles tl = tiles_of(a, s, t0, t1);
    const int all = (tl.nt + 1) / 2, nt = min(c1, all) - c0;      // steps c0 .. c0 + nt - 1 of the list
    const bool parted = slot >= 0;
    const size_t slot0 = (size_t)max(slot, 0) * TR;
    // what the workgroup's rows see between them
    vx_sight any = vx_paged_sight(s, t0, a.window, a.n_sink);
    if (any.i < 0) any.lo = 0;
    const int i_first = any.i, lo_last = vx_paged_sight(s, t1, a.window, a.n_sink).lo;
    any.i = vx_paged_sight(s, t1, a.window, a.n_sink).i;

    const int wr0 = r0 + 32 * wave;                               // this wave's first row; rows past R repeat row R - 1
    const int qr = min(wr0 + n, R - 1), qt = row_tok(a, qr);
    const vx_sight v = vx_paged_sight(s, qt, a.window, a.n_sink);
    const uint16_t *qp = a.q + (size_t)(s.start + qt) * a.q_ts + (size_t)row_head(a, kvh, qr, qt) * a.q_hs + 8 * g;
    const int wi = vx_paged_sight(s, row_tok(a, min(wr0, R - 1)), a.window, a.n_sink).i;                // the least of its rows' own rows
    const int wl = vx_paged_sight(s, row_tok(a, min(wr0 + 31, R - 1)), a.window, a.n_sink).lo;          // the highest of their windows' edges

    // key block h of step c: its first key, or none (past the list)
    auto key_of = [&](int c, int h) -> int {
        const int i = 2 * c + h;
        return i < tl.nt ? tl.at(i) * TILE : -1;
    };
    // this wave's loads go to key block `wave / 2` of a step: 8 KiB of K (16
    // rows) and of V (128 dims)
    // (of K, row r's unit u goes to slot u ^ kswz(r); over j only two bits of
    // kswz change, so four offsets serve the eight loads, j KiB apart)
    uint32_t ko[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int r = (wave & 1) * 16 + 2 * (j & 1) + 8 * (j >> 1) + (lane >> 5);
        ko[j] = (uint32_t)((lane >> 5) * HDG * 2 + (((lane & 31) ^ kswz(r)) << 4)) + (wave & 1) * 8192;
    }
    const uint32_t vo = (uint32_t)((lane >> 2) * TILE * 2 + (((lane & 3) ^ ((lane >> 3) & 3)) << 4)) + (wave & 1) * 8192;
    const uint32_t k_lds = vx_lds_addr(sm.k[0]) + wave * 8192, v_lds = vx_lds_addr(sm.v[0]) + wave * 8192;
    // Element offsets in the pools of this wave's key blocks: lane i holds the
    // block of step base + i (past the list: its last block again), so a step
    // reads a lane and not the page table.
    int base = c0;
    uint32_t at_lo, at_hi;
    auto fill_at = [&]() {
        const int key = tl.at(min(2 * (base + lane) + (wave >> 1), tl.nt - 1)) * TILE, slot = vx_page_slot(a.p, key);
        const int page = vx_page_checked(a.p, vx_table_word(a.p.table + (size_t)b * a.p.max_pages + slot));
        const uint64_t at = (((uint64_t)page * a.p.n_kv + kvh) * a.p.page_size + (key - slot * a.p.page_size)) * HDG;
        at_lo = (uint32_t)at;
        at_hi = (uint32_t)(at >> 32);
    };
    // The blocks of the list that some row does not see all of come first
    // (sinks, and what the window's lower edge crosses: before block lo of
    // the list) and last (past a token's own row: from block hi on).
    auto low = [&](int row_lo) { return tl.st + max((row_lo + TILE - 1) / TILE - tl.fm, 0); };
    auto high = [&](int row_i) { return tl.st + (row_i + 1) / TILE - tl.fm; };
    const int e_lo = low(lo_last), e_hi = high(i_first), w_lo = low(wl), w_hi = high(wi);
    auto bare = [&](int c) { return 2 * c < e_lo || 2 * c + 1 >= e_hi; };    // some row of the workgroup
    auto cut = [&](int c) { return 2 * c < w_lo || 2 * c + 1 >= w_hi; };     // some row of the wave
    auto at_of = [&](int c) -> size_t {
        return (uint64_t)(uint32_t)__builtin_amdgcn_readlane(at_hi, c - base) << 32 | (uint32_t)__builtin_amdgcn_readlane(at_lo, c - base);
    };
    auto dma = [&](const char *p, uint32_t off, uint32_t lds, int j) {   // 1 KiB load j of 8
        switch (j & 3) {
            case 0: dma16<0>(p + (j & 4) * 1024, off, lds + (j & 4) * 1024); break;
            case 1: dma16<1024>(p + (j & 4) * 1024, off, lds + (j & 4) * 1024); break;
            case 2: dma16<2048>(p + (j & 4) * 1024, off, lds + (j & 4) * 1024); break;
            default: dma16<3 * 1024>(p + (j & 4) * 1024, off, lds + (j & 4) * 1024); break;
        }
    };
    auto dma_k = [&](size_t at, int buf, int j) { dma((const char *)(a.k_pages + at), ko[(j & 1) | ((j >> 2) << 1)], k_lds + buf * 2 * HALF, j); };
    auto dma_v = [&](size_t at, int buf, int j) { dma((const char *)(a.v_pages + at), vo, v_lds + buf * 2 * HALF, j); };

    floatx16_t O[8];
#pragma unroll
    for (int db = 0; db < 8; db++)
#pragma unroll
        for (int i = 0; i < 16; i++) O[db][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    auto pin_o = [&]() {
#pragma unroll
        for (int db = 0; db < 8; db++) __asm__ volatile("" : "+a"(O[db]));
    };

    if (nt > 0) {
        fill_at();
        size_t at_v = at_of(c0), at_k = at_of(c0 + 1);
#pragma unroll
        for (int j = 0; j < 8; j++) dma_k(at_v, 0, j);
#pragma unroll
        for (int j = 0; j < 8; j++) dma_k(at_k, 1, j);
#pragma unroll
        for (int j = 0; j < 8; j++) dma_v(at_v, 0, j);
        at_v = at_k;
        at_k = at_of(c0 + 2);
        bf16x8_t q[16];
#pragma unroll
        for (int k = 0; k < 16; k++) q[k] = load8(qp + 16 * k);
        auto pin_q = [&]() {
#pragma unroll
            for (int k = 0; k < 16; k++) __asm__ volatile("" : "+a"(q[k]));
        };
        floatx16_t S[2];           // [key block]
        __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
        pin_q();
        vx_lds_barrier();
        // Operand addresses in LDS, one for each of the swizzle's values; the
        // rest are offsets of the instructions.  (From an opaque copy of the
        // lane: formed before the queries are in their registers they would
        // be spilled.)
        int ln = lane;
        __asm__ volatile("" : "+v"(ln));
        const int g = ln >> 5, n = ln & 31;
        const int krow = 16 * (n >> 4) + 8 * ((n >> 2) & 1) + 4 * ((n >> 3) & 1) + (n & 3);
        const char *ka[8], *va[2];
#pragma unroll
        for (int k = 0; k < 8; k++) ka[k] = sm.k[0] + krow * (HDG * 2) + (((2 * k + g) ^ kswz(krow)) << 4);
#pragma unroll
        for (int k = 0; k < 2; k++) va[k] = sm.v[0] + n * (TILE * 2) + (((2 * k + g) ^ ((n >> 1) & 3)) << 4);
        auto kload = [&](int i) { return lds8(ka[(i >> 1) & 7] + (i & 1) * HALF + (i >> 4) * 256); };                 // k-step i / 2, key block i % 2
        auto vload = [&](int i) { return lds8(va[(i >> 3) & 1] + (i >> 4) * HALF + (i & 7) * 32 * TILE * 2); };     // 16 keys i / 8, dims 32 (i % 8)

        floatx16_t sc[2];          // this step's scores
        auto mask = [&](int c) {
#pragma unroll
            for (int kb = 0; kb < 2; kb++) {
                const int key0 = key_of(c, kb);
                const uint32_t bits = key0 < 0 ? 0u : v.block(key0) >> (8 * g);
#pragma unroll
                for (int i = 0; i < 16; i++)
                    if (!(bits & (1u << (16 * (i >> 3) + (i & 7))))) sc[kb][i] = -INFINITY;
            }
        };
        auto row_max = [&]() {
            float x = sc[0][0];
#pragma unroll
            for (int i = 0; i < 32; i += 2) __asm__("v_max3_f32 %0, %0, %1, %2" : "+v"(x) : "v"(sc[i >> 4][i & 15]), "v"(sc[i >> 4][(i & 15) + 1]));
            return x;
        };
        // In steps with a key that some row of the workgroup does not see: V of
        // keys that none sees becomes zero, so that what stale rows hold cannot
        // get in; and so do infinite and NaN values (0 times these would reach
        // the rows that do not see them), which the output adds for the rows
        // that do.  Thread tid has dim tid.
        auto clear_v = [&](int c, int buf) {
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if (2 * c + h >= e_lo && 2 * c + h < e_hi) continue;
                const int key0 = key_of(c, h);
                const uint32_t seen = key0 < 0 ? 0u : any.block(key0);
                uint4 *row = (uint4 *)(sm.v[buf] + h * HALF + tid * (TILE * 2));
                if (seen != 0xffffffffu) {
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const uint32_t byte = seen >> (8 * (u ^ ((tid >> 1) & 3)));
                        uint4 x = row[u];
                        uint32_t *w = (uint32_t *)&x;
#pragma unroll
                        for (int e = 0; e < 4; e++) w[e] &= ((byte >> (2 * e)) & 1 ? 0xffffu : 0u) | ((byte >> (2 * e)) & 2 ? 0xffff0000u : 0u);
                        row[u] = x;
                    }
                }
                uint32_t hot = 0;   // bits 15 and 31: an exponent of all ones carries into them
#pragma unroll
                for (int i = 0; i < 4; i++) {   // (from a unit of each lane's own: 8 lanes then read 8 distinct slots)
                    const uint4 x = row[(i + (tid >> 1)) & 3];
                    const uint32_t *w = (const uint32_t *)&x;
#pragma unroll
                    for (int e = 0; e < 4; e++) hot |= (w[e] & 0x7f807f80u) + 0x00800080u;
                }
                if (hot & 0x80008000u) {
                    uint32_t *w = (uint32_t *)row;
                    for (int e = 0; e < TILE / 2; e++)
                        w[e] &= ((w[e] & 0x7f80u) == 0x7f80u ? 0u : 0xffffu) | ((w[e] & 0x7f800000u) == 0x7f800000u ? 0u : 0xffff0000u);
                    sm.odd = 1;
                }
            }
            vx_lds_barrier();
        };
        // The row's reference from its maximum x over a lane's keys; O and l
        // follow when it moves (not before the first step, where they are 0).
        float ms;
        auto refer = [&](float x, bool some) {
            x = fmaxf(x, __uint_as_float(vx_xor32_u32(__float_as_uint(x)))) * SC2;
            const bool up = x > m;
            x += LAZY;
            if (some && __any(up)) {
                const float al = up ? __builtin_amdgcn_exp2f(m - x) : 1.0f;
                l *= al;
#pragma unroll
                for (int db = 0; db < 8; db++) O[db] *= al;
            }
            m = up ? x : m;
            ms = m == -INFINITY ? 0.0f : m;
        };

#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int i = 0; i < 16; i++) S[kb][i] = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; i++) S[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kload(i), q[i >> 1], S[i & 1], 0, 0, 0);
#pragma unroll
        for (int k = 0; k < 8; k++) ka[k] += 2 * HALF;   // (the next step's)
        sc[0] = S[0];
        sc[1] = S[1];
        if (cut(c0)) mask(c0);
        refer(row_max(), false);

        // A step: S of the next step on the MFMAs with this step's softmax and
        // the loads of K(c+2) and V(c+1) beside it, then P V with the next
        // step's maxima beside it.  One MFMA at a time with its share of the
        // VALU's and the loads' work behind it, in this order: what stands
        // behind an MFMA that waits for the pipe waits too.
        constexpr int AHEAD = 6;   // operands read ahead of their MFMA
        bool edge = bare(c0), cutn = nt > 1 && cut(c0 + 1);
        for (int c = 0; c < nt; c++) {
            const int bk = c & 1;
            // K(c+1) and V(c) have landed; every wave is done with step c-1
            __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
            vx_lds_barrier();
            if (edge) clear_v(c0 + c, bk);
            bf16x8_t f[8];
#pragma unroll
            for (int i = 0; i < AHEAD; i++) f[i] = kload(i);
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int i = 0; i < 16; i++) S[kb][i] = 0.0f;
            pin_q();
            __builtin_amdgcn_sched_barrier(0);
            // Element t of the row goes through the softmax in three shares
            // (argument, exp2, sum and rounding), so that none waits for its
            // own result.
            bf16x8_t p[4];
            float e[32];
            auto weigh = [&](int t) {
                if (t >= 2 && t < 34) {
                    l += e[t - 2];
                    __asm__ volatile("" : "+v"(l));
                    p[(t - 2) >> 3][(t - 2) & 7] = (__bf16)e[t - 2];
                }
                if (t >= 1 && t < 33) e[t - 1] = __builtin_amdgcn_exp2f(e[t - 1]);
                if (t < 32) e[t] = __builtin_fmaf(sc[t >> 4][t & 15], SC2, -ms);
            };
#pragma unroll
            for (int i = 0; i < 32; i++) {
                if (i + AHEAD < 32) f[(i + AHEAD) & 7] = kload(i + AHEAD);
                else f[(i + AHEAD) & 7] = vload(i + AHEAD - 32);
                if (i < 16) {
                    if (i & 1) dma_v(at_v, bk ^ 1, i >> 1);
                    else dma_k(at_k, bk, i >> 1);
                }
                S[i & 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[i & 7], q[i >> 1], S[i & 1], 0, 0, 0);
                weigh(i);
                __builtin_amdgcn_sched_barrier(0);
            }
            weigh(32);
            weigh(33);
            pin_o();
            float x;
            bool edge2 = false, cut2 = false;
#pragma unroll
            for (int i = 0; i < 32; i++) {
                if (i + AHEAD < 32) f[(i + AHEAD) & 7] = vload(i + AHEAD);
                O[i & 7] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f[i & 7], p[i >> 3], O[i & 7], 0, 0, 0);
                sc[i >> 4][i & 15] = S[i >> 4][i & 15];
                // (in asm: here, not in a row behind the MFMAs, and without
                // the quieting of NaN that fmaxf puts before each)
                if (i == 0) x = sc[0][0];
                else if (i & 1) __asm__ volatile("v_max3_f32 %0, %0, %1, %2" : "+v"(x) : "v"(sc[i >> 4][(i & 15) - 1]), "v"(sc[i >> 4][i & 15]));
                // the next step's addresses, edges and buffers
                if (i == 1) at_v = at_k, at_k = at_of(c0 + c + 3);
                if (i == 3) edge2 = bare(c0 + c + 1);
                if (i == 5) cut2 = c + 2 < nt && cut(c0 + c + 2);
                if (i >= 8 && i < 16) ka[i - 8] += bk ? 2 * HALF : -2 * HALF;
                if (i >= 30) va[i - 30] += bk ? -2 * HALF : 2 * HALF;
                __builtin_amdgcn_sched_barrier(0);
            }
            pin_o();
            if (cutn) {
                mask(c0 + c + 1);
                x = row_max();
            }
            if (c + 1 < nt) refer(x, true);
            pin_o();
            edge = edge2;
            cutn = cut2;
            if (c0 + c + 5 > base + 63) {   // (one step in 60)
                base = c0 + c + 4;
                fill_at();
            }
        }
        __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the last (unused) loads
    }
    // Output rows of this wave: pairs (8 k + 2 wave, + 1), half a wave each,
    // lane L dims 8 (L % 32) .. +7.  Their bf16 gates are all loaded before the
    // first is used: a load behind the rows' stores would wait for them.
    constexpr int WR = TR / 8;
    uint4 gt[WR];
    const bool gated = a.gate && !parted;
    auto out_row = [&](int k) { return r0 + 8 * k + 2 * wave + (lane >> 5); };
    if (gated && a.gate_bf16) {
#pragma unroll
        for (int k = 0; k < WR; k++) {
            const int r = min(out_row(k), R - 1), t = row_tok(a, r);
            gt[k] = *(const uint4 *)((const uint16_t *)a.gate + (size_t)(s.start + t) * a.g_ts + (size_t)row_head(a, kvh, r, t) * a.g_hs + 8 * (lane & 31));
        }
    }
    l += __uint_as_float(vx_xor32_u32(__float_as_uint(l)));
    vx_lds_barrier();   // every wave is done with the tiles
    // O through LDS (16-byte units swizzled by the row)
    float *so = (float *)sm.k[0];
    {
        const int r = 32 * wave + n;
        const float il = parted ? 1.0f : (l > 0.0f || l != l ? 1.0f / l : 0.0f);
#pragma unroll
        for (int db = 0; db < 8; db++)
#pragma unroll
            for (int q4 = 0; q4 < 4; q4++) {
                const int u = (32 * db + 8 * q4 + 4 * g) >> 2;
                *(float4 *)(so + r * HDG + ((u ^ (r & 15)) << 2)) =
                    make_float4(O[db][4 * q4] * il, O[db][4 * q4 + 1] * il, O[db][4 * q4 + 2] * il, O[db][4 * q4 + 3] * il);
            }
        if (g == 0 && r0 + r < R) {
            if (parted) {
                a.part_ml[slot0 + r] = make_float2(m, l);
            } else {
                const int t = row_tok(a, r0 + r);
                stat_store<LAZY>(a, s.start + t, row_head(a, kvh, r0 + r, t), m, l);
            }
        }
    }
    vx_lds_barrier();
    if (sm.odd) {   // (the same for every thread)
        for (int c = c0; c < c0 + nt; c++) {
            if (!bare(c)) continue;
            for (int h = 0; h < 2; h++) {
                const int key0 = key_of(c, h);
                if (key0 < 0) continue;
                const int page = vx_paged_page(a.p, b, key0), at = key0 - vx_page_slot(a.p, key0) * a.p.page_size;
                const uint16_t *vp = a.v_pages + vx_v_index(a.p.n_kv, a.p.page_size, page, kvh, at, tid);
                for (int j = 0; j < TILE; j++) {
                    const float x = vx_bf16_to_f32(vp[j]);
                    if (is_finite(x)) continue;
                    for (int r = 0; r < TR && r0 + r < R; r++)
                        if (sight_of(a, s, r0 + r).sees(key0 + j)) so[r * HDG + ((((tid >> 2) ^ (r & 15)) << 2) | (tid & 3))] += x;
                }
            }
        }
        vx_lds_barrier();
    }
    auto orow = [&](int k, float4 &x, float4 &y) {
        const int r = out_row(k) - r0, u = 2 * (lane & 31);
        x = *(const float4 *)(so + r * HDG + ((u ^ (r & 15)) << 2));
        y = *(const float4 *)(so + r * HDG + (((u + 1) ^ (r & 15)) << 2));
    };
    if (parted) {
#pragma unroll 4
        for (int k = 0; k < WR; k++) {
            float4 x, y;
            orow(k, x, y);
            float4 *dst = (float4 *)(a.part_o + (slot0 + out_row(k) - r0) * HDG + 8 * (lane & 31));
            if (out_row(k) < R) {
                dst[0] = x;
                dst[1] = y;
            }
        }
        return;
    }
    float4 nx, ny;
    orow(0, nx, ny);
#pragma unroll
    for (int k = 0; k < WR; k++) {
        float x[8] = {nx.x, nx.y, nx.z, nx.w, ny.x, ny.y, ny.z, ny.w};
        if (k + 1 < WR) orow(k + 1, nx, ny);
        if (r0 + 8 * k + 2 * wave >= R) break;
        const int r = out_row(k), t = row_tok(a, r), tok = s.start + t, h = row_head(a, kvh, r, t);
        if (gated) {
            float z[8];
            if (a.gate_bf16) {
                const uint32_t u[4] = {gt[k].x, gt[k].y, gt[k].z, gt[k].w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    z[2 * e] = __uint_as_float(u[e] << 16);
                    z[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
                }
            } else {
                const float4 *gp = (const float4 *)((const float *)a.gate + (size_t)min(tok, a.p.n_tok - 1) * a.g_ts + (size_t)min(h, a.n_q - 1) * a.g_hs + 8 * (lane & 31));
                const float4 u = gp[0], w = gp[1];
                z[0] = u.x; z[1] = u.y; z[2] = u.z; z[3] = u.w; z[4] = w.x; z[5] = w.y; z[6] = w.z; z[7] = w.w;
            }
#pragma unroll
            for (int e = 0; e < 8; e++) x[e] *= fast_sigmoid(z[e]);
        }
        if (r < R) {
            const size_t at = ((size_t)tok * a.n_q + h) * HDG + 8 * (lane & 31);
            if (a.out_bf16) {
                *(uint4 *)((uint16_t *)a.out + at) = make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
            } else {
                float4 *dst = (float4 *)((float *)a.out + at);
                dst[0] = make_float4(x[0], x[1], x[2], x[3]);
                dst[1] = make_float4(x[4], x[5], x[6], x[7]);
            }
        }
    }
}

// grid any, block 256: adds up the parts of the cut items, in order, four
// rows a wave, their loads in flight together.  (Seven chunks of 701 tokens:
// 116 us the call with two workgroups a CU, 113 with four, 111 with eight.)
__global__ __launch_bounds__(256) void paged_rows_join(Args a) {
    constexpr int NR = 4, PER = TR / (4 * NR);
    const int lane = threadIdx.x & 63, todo = a.plan->joins * PER;
    for (int it = blockIdx.x; it < todo; it += gridDim.x) {
    const RowJoin jn = a.joins[it / PER];
    const vx_pseq s = vx_paged_seq(a.p, jn.b);
    const int q0 = it % PER * 16 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * NR, R = s.T * a.qg;
    if (jn.r0 + q0 >= R) continue;
    float M[NR], L[NR];
    float4 O[NR], gt[NR];
    int tok[NR], h[NR];
#pragma unroll
    for (int q = 0; q < NR; q++) {
        const int r = min(jn.r0 + q0 + q, R - 1), t = row_tok(a, r);
        tok[q] = s.start + t;
        h[q] = row_head(a, jn.kvh, r, t);
        gt[q] = a.gate ? gate_row(a, tok[q], h[q]) : make_float4(0.f, 0.f, 0.f, 0.f);
        M[q] = -INFINITY;
        L[q] = 0.0f;
        O[q] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int k = 0; k < jn.parts; k++) {
        const size_t at = (size_t)(jn.slot + k) * TR + q0;
        float2 ml[NR];
        float4 o[NR];
#pragma unroll
        for (int q = 0; q < NR; q++) {   // (rows past the last: slots that nobody wrote, unused)
            ml[q] = a.part_ml[at + q];
            o[q] = *(const float4 *)(a.part_o + (at + q) * HDG + 4 * lane);
        }
#pragma unroll
        for (int q = 0; q < NR; q++) {
            const float mn = fmaxf(M[q], ml[q].x), ref = mn == -INFINITY ? 0.0f : mn;
            const float w = __builtin_amdgcn_exp2f(M[q] - ref);
            L[q] *= w;
            O[q].x *= w; O[q].y *= w; O[q].z *= w; O[q].w *= w;
            add_part(O[q], L[q], o[q], ml[q].y, __builtin_amdgcn_exp2f(ml[q].x - ref));
            M[q] = mn;
        }
    }
#pragma unroll
    for (int q = 0; q < NR; q++) {
        if (jn.r0 + q0 + q >= R) break;
        const float il = L[q] > 0.0f || L[q] != L[q] ? 1.0f / L[q] : 0.0f;
        row_store(a, tok[q], h[q], make_float4(O[q].x * il, O[q].y * il, O[q].z * il, O[q].w * il), gt[q]);
        if (lane == 0) stat_store<LAZY>(a, tok[q], h[q], M[q], L[q]);
    }
    }
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
    if (vx_paged_fill(who, a.p, d->B, d->n_kv, d->hd, d->page_size, d->n_pages, d->max_pages, d->table, d->len)) return -1;
    if (vx_paged_tokens(who, a.p, d->q_start, d->n_tok, d->max_T)) return -1;
    VX_REQUIRE(d->n_q >= d->n_kv && d->n_q % d->n_kv == 0 && d->n_q / d->n_kv <= 16,
               "%s: need n_q = k*n_kv with k <= 16 (n_q=%d n_kv=%d)", who, d->n_q, d->n_kv);
    VX_REQUIRE(d->window >= 0 && d->n_sink >= 0, "%s: window and n_sink must not be negative (got %d, %d)", who, d->window, d->n_sink);
    VX_REQUIRE(d->q && d->k_pages && d->v_pages && d->out, "%s: null pointer in descriptor", who);
    VX_REQUIRE((d->out_dtype == VX27_F32 || d->out_dtype == VX27_BF16) && (!d->gate || d->gate_dtype == VX27_F32 || d->gate_dtype == VX27_BF16),
               "%s: out_dtype and gate_dtype must be VX27_F32 or VX27_BF16 (got %d, %d)", who, d->out_dtype, d->gate_dtype);
    a.q_hs = d->q_head_stride ? d->q_head_stride : HDG;
    a.q_ts = d->q_tok_stride ? d->q_tok_stride : (size_t)d->n_q * HDG;
    a.g_hs = d->gate_head_stride ? d->gate_head_stride : HDG;
    a.g_ts = d->gate_tok_stride ? d->gate_tok_stride : (size_t)d->n_q * HDG;
    VX_REQUIRE((((uintptr_t)d->q | (uintptr_t)d->k_pages | (uintptr_t)d->v_pages | (uintptr_t)d->out | (uintptr_t)d->gate) & 15) == 0 &&
                   ((a.q_hs | a.q_ts | a.g_hs | a.g_ts) & 7) == 0,
               "%s: q, gate, out and the pages must be 16-byte aligned, q and gate strides multiples of 8 elements", who);
    const int64_t cap = (int64_t)d->max_pages * d->page_size;
    VX_REQUIRE(!d->acc || (int64_t)d->acc_stride >= cap, "%s: acc_stride must be at least max_pages * page_size (got %zu, %lld)", who,
               d->acc_stride, (long long)cap);
    a.n_q = d->n_q; a.qg = d->n_q / d->n_kv; a.qg_magic = a.qg == 1 ? 0 : (uint32_t)((1ull << 32) / a.qg + 1); a.window = d->window; a.n_sink = d->n_sink;
    VX_REQUIRE((int64_t)d->max_T * a.qg < (1 << 28), "%s: max_T * n_q/n_kv is past 2^28 (max_T=%d)", who, d->max_T);
    if (vx_ctx_enter(ctx)) return -1;
    if (d->n_tok == 0) return 0;
    a.p.err_flag = ctx->err_flag;
    a.q = d->q; a.k_pages = d->k_pages; a.v_pages = d->v_pages;
    a.gate = d->gate; a.gate_bf16 = d->gate_dtype == VX27_BF16;
    a.out = d->out; a.out_bf16 = d->out_dtype == VX27_BF16;
    a.lse = d->lse; a.acc = d->acc; a.acc_stride = d->acc_stride;

    // most tiles a sequence can have: its capacity, or sinks, window and new tokens (each range may touch one tile more)
    int64_t tile_cap = cap / TILE;
    if (d->window) tile_cap = std::min<int64_t>(tile_cap, ((int64_t)d->window + d->max_T) / TILE + 2 + (d->n_sink + (int64_t)TILE - 1) / TILE);
    a.tile_cap = (int)tile_cap;
    const int rows = d->max_T * a.qg;
    const size_t stat_bytes = d->acc ? ((size_t)d->n_tok * d->n_q * sizeof(float2) + 255) / 256 * 256 : 0;
    if (rows <= 16) {
        VX_REQUIRE((int64_t)d->B * d->n_kv * tile_cap < (1ll << 31) - 65536, "%s: more than 2^31 key tiles (B=%d n_kv=%d, %lld tiles each)", who,
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
        if (a.before) VX_LAUNCH(ctx, paged_units, dim3(1), dim3(1024), a);
        VX_LAUNCH(ctx, paged_split, dim3(grid), dim3(256), a);
        VX_LAUNCH(ctx, paged_join, dim3(rows, d->n_kv, d->B), dim3(256), a, grid);
        if (d->acc) VX_LAUNCH(ctx, paged_weigh, dim3((a.tile_cap + 7) / 8, d->n_kv, d->B), dim3(256), a);
        return 0;
    }
    // (a 32-row tile's queries are addressed by 32-bit offsets from its first)
    VX_REQUIRE(!d->acc || (a.q_ts < (1u << 26) && a.q_hs < (1u << 26)), "%s: q strides past 2^26 elements with acc (got %zu, %zu)", who, a.q_ts, a.q_hs);
    const int n_rt = (rows + TR - 1) / TR, n_cu = a.cus = ctx->n_cu;
    VX_REQUIRE((int64_t)d->B * n_rt < (1ll << 31) - PLAN, "%s: more than 2^31 row tiles (B=%d max_T=%d)", who, d->B, d->max_T);
    // every token range ends in one tile that it need not fill; paged_plan makes at most 3/2 n_cu cuts, so twice
    // as many parts at most
    const int64_t cuts = (int64_t)n_cu * 3 / 2, items = ((int64_t)d->n_tok * a.qg / TR + d->B) * d->n_kv;
    VX_REQUIRE(items + cuts < (1 << 24), "%s: more than 2^24 row tiles (B=%d n_kv=%d n_tok=%d)", who, d->B, d->n_kv, d->n_tok);
    const size_t ml_bytes = (size_t)2 * cuts * TR * sizeof(float2), plan_bytes = 256, piece_bytes = (size_t)(items + cuts) * sizeof(RowPiece);
    const size_t join_bytes = ((size_t)cuts * sizeof(RowJoin) + 255) / 256 * 256;
    void *scr;
    if (vx_ctx_scratch(ctx, stat_bytes + ml_bytes + plan_bytes + join_bytes + (size_t)2 * cuts * TR * HDG * 4 + piece_bytes, &scr)) return -1;
    char *at = (char *)scr;
    a.stat = d->acc ? (float2 *)at : nullptr;
    a.part_ml = (float2 *)(at += stat_bytes);
    a.plan = (RowPlan *)(at += ml_bytes);
    a.joins = (RowJoin *)(at += plan_bytes);
    a.part_o = (float *)(at += join_bytes);
    a.pieces = (RowPiece *)(at += (size_t)2 * cuts * TR * HDG * 4);
    VX_LAUNCH(ctx, paged_plan, dim3(1), dim3(PLAN), a, n_rt, n_cu, (int)(items + cuts));
    VX_LAUNCH(ctx, paged_rows, dim3((unsigned)(items + cuts)), dim3(256), a);
    VX_LAUNCH(ctx, paged_rows_join, dim3(8 * n_cu), dim3(256), a);
    if (d->acc) VX_LAUNCH(ctx, paged_rows_weigh, dim3((a.tile_cap + 7) / 8, d->n_kv, d->B), dim3(256), a);
    return 0;
}
