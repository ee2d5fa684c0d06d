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

#include "vx_paged.h"

namespace {

constexpr int HDG = VX_GQA_HD, TILE = VX_PG_TILE;
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float floatx4_t __attribute__((ext_vector_type(4)));
constexpr float SC2 = 0.0625f * 1.4426950408889634f;   // 1/sqrt(256) * log2(e): scores in the exp2 domain

struct Args {
    vx_paged p;
    int n_q, qg, window, n_sink;
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
    float *stash;                // with acc: raw scores [B][n_kv][max rows][tile_cap * 32]
};

__device__ __forceinline__ vx_tiles tiles_of(const Args &a, const vx_pseq &s, int t0, int t1) {
    return vx_paged_tiles(s, t0, t1, a.window, a.n_sink);
}
// What query row r of a sequence sees (rows past the last see nothing).
__device__ __forceinline__ vx_sight sight_of(const Args &a, const vx_pseq &s, int r) {
    return vx_paged_sight(s, r / a.qg, a.window, a.n_sink);
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
    const int lane = threadIdx.x & 63, g = lane >> 4, n = lane & 15, r = r0 + n, t = r / a.qg;
    const bool live = t < s.T;
    const uint16_t *qp = a.q + (size_t)(s.start + (live ? t : 0)) * a.q_ts + (size_t)(kvh * a.qg + (live ? r % a.qg : 0)) * a.q_hs + 8 * g;
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

// Online softmax and P V of one tile.  NP bf16 parts of each weight: three
// hold all 24 bits of it.  V of keys no row of the wave sees is zeroed, so
// that what stale rows hold cannot get in.
template <int NP>
__device__ __forceinline__ void attend_tile(Rows &w, const float (&s)[8], const vx_sight &v, int key0, bf16x8_t (&va)[16]) {
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
    const float m_new = fmaxf(w.m, mt * SC2);
    const bool none = m_new == -INFINITY;
    const float alpha = none ? 1.0f : __builtin_amdgcn_exp2f(w.m - m_new);
    bf16x8_t p[NP];
    float ls = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        float pe = none ? 0.0f : __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], SC2, -m_new));
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
#pragma unroll
        for (int e = 0; e < 8; e++) {
            // any of the 16 rows of this lane group sees key 8g + e
            const uint64_t seen = __ballot(v.sees(key0 + 8 * g + e));
            if (((seen >> (16 * g)) & 0xffff) == 0) {
#pragma unroll
                for (int d = 0; d < 16; d++) va[d][e] = (__bf16)0.0f;
            }
        }
    }
#pragma unroll
    for (int k = 0; k < NP; k++)
#pragma unroll
        for (int d = 0; d < 16; d++) w.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(va[d], p[k], w.o[d], 0, 0, 0);
}

__device__ __forceinline__ float gate_of(const Args &a, int tok, int h, int d) {
    const size_t at = (size_t)tok * a.g_ts + (size_t)h * a.g_hs + d;
    return a.gate_bf16 ? vx_bf16_to_f32(((const uint16_t *)a.gate)[at]) : ((const float *)a.gate)[at];
}
// One finished value: O / l (0 where nothing was seen), gated.
__device__ __forceinline__ void out_store(const Args &a, int tok, int h, int d, float O, float L) {
    float r = L > 0.0f || L != L ? O / L : 0.0f;
    if (a.gate) r = r * (1.0f / (1.0f + expf(-gate_of(a, tok, h, d))));
    const size_t at = ((size_t)tok * a.n_q + h) * HDG + d;
    if (a.out_bf16) ((uint16_t *)a.out)[at] = vx_f32_to_bf16(r);
    else ((float *)a.out)[at] = r;
}
__device__ __forceinline__ void stat_store(const Args &a, int tok, int h, float m, float L) {
    const size_t at = (size_t)tok * a.n_q + h;
    if (a.lse) a.lse[at] = L > 0.0f || L != L ? (m + log2f(L)) * 0.6931471805599453f : -INFINITY;
    if (a.stat) a.stat[at] = make_float2(m, L > 0.0f || L != L ? 1.0f / L : 0.0f);
}

// ---------------------------------------------------------------- decode
// At most 16 query rows a KV head.  The tiles of every (sequence, KV head)
// pair form one list; workgroup w of G takes tiles [w c, (w+1) c) of it, so
// a ragged batch is as even as an equal one.  A pair wholly inside one
// workgroup is finished there; the first and the last piece of a
// workgroup's range may be parts of a pair and go to its two partial slots,
// which paged_join merges in order.
struct Plan {
    int total, chunk;
};
__device__ __forceinline__ int seq_units(const Args &a, int b, int &nt) {
    const vx_pseq s = vx_paged_seq(a.p, b);
    nt = tiles_of(a, s, 0, s.T - 1).nt;
    return nt * a.p.n_kv;
}
__device__ __forceinline__ int wave_sum_i(int v) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}
__device__ __forceinline__ Plan plan_of(const Args &a, int grid) {
    const int lane = threadIdx.x & 63;
    int sum = 0, nt;
    for (int b = lane; b < a.p.B; b += 64) sum += seq_units(a, b, nt);
    Plan p;
    p.total = __builtin_amdgcn_readfirstlane(wave_sum_i(sum));
    p.chunk = max((p.total + grid - 1) / grid, a.min_tiles);
    return p;
}

__global__ __launch_bounds__(256, 2) void paged_split(Args a) {
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, n = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    __shared__ __attribute__((aligned(16))) float s_o[4][16 * HDG];
    __shared__ float s_m[4][16], s_l[4][16];
    const Plan pl = plan_of(a, gridDim.x);
    const int u0 = blockIdx.x * pl.chunk, u1 = min(u0 + pl.chunk, pl.total);
    if (u0 >= u1) return;
    // the sequence of unit u0, and the units before it
    int b = 0, before = 0;
    {
        int done = 0;
        for (int b0 = 0; b0 < a.p.B; b0 += 64) {
            int nt, x = b0 + lane < a.p.B ? seq_units(a, b0 + lane, nt) : 0;
            const int own_x = x;
            for (int off = 1; off < 64; off <<= 1) {
                const int y = __shfl_up(x, off, 64);
                if (lane >= off) x += y;
            }
            const uint64_t past = __ballot(done + x > u0);
            if (past) {
                const int f = __builtin_ctzll(past);
                b = b0 + f;
                before = done + __shfl(x - own_x, f, 64);
                break;
            }
            done += __shfl(x, 63, 64);
        }
        b = __builtin_amdgcn_readfirstlane(b);
        before = __builtin_amdgcn_readfirstlane(before);
    }
    const int krow0 = 8 * (n >> 2) + (n & 3);
    for (int u = u0; u < u1;) {
        const vx_pseq s = vx_paged_seq(a.p, b);
        const vx_tiles tl = tiles_of(a, s, 0, s.T - 1);
        if (u >= before + tl.nt * a.p.n_kv) {
            before += tl.nt * a.p.n_kv;
            b++;
            continue;
        }
        const int kvh = (u - before) / tl.nt, i0 = (u - before) % tl.nt;
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
            attend_tile<3>(w, sc, v, key0, va);
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
        const bool whole = cnt == tl.nt;
        const int slot = 2 * blockIdx.x + (u == u0 ? 0 : 1);
        for (int r = 0; r < R; r++) {
            float M = -INFINITY;
#pragma unroll
            for (int k = 0; k < 4; k++) M = fmaxf(M, s_m[k][r]);
            float L = 0.0f, O = 0.0f;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float sc = s_m[k][r] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_m[k][r] - M);
                L += s_l[k][r] * sc;
                O += s_o[k][r * HDG + ((((tid >> 2) ^ r) << 2) | (tid & 3))] * sc;
            }
            if (whole) {
                const int tok = s.start + r / a.qg, h = kvh * a.qg + r % a.qg;
                out_store(a, tok, h, tid, O, L);
                if (tid == 0) stat_store(a, tok, h, M, L);
            } else {
                a.part_o[((size_t)slot * a.part_rows + r) * HDG + tid] = O;
                if (tid == 0) a.part_ml[(size_t)slot * a.part_rows + r] = make_float2(M, L);
            }
        }
        __syncthreads();
        u += cnt;
    }
}

// grid (max rows, n_kv, B), block 256: merges the parts of one query row, in
// their order: wave w takes parts w, w + 4, ...; a row of a sequence without
// rows gets 0.
__global__ __launch_bounds__(256) void paged_join(Args a, int grid) {
    const int r = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const vx_pseq s = vx_paged_seq(a.p, b);
    if (r >= s.T * a.qg) return;
    const int tok = s.start + r / a.qg, h = kvh * a.qg + r % a.qg;
    const int nt = tiles_of(a, s, 0, s.T - 1).nt;
    if (nt == 0) {
        out_store(a, tok, h, tid, 0.0f, 0.0f);
        if (tid == 0) stat_store(a, tok, h, -INFINITY, 0.0f);
        return;
    }
    const Plan pl = plan_of(a, grid);
    int sum = 0, x;
    for (int c = lane; c < b; c += 64) sum += seq_units(a, c, x);
    const int p0 = __builtin_amdgcn_readfirstlane(wave_sum_i(sum)) + kvh * nt, p1 = p0 + nt;
    const int g0 = p0 / pl.chunk, g1 = (p1 - 1) / pl.chunk;
    if (g0 == g1) return;
    __shared__ float4 s_o[4][64];
    __shared__ float s_m[4], s_l[4];
    float M = -INFINITY, L = 0.0f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int w = g0 + wave; w <= g1; w += 4) {
        const size_t pi = (size_t)(2 * w + (w == g0 && p0 != w * pl.chunk ? 1 : 0)) * a.part_rows + r;
        const float2 ml = a.part_ml[pi];
        const float4 o = ((const float4 *)(a.part_o + pi * HDG))[lane];
        const float mn = fmaxf(M, ml.x);
        if (mn == -INFINITY) continue;
        const float sa = __builtin_amdgcn_exp2f(M - mn), sb = __builtin_amdgcn_exp2f(ml.x - mn);
        L = L * sa + ml.y * sb;
        O.x = O.x * sa + o.x * sb; O.y = O.y * sa + o.y * sb;
        O.z = O.z * sa + o.z * sb; O.w = O.w * sa + o.w * sb;
        M = mn;
    }
    s_o[wave][lane] = O;
    if (lane == 0) {
        s_m[wave] = M;
        s_l[wave] = L;
    }
    __syncthreads();
    float Mt = -INFINITY;
#pragma unroll
    for (int k = 0; k < 4; k++) Mt = fmaxf(Mt, s_m[k]);
    float Lt = 0.0f, Ot = 0.0f;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float sc = s_m[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(s_m[k] - Mt);
        Lt += s_l[k] * sc;
        Ot += ((const float *)s_o[k])[tid] * sc;
    }
    out_store(a, tok, h, tid, Ot, Lt);
    if (tid == 0) stat_store(a, tok, h, Mt, Lt);
}

// grid (tile_cap / 8, n_kv, B), block 256: one thread per key; the stashed
// scores become weights, summed over the rows that see the key.
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
        const float2 ml = a.stat[(size_t)(s.start + r / a.qg) * a.n_q + kvh * a.qg + r % a.qg];
        sum += __builtin_amdgcn_exp2f(__builtin_fmaf(st[r * stride], SC2, -ml.x)) * ml.y;
        any = true;
    }
    if (any) a.acc[((size_t)b * a.p.n_kv + kvh) * a.acc_stride + j] += sum;
}

// ------------------------------------------------------------------ tiles
// More than 16 query rows a KV head.  grid (64-row blocks, n_kv, B), block
// 256: wave w takes 16 rows.
__global__ __launch_bounds__(256) void paged_tile(Args a) {
    const int kvh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63, g = lane >> 4, n = lane & 15;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const vx_pseq s = vx_paged_seq(a.p, b);
    const int R = s.T * a.qg, r0 = blockIdx.x * 64 + wave * 16;
    if (r0 >= R) return;
    const vx_tiles tl = tiles_of(a, s, r0 / a.qg, min(r0 + 15, R - 1) / a.qg);
    Rows w;
    rows_begin(a, s, kvh, r0, w);
    const vx_sight v = sight_of(a, s, r0 + n);
    const int krow0 = 8 * (n >> 2) + (n & 3);
    for (int i = 0; i < tl.nt; i++) {
        const int key0 = tl.at(i) * TILE;
        const int page = vx_paged_page(a.p, b, key0), at = key0 - vx_page_slot(a.p, key0) * a.p.page_size;
        const uint16_t *kr0 = a.k_pages + vx_k_index(a.p.n_kv, a.p.page_size, page, kvh, at + krow0, 8 * g);
        const uint16_t *vt = a.v_pages + vx_v_index(a.p.n_kv, a.p.page_size, page, kvh, at, n) + 8 * g;
        bf16x8_t ka[8], kb[8], va[16];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            ka[k] = load8(kr0 + 32 * k);
            kb[k] = load8(kr0 + 4 * HDG + 32 * k);
        }
#pragma unroll
        for (int d = 0; d < 16; d++) va[d] = load8(vt + (size_t)d * 16 * TILE);
        float sc[8];
        score_tile(ka, kb, w.q, sc);
        attend_tile<1>(w, sc, v, key0, va);
    }
    w.l += __shfl_xor(w.l, 16, 64);
    w.l += __shfl_xor(w.l, 32, 64);
    const int r = r0 + n;
    if (r >= R) return;
    const int tok = s.start + r / a.qg, h = kvh * a.qg + r % a.qg;
#pragma unroll
    for (int d = 0; d < 16; d++)
#pragma unroll
        for (int e = 0; e < 4; e++) out_store(a, tok, h, 16 * d + 4 * g + e, w.o[d][e], w.l);
    if (g == 0) stat_store(a, tok, h, w.m, w.l);
}

// grid (tile_cap / 4, n_kv, B), block 256: one wave per key tile adds the
// weights of every query row to it, the scores formed again.
__global__ __launch_bounds__(256) void paged_tile_weigh(Args a) {
    const int kvh = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63, g = lane >> 4, n = lane & 15;
    const int i = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(tid >> 6);
    const vx_pseq s = vx_paged_seq(a.p, b);
    const vx_tiles tl = tiles_of(a, s, 0, s.T - 1);
    if (i >= tl.nt) return;
    const int key0 = tl.at(i) * TILE;
    const int page = vx_paged_page(a.p, b, key0), at = key0 - vx_page_slot(a.p, key0) * a.p.page_size;
    const uint16_t *kr0 = a.k_pages + vx_k_index(a.p.n_kv, a.p.page_size, page, kvh, at + 8 * (n >> 2) + (n & 3), 8 * g);
    bf16x8_t ka[8], kb[8];
#pragma unroll
    for (int k = 0; k < 8; k++) {
        ka[k] = load8(kr0 + 32 * k);
        kb[k] = load8(kr0 + 4 * HDG + 32 * k);
    }
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    int any = 0;
    for (int r0 = 0; r0 < s.T * a.qg; r0 += 16) {
        Rows w;
        rows_begin(a, s, kvh, r0, w);
        const vx_sight v = sight_of(a, s, r0 + n);
        const int r = min(r0 + n, s.T * a.qg - 1);
        const float2 ml = a.stat[(size_t)(s.start + r / a.qg) * a.n_q + kvh * a.qg + r % a.qg];
        float sc[8];
        score_tile(ka, kb, w.q, sc);
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (v.sees(key0 + 8 * g + e)) {
                sum[e] += __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], SC2, -ml.x)) * ml.y;
                any |= 1 << e;
            }
    }
#pragma unroll
    for (int off = 1; off < 16; off <<= 1) {
#pragma unroll
        for (int e = 0; e < 8; e++) sum[e] += __shfl_xor(sum[e], off, 64);
        any |= __shfl_xor(any, off, 64);
    }
    float *dst = a.acc + ((size_t)b * a.p.n_kv + kvh) * a.acc_stride + key0 + 8 * g;
    if (n == 0)
#pragma unroll
        for (int e = 0; e < 8; e++)
            if (any >> e & 1) dst[e] += sum[e];
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
    a.n_q = d->n_q; a.qg = d->n_q / d->n_kv; a.window = d->window; a.n_sink = d->n_sink;
    VX_REQUIRE((int64_t)d->max_T * a.qg < (1 << 30), "%s: max_T * n_q/n_kv is past 2^30 (max_T=%d)", who, d->max_T);
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
        a.min_tiles = 4;   // one a wave
        const int64_t most = ((int64_t)d->B * d->n_kv * tile_cap + a.min_tiles - 1) / a.min_tiles;
        const int grid = (int)std::min<int64_t>(most, 2 * ctx->n_cu);
        a.part_rows = rows;
        const size_t n_part = (size_t)2 * grid * rows;
        const size_t o_bytes = n_part * HDG * 4, ml_bytes = (n_part * sizeof(float2) + 255) / 256 * 256;
        const size_t st_bytes = d->acc ? (size_t)d->B * d->n_kv * rows * tile_cap * TILE * 4 : 0;
        void *scr;
        if (vx_ctx_scratch(ctx, o_bytes + ml_bytes + stat_bytes + st_bytes, &scr)) return -1;
        a.part_o = (float *)scr;
        a.part_ml = (float2 *)((char *)scr + o_bytes);
        a.stat = d->acc ? (float2 *)((char *)scr + o_bytes + ml_bytes) : nullptr;
        a.stash = d->acc ? (float *)((char *)scr + o_bytes + ml_bytes + stat_bytes) : nullptr;
        VX_LAUNCH(ctx, paged_split, dim3(grid), dim3(256), a);
        VX_LAUNCH(ctx, paged_join, dim3(rows, d->n_kv, d->B), dim3(256), a, grid);
        if (d->acc) VX_LAUNCH(ctx, paged_weigh, dim3((a.tile_cap + 7) / 8, d->n_kv, d->B), dim3(256), a);
        return 0;
    }
    void *scr = nullptr;
    if (d->acc && vx_ctx_scratch(ctx, stat_bytes, &scr)) return -1;
    a.stat = (float2 *)scr;
    VX_LAUNCH(ctx, paged_tile, dim3((rows + 63) / 64, d->n_kv, d->B), dim3(256), a);
    if (d->acc) VX_LAUNCH(ctx, paged_tile_weigh, dim3((a.tile_cap + 3) / 4, d->n_kv, d->B), dim3(256), a);
    return 0;
}
