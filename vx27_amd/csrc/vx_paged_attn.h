// Attention over the paged KV caches: what the kernels of the bf16 and of the
// 4-bit pages share.  Query rows, their outputs, and the decode calls' list of
// key tiles with the join of its parts.
#pragma once
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
    int block_rows;              // 4-bit pages: query rows of a list entry (16 or 8)
    int *before;                 // B > 64: [B + 1] units before each sequence
    // tiles (scratch)
    int cus;
    RowPlan *plan;
    RowPiece *pieces;
    RowJoin *joins;
    uint16_t *flat_k, *flat_v;   // 4-bit pages: values in scratch, [B][n_kv][tile_cap][32 x 256]
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
__device__ __forceinline__ bool is_finite(float x) { return __builtin_fabsf(x) < INFINITY; }

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

// A decode call's list of tiles.
// 16 rows are what one MFMA tile holds, so this form ends there: a third token
// of 6 heads goes to the tiles below (4 x 131072 rows: 328 us for two tokens
// a sequence, 377 for three there; one of 1000 rows: 14 and 26).
// The list of a call's tiles: up to 64 sequences are held one a lane and read
// once; of more, paged_units adds up the units before each first (each
// workgroup doing so for itself took 3.2 ms for 4096 sequences of 100 rows).
// BL: a sequence's query rows are cut into blocks of block_rows, and the list
// holds every (KV head, block)'s tiles; else a KV head's rows are one block.
template <bool BL>
__device__ __forceinline__ int seq_blocks(const Args &a, const vx_pseq &s) { return BL ? (s.T * a.qg + a.block_rows - 1) / a.block_rows : 1; }
// A block's tiles in units of the list.  BL: rounded up to min_tiles, as a
// workgroup's share is: in small calls, where that is the share, none takes the
// end of one block and the start of the next, which costs it the queries, first
// loads and merge of both (one sequence of 4000 rows 20 us, so 14; 16 of 200 rows
// 19, 14; a prompt of 20 tokens 22, 14).  Rounded shares are the better where
// they are a few tiles too (200 x 100 rows 39 us against 46, 24 x 700 22, 24;
// but 64 x 300 28, 23).
template <bool BL>
__device__ __forceinline__ int list_tiles(const Args &a, int nt) { return BL ? (nt + a.min_tiles - 1) / a.min_tiles * a.min_tiles : nt; }
// (a workgroup's share may end that much past the list)
constexpr int64_t MOST_UNITS = (1ll << 31) - 65536;
struct Units {
    vx_pseq s;          // of sequence `lane` (B <= 64)
    vx_tiles t;
    int upto;           // units of sequences 0 .. lane
    int total, chunk;
};
template <bool BL>
__device__ __forceinline__ int seq_units(const Args &a, int b, vx_pseq &s, vx_tiles &t) {
    s = vx_paged_seq(a.p, b);
    t = tiles_of(a, s, 0, s.T - 1);
    return list_tiles<BL>(a, t.nt) * a.p.n_kv * seq_blocks<BL>(a, s);
}
template <bool BL>
__device__ __forceinline__ Units units_of(const Args &a, int grid) {
    const int lane = threadIdx.x & 63;
    Units u;
    if (a.p.B <= 64) {
        const int n = seq_units<BL>(a, min(lane, a.p.B - 1), u.s, u.t);
        u.upto = vx_wave_scan(lane < a.p.B ? n : 0);
        u.total = __builtin_amdgcn_readlane(u.upto, 63);
    } else {
        u.total = a.before[a.p.B];
    }
    u.chunk = list_tiles<BL>(a, max((u.total + grid - 1) / grid, a.min_tiles));
    return u;
}
// Sequence b: itself, its tiles, and the units before it.
template <bool BL>
__device__ __forceinline__ int units_before(const Args &a, const Units &u, int b, vx_pseq &s, vx_tiles &t) {
    if (a.p.B <= 64) {
        auto get = [&](int x) { return __builtin_amdgcn_readlane(x, b); };
        s = {get(u.s.start), get(u.s.T), get(u.s.len), get(u.s.row0)};
        t = {get(u.t.st), get(u.t.fm), get(u.t.nt)};
        return get(u.upto) - list_tiles<BL>(a, t.nt) * a.p.n_kv * seq_blocks<BL>(a, s);
    }
    seq_units<BL>(a, b, s, t);
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

// grid 1, block 1024: the units before each sequence, and in all.  CHECK: where
// token ranges that overlap, an error that vx_paged_seq flags, could list more
// than the host has room for: then none (a barrier and sums in 64 bits, 0.8 us).
template <bool BL, bool CHECK>
__global__ __launch_bounds__(1024) void paged_units(Args a) {
    __shared__ int s_sum[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (a.p.B + 1023) / 1024, b0 = min(tid * per, a.p.B), b1 = min(b0 + per, a.p.B);
    vx_pseq s;
    vx_tiles t;
    int sum = 0;
    bool over = false;
    if constexpr (CHECK) {
        __shared__ int64_t s_all[16];
        int64_t all = 0;
        for (int b = b0; b < b1; b++) all += seq_units<BL>(a, b, s, t);
        sum = (int)all;
        for (int off = 32; off >= 1; off >>= 1) all += __shfl_xor(all, off, 64);
        if (lane == 0) s_all[wave] = all;
        __syncthreads();
        all = 0;
        for (int w = 0; w < 16; w++) all += s_all[w];
        over = all >= MOST_UNITS;
        if (over) sum = 0, *a.p.err_flag = 1;
    } else {
        for (int b = b0; b < b1; b++) sum += seq_units<BL>(a, b, s, t);
    }
    int at = vx_wave_scan(sum);
    if (lane == 63) s_sum[wave] = at;
    __syncthreads();
    for (int w = 0; w < wave; w++) at += s_sum[w];
    if (tid == 1023) a.before[a.p.B] = at;
    at -= sum;
    for (int b = b0; b < b1; b++) {
        a.before[b] = at;
        if (!CHECK || !over) at += seq_units<BL>(a, b, s, t);
    }
}

// grid (most rows of a block, n_kv, B), or BL (n_kv x most blocks, most rows of
// a block, B), block 256 (4-7 us): merges the parts of one query row, in
// their order: wave w takes parts w, w + 4, ..., eight in flight; a row of a
// sequence without rows gets 0.
template <bool BL>
__global__ __launch_bounds__(256) void paged_join(Args a, int grid) {
    const int b = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Units un = units_of<BL>(a, grid);
    vx_pseq s;
    vx_tiles tl;
    const int before = units_before<BL>(a, un, b, s, tl), nb = seq_blocks<BL>(a, s);
    const int kvh = BL ? (int)blockIdx.x % a.p.n_kv : (int)blockIdx.y, blk = BL ? (int)blockIdx.x / a.p.n_kv : 0;
    const int pr = BL ? blockIdx.y : blockIdx.x, r = BL ? blk * a.block_rows + pr : pr;   // the row, in its block and in all
    if (r >= s.T * a.qg) return;
    const int n_list = list_tiles<BL>(a, tl.nt), p0 = before + (kvh * nb + blk) * n_list, p1 = p0 + n_list;
    const int t = row_tok(a, r), tok = s.start + t, h = row_head(a, kvh, r, t);
    const int g0 = p0 / un.chunk, g1 = (p1 - 1) / un.chunk;
    if ((tl.nt > 0 && g0 == g1) || (BL && p1 > un.total)) return;   // (whole, or no list: paged_units)
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
            const size_t pi = (size_t)(2 * w + (w == g0 && p0 != w * un.chunk ? 1 : 0)) * a.part_rows + pr;
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

// The checks and arguments of an attention call: 1, 0 where there is nothing
// to do, or -1.
int attn_fill(const char *who, vx27_hip_ctx *ctx, const vx27_paged_attn_desc *d, Args &a) {
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
    return 1;
}

}  // namespace
