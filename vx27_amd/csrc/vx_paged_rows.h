// The tile kernel of the paged KV caches: attention of more query rows than a
// decode call's (vx_paged_attn.h).
#pragma once
#include "vx_paged_attn.h"
#include "vx_paged_q4.h"

namespace {

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

template <bool Q4>
struct TileSmem {
    char k[2][2 * HALF], v[2][2 * HALF];     // [buffer][key block]
    char sm[Q4 ? 2 : 1][Q4 ? 4 * 512 : 16];  // 4-bit pages: s and m of a step's K blocks and V blocks, [buffer]
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

// 4-bit pages: row tiles of the longest token range from which the values are
// laid out in scratch, and the most tiles there (32 KiB each, K and V: 256 MiB).
// (In us with and without, 4 x 6000 | 1 x 30000 rows, tokens of 6 heads: 86
// tokens, five row tiles, 110, 108 | 138, 133; 107, six, 128, 144 | 151, 150;
// 170, eight, 191, 249 | 180, 194.)
constexpr int FLAT_ROWS = 6;
constexpr size_t FLAT_TILES = 8192;

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

// The values of 4-bit pages in scratch: every (sequence, KV head) has room for
// the tiles that its tokens see, in the order of their list; a tile is a block
// of K [32][256] and one of V [256][32], as in bf16 pages.
__device__ __forceinline__ size_t flat_at(const Args &a, const vx_pseq &s, int b, int kvh, int key) {
    const vx_tiles tl = tiles_of(a, s, 0, s.T - 1);
    const int tile = key / TILE, i = tile < tl.st ? tile : tile - tl.fm + tl.st;
    return (((size_t)b * a.p.n_kv + kvh) * a.tile_cap + i) * TILE * HDG;
}

// grid the most pieces there can be, block 256.
//
// PG_Q4, over 4-bit pages: the same kernel over values rounded to bf16.  A wave
// loads the codes of its quarter of a step a step earlier into registers, and
// the masks, fp32 FMAs and packs that make 16 bytes of LDS of a dword take the
// places of the direct loads between the MFMAs; s and m come through LDS.
// That makes a step a fifth longer (8192 tokens, window of 1024: 381 us), and
// every row tile does it again, so long token ranges have the values of what
// they see laid out once in scratch and read them from there: PG_FLAT.
enum { PG_BF16, PG_Q4, PG_FLAT };
template <int PAGES>
__global__ __launch_bounds__(256, 1) void paged_rows(Args a) {
    constexpr bool Q4 = PAGES == PG_Q4;
    __shared__ __attribute__((aligned(16))) TileSmem<Q4> sm;
    const uint16_t *const k_pool = PAGES == PG_FLAT ? a.flat_k : a.k_pages, *const v_pool = PAGES == PG_FLAT ? a.flat_v : a.v_pages;
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
    // Element (4-bit pages: byte) offsets in the pools of this wave's key blocks: lane i holds the
    // block of step base + i (past the list: its last block again), so a step
    // reads a lane and not the page table.
    int base = c0;
    uint32_t at_lo, at_hi;
    auto fill_at = [&]() {
        const int key = tl.at(min(2 * (base + lane) + (wave >> 1), tl.nt - 1)) * TILE;
        if constexpr (PAGES == PG_FLAT) {
            const uint64_t at = flat_at(a, s, b, kvh, key);
            at_lo = (uint32_t)at;
            at_hi = (uint32_t)(at >> 32);
            return;
        }
        const int slot = vx_page_slot(a.p, key);
        const int page = vx_page_checked(a.p, vx_table_word(a.p.table + (size_t)b * a.p.max_pages + slot));
        const uint64_t at = Q4 ? (uint64_t)vx_q4_block(a.p, page, kvh, key - slot * a.p.page_size) * VX_Q4_BLOCK
                               : (((uint64_t)page * a.p.n_kv + kvh) * a.p.page_size + (key - slot * a.p.page_size)) * HDG;
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
    auto dma_k = [&](size_t at, int buf, int j) { dma((const char *)(k_pool + at), ko[(j & 1) | ((j >> 2) << 1)], k_lds + buf * 2 * HALF, j); };
    auto dma_v = [&](size_t at, int buf, int j) { dma((const char *)(v_pool + at), vo, v_lds + buf * 2 * HALF, j); };

    // 4-bit pages: this wave's codes of a step, 16 rows of K (rows m of
    // operand block `wave % 2`) and 128 dims of V, and the places of their
    // 16-byte units in LDS.
    uint4 kc[2], vc[2];
    const int qg4 = lane >> 4, qn = lane & 15;
    const uint32_t kd = (uint32_t)((wave >> 1) * HALF + (8 * (qn >> 2) + 4 * (wave & 1) + (qn & 3)) * (HDG * 2) + ((qg4 ^ qn) << 4));
    const uint32_t vd = (uint32_t)((wave >> 1) * HALF + (128 * (wave & 1) + qn) * (TILE * 2) + ((qg4 ^ ((qn >> 1) & 3)) << 4));
    auto load_codes = [&](size_t at, const uint16_t *pool, uint4 (&x)[2]) {   // quads 2 (wave % 2), + 1
        const char *p = (const char *)pool + at + (128 * (wave & 1) + lane) * 16;
        x[0] = *(const uint4 *)p;
        x[1] = *(const uint4 *)(p + 1024);
    };
    // s and m of key block `wave / 2`: wave w % 2 = 0 takes K's, 1 V's
    auto load_scales = [&](size_t at_k, size_t at_v, int buf) {
        const uint32_t lds = __builtin_amdgcn_readfirstlane(vx_lds_addr(sm.sm[buf]) + wave * 512);
        if (lane < 32) dma16<0>((const char *)(wave & 1 ? a.v_pages : a.k_pages) + (wave & 1 ? at_v : at_k) + VX_Q4_S, lane * 16, lds);
    };
    float ksm[8];                              // s and m of this lane's row of K
    auto k_scales = [&](int buf) {
        const char *p = sm.sm[buf] + (wave & 2) * 512;
        const int row = 8 * (qn >> 2) + 4 * (wave & 1) + (qn & 3);
        const uint2 m = *(const uint2 *)(p + 256 + row * 8);
#pragma unroll
        for (int c = 0; c < 4; c++) {
            ksm[c] = vx_bf16_to_f32(*(const uint16_t *)(p + c * 64 + row * 2));
            ksm[4 + c] = __uint_as_float(c & 1 ? (c & 2 ? m.y : m.x) & 0xffff0000u : (c & 2 ? m.y : m.x) << 16);
        }
    };
    auto put8 = [&](char *p, const float (&x)[8]) { *(uint4 *)p = make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7])); };
    auto word4 = [](const uint4 &x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; };
    // dword j of this wave's eight of K: dims 128 (j / 4) + 32 (j % 4) + 8 g .. + 7 of its row
    auto put_k = [&](int buf, int j) {
        float x[8];
        vx_q4_codes_f32(word4(kc[j >> 2], j & 3), x);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = __builtin_fmaf(x[e], ksm[j >> 1], ksm[4 + (j >> 1)]);
        put8(sm.k[buf] + (kd ^ ((j & 3) << 6)) + (j >> 2) * 256, x);
    };
    // dword j of V: dim 64 (j / 4) + 16 (j % 4) + n of its 128, keys 8 g .. + 7
    // (s and m are read from LDS two dwords ahead of their use, v_scales(0) by the caller)
    uint4 vsm[2];
    float s8[8], m8[8];
    auto v_scales = [&](int scales, int half) {
        const char *p = sm.sm[scales] + ((wave & 2) + 1) * 512 + (2 * (wave & 1) + half) * 64 + qg4 * 16;
        vsm[0] = *(const uint4 *)p;
        vsm[1] = *(const uint4 *)(p + 256);
    };
    auto put_v = [&](int buf, int scales, int j) {
        float x[8];
        if ((j & 3) == 0) {
            vx_q4_f32(vsm[0], s8);
            vx_q4_f32(vsm[1], m8);
        }
        if (j == 2) v_scales(scales, 1);
        vx_q4_codes_f32(word4(vc[j >> 2], j & 3), x);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = __builtin_fmaf(x[e], s8[e], m8[e]);
        put8(sm.v[buf] + vd + j * 16 * TILE * 2, x);
    };

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
        if constexpr (Q4) {
            // K and V of the first step, then K of the second and the codes that the loop's first step stores
            load_codes(at_v, a.k_pages, kc);
            load_codes(at_v, a.v_pages, vc);
            load_scales(at_v, at_v, 0);
            load_scales(at_k, at_k, 1);
            __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
            vx_lds_barrier();
            k_scales(0);
#pragma unroll
            for (int j = 0; j < 8; j++) put_k(0, j);
            load_codes(at_k, a.k_pages, kc);
            v_scales(0, 0);
#pragma unroll
            for (int j = 0; j < 8; j++) put_v(0, 0, j);
            load_codes(at_k, a.v_pages, vc);
            k_scales(1);
#pragma unroll
            for (int j = 0; j < 8; j++) put_k(1, j);
            const size_t at_2 = at_of(c0 + 2);
            load_codes(at_2, a.k_pages, kc);
            vx_lds_barrier();                            // (buffer 0's scales have been read)
            load_scales(at_2, at_k, 0);                  // K's of step 2 and V's of step 1, as in the loop
            at_v = at_2;
            at_k = at_of(c0 + 3);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) dma_k(at_v, 0, j);
#pragma unroll
            for (int j = 0; j < 8; j++) dma_k(at_k, 1, j);
#pragma unroll
            for (int j = 0; j < 8; j++) dma_v(at_v, 0, j);
            at_v = at_k;
            at_k = at_of(c0 + 2);
        }
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
            if constexpr (Q4) k_scales(bk), v_scales(bk, 0);
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
                // (4-bit pages: the codes of K(c+2) and V(c+1) are in registers, those of K(c+3) and V(c+2) follow)
                if constexpr (Q4) {
                    if (i < 16) {
                        if (i & 1) put_v(bk ^ 1, bk, i >> 1);
                        else put_k(bk, i >> 1);
                    }
                    if (i == 16) load_codes(at_k, a.k_pages, kc);
                    if (i == 18) load_codes(at_v, a.v_pages, vc);
                    if (i == 20) load_scales(at_k, at_v, bk ^ 1);
                } else if (i < 16) {
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
                if (i == 1) at_v = at_k, at_k = at_of(c0 + c + (Q4 ? 4 : 3));
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
            if (c0 + c + (Q4 ? 6 : 5) > base + 63) {   // (one step in 60)
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
                const char *blk = (const char *)a.v_pages + (size_t)vx_q4_block(a.p, page, kvh, at) * VX_Q4_BLOCK;   // (4-bit pages)
                const uint16_t *vp = PAGES == PG_FLAT ? a.flat_v + flat_at(a, s, b, kvh, key0) + tid * TILE
                                                      : a.v_pages + vx_v_index(a.p.n_kv, a.p.page_size, page, kvh, at, tid);
                for (int j = 0; j < TILE; j++) {   // (of 4-bit pages as the steps rounded it: a value of 2^127 and more may be an infinity)
                    const float x = Q4 ? __uint_as_float(pack2(vx_q4_v_value(blk, j, tid), 0.0f) << 16) : vx_bf16_to_f32(vp[j]);
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

// grid (most tiles, n_kv, B), block 256: a tile's values into scratch; thread u
// takes 16-byte unit u of K's codes and of V's.
template <int PAGES>   // (PG_FLAT: only where it is launched)
__global__ __launch_bounds__(256) void paged_q4_flat(Args a) {
    const int i = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z, u = threadIdx.x, g = (u >> 4) & 3, n = u & 15;
    const vx_pseq s = vx_paged_seq(a.p, b);
    const vx_tiles tl = tiles_of(a, s, 0, s.T - 1);
    if (i >= tl.nt) return;
    const int key = tl.at(i) * TILE, page = vx_paged_page(a.p, b, key);
    const size_t block = (size_t)vx_q4_block(a.p, page, kvh, key - vx_page_slot(a.p, key) * a.p.page_size) * VX_Q4_BLOCK;
    const size_t out = (((size_t)b * a.p.n_kv + kvh) * a.tile_cap + i) * TILE * HDG;
    const char *kp = (const char *)a.k_pages + block, *vp = (const char *)a.v_pages + block;
    const uint4 kc = *(const uint4 *)(kp + u * 16), vc = *(const uint4 *)(vp + u * 16);
    const uint32_t kw[4] = {kc.x, kc.y, kc.z, kc.w}, vw[4] = {vc.x, vc.y, vc.z, vc.w};
    const int row = vx_q4_k_row(u), kh = (u >> 6) & 1, j = u >> 6;
    float ks[2], km[2], vs[8], vm[8];
#pragma unroll
    for (int c = 0; c < 2; c++) {
        ks[c] = vx_bf16_to_f32(*(const uint16_t *)(kp + VX_Q4_S + (2 * kh + c) * 64 + row * 2));
        km[c] = vx_bf16_to_f32(*(const uint16_t *)(kp + VX_Q4_M + row * 8 + (2 * kh + c) * 2));
    }
    vx_q4_f32(*(const uint4 *)(vp + VX_Q4_S + j * 64 + g * 16), vs);
    vx_q4_f32(*(const uint4 *)(vp + VX_Q4_M + j * 64 + g * 16), vm);
#pragma unroll
    for (int q = 0; q < 4; q++) {
        float x[8];
        vx_q4_codes_f32(kw[q], x);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = __builtin_fmaf(x[e], ks[q >> 1], km[q >> 1]);
        *(uint4 *)(a.flat_k + out + row * HDG + 128 * kh + 32 * q + 8 * g) = make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
        vx_q4_codes_f32(vw[q], x);
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = __builtin_fmaf(x[e], vs[e], vm[e]);
        *(uint4 *)(a.flat_v + out + (64 * j + 16 * q + n) * TILE + 8 * g) = make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
    }
}

// Launches the tile kernel's calls, with `stat_bytes` of scratch for the rows'
// statistics.
template <bool Q4>
int rows_launch(const char *who, vx27_hip_ctx *ctx, const vx27_paged_attn_desc *d, Args &a, int rows, size_t stat_bytes) {
    const int n_rt = (rows + TR - 1) / TR, n_cu = a.cus = ctx->n_cu;
    VX_REQUIRE((int64_t)d->B * n_rt < (1ll << 31) - PLAN, "%s: more than 2^31 row tiles (B=%d max_T=%d)", who, d->B, d->max_T);
    // every token range ends in one tile that it need not fill; paged_plan makes at most 3/2 n_cu cuts, so twice
    // as many parts at most
    const int64_t cuts = (int64_t)n_cu * 3 / 2, items = ((int64_t)d->n_tok * a.qg / TR + d->B) * d->n_kv;
    VX_REQUIRE(items + cuts < (1 << 24), "%s: more than 2^24 row tiles (B=%d n_kv=%d n_tok=%d)", who, d->B, d->n_kv, d->n_tok);
    const size_t ml_bytes = (size_t)2 * cuts * TR * sizeof(float2), plan_bytes = 256, piece_bytes = (size_t)(items + cuts) * sizeof(RowPiece);
    const size_t join_bytes = ((size_t)cuts * sizeof(RowJoin) + 255) / 256 * 256;
    void *scr;
    const size_t flat_tiles = (size_t)d->B * d->n_kv * a.tile_cap;
    const bool flat = Q4 && n_rt >= FLAT_ROWS && flat_tiles <= FLAT_TILES;
    const size_t flat_bytes = flat ? flat_tiles * HALF : 0, parts_bytes = (size_t)2 * cuts * TR * HDG * 4;
    if (vx_ctx_scratch(ctx, 2 * flat_bytes + stat_bytes + ml_bytes + plan_bytes + join_bytes + parts_bytes + piece_bytes, &scr)) return -1;
    char *at = (char *)scr + 2 * flat_bytes;
    a.stat = d->acc ? (float2 *)at : nullptr;
    a.part_ml = (float2 *)(at += stat_bytes);
    a.plan = (RowPlan *)(at += ml_bytes);
    a.joins = (RowJoin *)(at += plan_bytes);
    a.part_o = (float *)(at += join_bytes);
    a.pieces = (RowPiece *)(at += parts_bytes);
    VX_LAUNCH(ctx, paged_plan, dim3(1), dim3(PLAN), a, n_rt, n_cu, (int)(items + cuts));
    const dim3 grid((unsigned)(items + cuts));
    if constexpr (Q4) if (flat) {
        a.flat_k = (uint16_t *)scr;
        a.flat_v = (uint16_t *)((char *)scr + flat_bytes);
        VX_LAUNCH_NAMED(ctx, "paged_q4_flat", (paged_q4_flat<PG_FLAT>), dim3(a.tile_cap, d->n_kv, d->B), dim3(256), a);
        VX_LAUNCH_NAMED(ctx, "paged_rows_flat", (paged_rows<PG_FLAT>), grid, dim3(256), a);
    }
    if (!flat) VX_LAUNCH_NAMED(ctx, Q4 ? "paged_rows_q4" : "paged_rows", (paged_rows<Q4 ? PG_Q4 : PG_BF16>), grid, dim3(256), a);
    VX_LAUNCH(ctx, paged_rows_join, dim3(8 * n_cu), dim3(256), a);
    return 0;
}

}  // namespace
