// Attention over a paged 4-bit KV cache on gfx950 (layout: vx_paged_q4.h):
// what vx27_hip_paged_attn computes, over the values that the codes stand for.
//
// With a row's scales s_g and minima m_g of its four groups of 64 dims,
//   q . k_j = sum_g s_jg (q_g . c_jg) + m_jg (sum of q_g)
//   sum_j p_j v_j = sum_j (p_j s_jg) c_jg + p_j m_jg      for the dims of group g,
// so no dim is ever decoded: the codes are exact bf16 operands, s multiplies
// the scores of a group on their way out of the MFMAs and the weights on their
// way in, and the minima's sums are MFMAs of their own (one for 16 keys' scores,
// one for a tile's outputs).
//
// The split kernel on 4 x 131072 rows of 4 KV heads (604 MB): 108 us, 5.6 TB/s
// of 7.2 (its loads alone 90).  A tile is 670 VALU instructions, half of them the
// codes' masks and conversions and the weights' parts, which keep the VALU busy
// for two thirds of the time at the two waves a SIMD that 235 registers allow.
// Ragged windows of 32 sequences: 41 us for 141 MB, of which some 10 are the
// first loads' chain (lengths, table, blocks) and the waves' merge.
#include "vx_paged_q4.h"
#include "vx_paged_rows.h"

namespace {

constexpr int GROUPS = HDG / VX_Q4_GROUP;

// The lane, opaque: what is formed from it stays where it is used, and does not
// take a register through the loops around.
__device__ __forceinline__ int lane_here() {
    int lane = threadIdx.x & 63;
    __asm__ volatile("" : "+v"(lane));
    return lane;
}
// Block `block` of a pool into LDS, a wave's five loads (in flight: the caller
// counts them).  ONCE: codes that no other workgroup reads, nontemporal (4 x
// 131072 rows 111 us against 122; tiles that three blocks of rows read 55 against
// 53).
constexpr int LOADS = 5;
template <bool ONCE>
__device__ __forceinline__ void load_block(const uint16_t *pool, uint32_t block, uint32_t lds) {
    const int lane = lane_here();
    const char *base = (const char *)pool + (size_t)block * VX_Q4_BLOCK;
    uint32_t saved;
    if (ONCE) {
        __asm__ volatile(
            "s_mov_b32 %0, m0\n\t"
            "s_mov_b32 m0, %3\n\t"
            "s_nop 0\n\t"
            "global_load_lds_dwordx4 %1, %2 nt\n\t"
            "global_load_lds_dwordx4 %1, %2 offset:1024 nt\n\t"
            "global_load_lds_dwordx4 %1, %2 offset:2048 nt\n\t"
            "global_load_lds_dwordx4 %1, %2 offset:%4 nt\n\t"
            "s_mov_b32 m0, %0"
            : "=&s"(saved)
            : "v"(lane * 16), "s"(base), "s"(lds), "n"(3 * 1024)
            : "memory");
    } else {
        __asm__ volatile(
            "s_mov_b32 %0, m0\n\t"
            "s_mov_b32 m0, %3\n\t"
            "s_nop 0\n\t"
            "global_load_lds_dwordx4 %1, %2\n\t"
            "global_load_lds_dwordx4 %1, %2 offset:1024\n\t"
            "global_load_lds_dwordx4 %1, %2 offset:2048\n\t"
            "global_load_lds_dwordx4 %1, %2 offset:%4\n\t"
            "s_mov_b32 m0, %0"
            : "=&s"(saved)
            : "v"(lane * 16), "s"(base), "s"(lds), "n"(3 * 1024)
            : "memory");
    }
    if (lane < 32) vx_dma16(base + VX_Q4_S, lane * 16, lds + VX_Q4_S);
}
// Waits until at most `blocks` of this wave's blocks are in flight.
__device__ __forceinline__ void wait_blocks(int blocks) {
    if (blocks >= 3) __asm__ volatile("s_waitcnt vmcnt(%0)" : : "n"(3 * LOADS) : "memory");
    else if (blocks == 2) __asm__ volatile("s_waitcnt vmcnt(%0)" : : "n"(2 * LOADS) : "memory");
    else if (blocks == 1) __asm__ volatile("s_waitcnt vmcnt(%0)" : : "n"(LOADS) : "memory");
    else __asm__ volatile("s_waitcnt vmcnt(0)" : : : "memory");
}
__device__ __forceinline__ uint32_t word(const uint4 &x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; }

// A lane's share of a block's codes and scales; m as it is used.
struct Tile {
    uint4 c[4], s[GROUPS];
};
struct KTile : Tile {
    uint2 m[2];
};
struct VTile : Tile {
    bf16x8_t m;
};
__device__ __forceinline__ void read_tile(const char *blk, int lane, Tile &t) {
#pragma unroll
    for (int j = 0; j < 4; j++) t.c[j] = *(const uint4 *)(blk + lane * 16 + j * 1024);
#pragma unroll
    for (int j = 0; j < GROUPS; j++) t.s[j] = *(const uint4 *)(blk + VX_Q4_S + (lane >> 4) * 16 + j * 64);
}
__device__ __forceinline__ void read_k(const char *blk, KTile &t) {
    const int lane = lane_here(), n = lane & 15;
    read_tile(blk, lane, t);
#pragma unroll
    for (int r = 0; r < 2; r++) t.m[r] = *(const uint2 *)(blk + VX_Q4_M + (8 * (n >> 2) + (n & 3)) * 8 + r * 32);
}
__device__ __forceinline__ void read_v(const char *blk, VTile &t) {
    const int lane = lane_here();
    read_tile(blk, lane, t);
    t.m = *(const bf16x8_t *)(blk + VX_Q4_M + (lane & 3) * 64 + (lane >> 4) * 16);
}

// One wave's state for ROWS query rows: 16, or 8 that take the 16 columns
// twice, the first with the weights rounded to bf16 and the second with what
// that left (two parts at the price of one).
template <int ROWS>
struct Rows {
    bf16x8_t q[8], qs;           // qs: the groups' sums of q against the minima
    floatx4_t o[16], om;         // om: lanes g = 0, element e: group e's sum of p m
    float m, l;
};
template <int ROWS>
__device__ __forceinline__ void rows_begin(const Args &a, const vx_pseq &s, int kvh, int r0, Rows<ROWS> &w) {
    const int lane = lane_here(), g = lane >> 4, n = lane & 15, r = r0 + n % ROWS, t = row_tok(a, r);
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
    // The sums in three bf16 parts (all 24 bits): k-slots 0-3 and 4-7 of lane
    // group 0 and 0-3 of group 1, against operands that hold the minima in
    // each of these places.
#pragma unroll
    for (int e = 0; e < 8; e++) w.qs[e] = (__bf16)0.0f;
#pragma unroll
    for (int c = 0; c < GROUPS; c++) {
        float x = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) x += (float)w.q[2 * c][e] + (float)w.q[2 * c + 1][e];
        x += __shfl_xor(x, 16, 64);
        x += __shfl_xor(x, 32, 64);
        const __bf16 hi = (__bf16)x, mid = (__bf16)(x - (float)hi), lo = (__bf16)(x - (float)hi - (float)mid);
        w.qs[c] = g == 0 ? hi : g == 1 ? lo : (__bf16)0.0f;
        w.qs[4 + c] = g == 0 ? mid : (__bf16)0.0f;
    }
#pragma unroll
    for (int d = 0; d < 16; d++) w.o[d] = (floatx4_t){0.f, 0.f, 0.f, 0.f};
    w.om = (floatx4_t){0.f, 0.f, 0.f, 0.f};
    w.m = -INFINITY;
    w.l = 0.0f;
}

// Scores of 32 keys: lane (g,n) gets keys 8g + 0..7 of row n.
template <int ROWS>
__device__ __forceinline__ void score_tile(const KTile &t, const Rows<ROWS> &w, float (&s)[8]) {
    floatx4_t acc[2];
#pragma unroll
    for (int r = 0; r < 2; r++) {
        const uint4 m = make_uint4(t.m[r].x, t.m[r].y, t.m[r].x, t.m[r].y);
        acc[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, m), w.qs, (floatx4_t){0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
    }
#pragma unroll
    for (int c = 0; c < GROUPS; c++) {
        float sc[8];
        vx_q4_f32(t.s[c], sc);
#pragma unroll
        for (int r = 0; r < 2; r++) {
            floatx4_t x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < 2; i++)
                x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vx_q4_codes(word(t.c[2 * r + c / 2], 2 * (c & 1) + i)), w.q[2 * c + i], x, 0, 0, 0);
#pragma unroll
            for (int e = 0; e < 4; e++) acc[r][e] = __builtin_fmaf(x[e], sc[4 * r + e], acc[r][e]);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int e = 0; e < 8; e++) s[e] = acc[e >> 2][e & 3];
}

// Eight weights as two bf16 parts, h and x - h.  (One part is not enough for
// bf16 outputs either: the codes' and the minima's sums are each some 2.5 times
// a value and cancel, so that its rounding of 2^-9 became 0.005 of the output.)
// Of 16 rows they are operands of two MFMAs; of 8 the two halves of the 16
// columns, -h (rest 0) and x - h (rest 1), and the difference of the columns is
// the sum.  h is x rounded, which leaves 2^-18 of x; CUT: cut off, which leaves
// 2^-16 and is less work (the windows of 32 sequences 46.5 us against 48.5):
// enough below an output in bf16.
struct Weights {
    bf16x8_t hi, lo;
};
template <int ROWS, bool CUT>
__device__ __forceinline__ Weights weights8(const float (&x)[8], float rest) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float u = __uint_as_float(__float_as_uint(x[2 * i]) & 0xffff0000u), v = __uint_as_float(__float_as_uint(x[2 * i + 1]) & 0xffff0000u);
        if (!CUT) {
            h[i] = pack2(x[2 * i], x[2 * i + 1]);
            u = __uint_as_float(h[i] << 16);
            v = __uint_as_float(h[i] & 0xffff0000u);
        }
        if (ROWS == 16) l[i] = pack2(x[2 * i] - u, x[2 * i + 1] - v);
        else h[i] = pack2(__builtin_fmaf(x[2 * i], rest, -u), __builtin_fmaf(x[2 * i + 1], rest, -v));
    }
    Weights w;
    w.hi = __builtin_bit_cast(bf16x8_t, make_uint4(h[0], h[1], h[2], h[3]));
    if (ROWS == 16) w.lo = __builtin_bit_cast(bf16x8_t, make_uint4(l[0], l[1], l[2], l[3]));
    return w;
}
template <int ROWS>
__device__ __forceinline__ floatx4_t weigh(bf16x8_t x, const Weights &w, floatx4_t o) {
    o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, w.hi, o, 0, 0, 0);
    if (ROWS == 16) o = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, w.lo, o, 0, 0, 0);
    return o;
}

// A row's reference lies 2^AHEAD above the maximum at which it last moved, and
// moves once a score is past it, so that O (68 instructions) is rescaled in fewer
// tiles than every second, as where it follows the maximum.  Weights are at most 1.
// (The further ahead, the more rows' heaviest weights are no powers of two, whose
// parts are exact: with 2^8 the error of fp32 outputs over 131072 rows grows from
// 4e-6 to 8e-6, for 1% of the time.)
constexpr int AHEAD = 1;

// The maximum over lanes l, l ^ 16, l ^ 32, l ^ 48 (the VALU's exchanges: a
// swapped pair holds a lane's own value and its partner's).
__device__ __forceinline__ float over_groups(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
// x over the 16 lanes of a lane group, by OR or AND.
template <bool AND>
__device__ __forceinline__ uint32_t over_rows(uint32_t x) {
    auto with = [&](int y) { x = AND ? x & (uint32_t)y : x | (uint32_t)y; };
    with(vx_dpp_i<0xB1, 0xF>((int)x));
    with(vx_dpp_i<0x4E, 0xF>((int)x));
    with(vx_dpp_i<0x124, 0xF>((int)x));
    with(vx_dpp_i<0x128, 0xF>((int)x));
    return x;
}

// Online softmax and P V of one tile.  `whole`: every row sees every key.  Else
// s and m of keys that no row sees become zero, so that what stale rows hold
// cannot get in.
template <int ROWS, bool CUT>
__device__ __forceinline__ void attend_tile(Rows<ROWS> &w, bool whole, float (&x)[8], const vx_sight &v, int key0, VTile &t) {
    const int lane = lane_here(), g = lane >> 4;
    const float rest = ROWS == 8 && (lane & 8) ? 1.0f : 0.0f;
    uint32_t any = 0xffu, all = 0xffu;           // of keys 8g + 0..7: those that some row sees, and that every row does
    if (!whole) {
        const uint32_t sees = (v.block(key0) >> (8 * g)) & 0xffu;
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (sees >> e) & 1 ? x[e] : -INFINITY;
        any = over_rows<false>(sees);
        all = over_rows<true>(sees);
    }
    float mt = x[0];
#pragma unroll
    for (int e = 1; e < 8; e++) mt = fmaxf(mt, x[e]);
    mt = over_groups(mt) * SC2;
    if (__any(mt > w.m)) {
        const bool up = mt > w.m;
        const float to = mt + AHEAD, alpha = up ? __builtin_amdgcn_exp2f(w.m - to) : 1.0f;
        w.m = up ? to : w.m;
        w.l *= alpha;
#pragma unroll
        for (int d = 0; d < 16; d++) w.o[d] *= alpha;
        w.om *= alpha;
    }
    // (nothing seen yet, or NaN scores alone: the reference is 0, so that those stay NaN)
    const float ref = w.m == -INFINITY ? 0.0f : w.m;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        x[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[e], SC2, -ref));
        w.l += x[e];
    }
    if (!whole) {
        uint32_t m[4], keep[4], odd = 0;         // odd: bits 15 and 31, where an exponent of all ones carries into them
#pragma unroll
        for (int i = 0; i < 4; i++) {
            keep[i] = ((any >> (2 * i)) & 1) * 0xffffu | ((any >> (2 * i + 1)) & 1) * 0xffff0000u;
            m[i] = word(__builtin_bit_cast(uint4, t.m), i) & keep[i];
            odd |= (m[i] & 0x7f807f80u) + 0x00800080u;
        }
        t.m = __builtin_bit_cast(bf16x8_t, make_uint4(m[0], m[1], m[2], m[3]));
#pragma unroll
        for (int c = 0; c < GROUPS; c++) t.s[c] = make_uint4(t.s[c].x & keep[0], t.s[c].y & keep[1], t.s[c].z & keep[2], t.s[c].w & keep[3]);
        if (__builtin_expect(__any((odd & 0x80008000u) && any != all), 0)) {
            // A key that some rows see and others do not, with a minimum of NaN
            // (a group that held an infinity or a NaN): 0 times that would
            // reach the others.  It goes to the rows that see it by addition
            // and out of the product.
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const bool bad_here = ((any & ~all) >> e) & 1 && !is_finite((float)t.m[e]);
                uint64_t bad = __ballot(bad_here);
                while (bad) {
                    const int gk = __builtin_ctzll(bad) >> 4;
                    bad &= ~(0xffffull << (16 * gk));
                    const bool own = v.sees(key0 + 8 * gk + e);
#pragma unroll
                    for (int c = 0; c < GROUPS; c++) {
                        const float y = __shfl((float)t.m[e], 16 * gk + c, 64);
                        if (own && !is_finite(y)) w.om[c] += y;
                    }
                }
                if (bad_here) t.m[e] = (__bf16)0.0f;
            }
        }
    }
    w.om = weigh<ROWS>(t.m, weights8<ROWS, CUT>(x, rest), w.om);
#pragma unroll
    for (int c = 0; c < GROUPS; c++) {
        float y[8];
        vx_q4_f32(t.s[c], y);
#pragma unroll
        for (int e = 0; e < 8; e++) y[e] *= x[e];
        const Weights pw = weights8<ROWS, CUT>(y, rest);
#pragma unroll
        for (int i = 0; i < 4; i++) w.o[4 * c + i] = weigh<ROWS>(vx_q4_codes(word(t.c[c], i)), pw, w.o[4 * c + i]);
        __builtin_amdgcn_sched_barrier(0);
    }
}

__device__ __forceinline__ float both_halves(float x) {   // what lane ^ 8 has less the lane's own (weights8)
    return __int_as_float(vx_dpp_i<0x128, 0xF>(__float_as_int(x))) - x;
}

// The list of tiles is cut evenly over the workgroups, as the bf16 pages' (see
// paged_split): every (sequence, KV head, block of ROWS query rows) takes its
// tiles, wave w of a workgroup tiles w, w + 4, ...  A wave has a ring of DEPTH
// tiles in LDS (K's block, V's block), filled by direct loads that many tiles
// ahead.
constexpr int DEPTH = 2, RING = DEPTH * 2 * VX_Q4_BLOCK;
template <int ROWS, bool CUT>
__global__ __launch_bounds__(256, 2) void paged_q4_split(Args a) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    static_assert(RING >= ROWS * HDG * 4 && DEPTH == 2, "the waves' results take the rings' place; the waits count two tiles");
    __shared__ __attribute__((aligned(16))) char ring[4][RING];
    __shared__ float s_m[4][ROWS], s_l[4][ROWS];
    float (*s_o)[ROWS * HDG] = (float (*)[ROWS * HDG])ring;
    const Units un = units_of<true>(a, gridDim.x);
    // The dispatcher deals workgroups round-robin over the 8 XCDs: each XCD takes a
    // run of the shares, so that the blocks of rows that read the same tiles at the
    // same time share its L2 (8 x 20011 rows of 6 tokens 53.0 us, so 51.8; one block,
    // windows of 32 sequences 46.1, 45.3).
    const int xcd = blockIdx.x & 7, more = gridDim.x & 7, wg = xcd * (int)(gridDim.x >> 3) + min(xcd, more) + (int)(blockIdx.x >> 3);
    const int u0 = wg * un.chunk, u1 = min(u0 + un.chunk, un.total);
    if (u0 >= u1) return;
    int b = units_find(a, un, u0);
    vx_pseq s;
    vx_tiles tl;
    int before = units_before<true>(a, un, b, s, tl);
    for (int u = u0; u < u1;) {
        const int nb = seq_blocks<true>(a, s), n_list = list_tiles<true>(a, tl.nt), all = n_list * a.p.n_kv * nb;
        if (u >= before + all) {
            before += all;
            b++;
            if (a.p.B <= 64) units_before<true>(a, un, b, s, tl);
            else seq_units<true>(a, b, s, tl);
            continue;
        }
        const int item = (u - before) / n_list, i0 = (u - before) - item * n_list;
        const int kvh = item / nb, r0 = (item - kvh * nb) * ROWS;
        const int cnt = min(n_list - i0, u1 - u), real = min(cnt, tl.nt - i0);
        const int R = min(s.T * a.qg - r0, ROWS);
        const int mine = (real - wave + 3) / 4;     // this wave's tiles: i0 + wave + 4 j
        // lane i holds the block of this wave's tile 64 k + i
        uint32_t blocks = 0;
        auto look_up = [&](int j) {
            const int key = tl.at(i0 + wave + 4 * min(j + lane, mine - 1)) * TILE;
            const int page = vx_paged_page(a.p, b, key);
            blocks = vx_q4_block(a.p, page, kvh, key - vx_page_slot(a.p, key) * a.p.page_size);
        };
        const uint32_t ring_lds = vx_lds_addr(ring[0]) + wave * RING;
        auto slot_of = [&](int j) { return (j % DEPTH) * 2 * VX_Q4_BLOCK; };
        __asm__ volatile("s_waitcnt vmcnt(0)" : : : "memory");   // (nothing else is counted from here on)
        if (mine > 0) {
            look_up(0);
#pragma unroll
            for (int j = 0; j < DEPTH; j++) {
                if (j >= mine) break;
                load_block<ROWS == 8>(a.k_pages, __builtin_amdgcn_readlane(blocks, j), ring_lds + slot_of(j));
                load_block<ROWS == 8>(a.v_pages, __builtin_amdgcn_readlane(blocks, j), ring_lds + slot_of(j) + VX_Q4_BLOCK);
            }
        }
        Rows<ROWS> w;
        rows_begin<ROWS>(a, s, kvh, r0, w);
        const vx_sight v = sight_of(a, s, r0 + min(lane % ROWS, R - 1));   // (columns past the last row: as the last, unused)
        // tiles whose keys all rows see: from row `from` on or below the sinks' end, up to row `upto`
        const int upto = vx_paged_sight(s, row_tok(a, r0), a.window, a.n_sink).i, from = vx_paged_sight(s, row_tok(a, r0 + R - 1), a.window, a.n_sink).lo;
        auto whole_tile = [&](int key0) { return key0 + TILE - 1 <= upto && (key0 >= from || key0 + TILE <= a.n_sink); };
        for (int j = 0; j < mine; j++) {
            const char *blk = ring[wave] + slot_of(j);
            const int left = mine - 1 - j;
            const bool more = left >= DEPTH;     // the places of this tile's blocks then take the tile's DEPTH on
            float sc[8];
            {
                KTile kt;
                wait_blocks(left ? 3 : 1);       // (V, and K and V of the next tile, may be in flight)
                read_k(blk, kt);
                score_tile<ROWS>(kt, w, sc);
            }
            __asm__ volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
            if (more) {
                if (((j + DEPTH) & 63) == 0) look_up(j + DEPTH);
                load_block<ROWS == 8>(a.k_pages, __builtin_amdgcn_readlane(blocks, (j + DEPTH) & 63), ring_lds + slot_of(j));
            }
            VTile vt;
            wait_blocks(more ? 3 : left ? 2 : 0);
            read_v(blk + VX_Q4_BLOCK, vt);
            const int key0 = tl.at(i0 + wave + 4 * j) * TILE;
            attend_tile<ROWS, CUT>(w, whole_tile(key0), sc, v, key0, vt);
            __asm__ volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
            if (more) load_block<ROWS == 8>(a.v_pages, __builtin_amdgcn_readlane(blocks, (j + DEPTH) & 63), ring_lds + slot_of(j) + VX_Q4_BLOCK);
        }
        const int ln = lane_here(), g = ln >> 4, n = ln & 15;
        w.l += __shfl_xor(w.l, 16, 64);
        w.l += __shfl_xor(w.l, 32, 64);
#pragma unroll
        for (int c = 0; c < GROUPS; c++) {
            float om = w.om[c];
            if (ROWS == 8) om = both_halves(om);
            om = __shfl(om, n, 64);
#pragma unroll
            for (int i = 0; i < 4; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) w.o[4 * c + i][e] = (ROWS == 8 ? both_halves(w.o[4 * c + i][e]) : w.o[4 * c + i][e]) + om;
        }
        // the four waves' results through LDS (16-byte units swizzled by the row)
        vx_lds_barrier();                        // (every wave is done with its ring)
        if (n < R) {
#pragma unroll
            for (int d = 0; d < 16; d++) *(floatx4_t *)&s_o[wave][n * HDG + (((4 * d + g) ^ n) << 2)] = w.o[d];
            if (g == 0) {
                s_m[wave][n] = w.m;
                s_l[wave][n] = w.l;
            }
        }
        vx_lds_barrier();
        // wave w merges rows w, w + 4, ..., lane L dims 4L .. 4L + 3
        const bool whole = cnt == n_list;
        const int slot = 2 * wg + (u == u0 ? 0 : 1);
        for (int r = wave; r < R; r += 4) {
            const int t = row_tok(a, r0 + r), tok = s.start + t, h = row_head(a, kvh, r0 + r, t);
            float4 gt = make_float4(0.f, 0.f, 0.f, 0.f);
            if (whole && a.gate) gt = gate_row(a, tok, h);
            float m[4], l[4];
            float4 o[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                m[k] = s_m[k][r];
                l[k] = s_l[k][r];
                o[k] = *(const float4 *)&s_o[k][r * HDG + ((ln ^ r) << 2)];
            }
            const float M = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
            float L = 0.0f;
            float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < 4; k++) add_part(O, L, o[k], l[k], m[k] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[k] - M));
            if (whole) {
                row_finish(a, tok, h, O, M, L, gt);
            } else {
                *(float4 *)(a.part_o + ((size_t)slot * a.part_rows + r) * HDG + 4 * ln) = O;
                if (ln == 0) a.part_ml[(size_t)slot * a.part_rows + r] = make_float2(M, L);
            }
        }
        vx_lds_barrier();
        u += cnt;
    }
}

}  // namespace

extern "C" int vx27_hip_paged_attn_q4(vx27_hip_ctx *ctx, const vx27_paged_attn_desc *d) {
    static const char who[] = "vx27_hip_paged_attn_q4";
    VX_REQUIRE(d != nullptr, "%s: null descriptor", who);
    VX_REQUIRE(!d->acc, "%s: acc must be NULL (the rows' weights are added up over bf16 pages only)", who);
    if (vx_q4_fits(who, d->n_pages, d->n_kv, d->page_size)) return -1;
    Args a = {};
    const int todo = attn_fill(who, ctx, d, a);
    if (todo <= 0) return todo;
    const int rows = d->max_T * a.qg;
    // The split kernel reads and decodes a tile for every 16 rows, the tile kernel
    // once for 128.  Tokens of 6 heads, us by the split and by the tile kernel,
    // 4 x 6000 | 1 x 30000 | 32 x 8000 rows: 8 tokens 41, 53 | 44, 95 | 187, 320;
    // 16 tokens 55, 56 | 59, 99 | 349, 323; 24 tokens 73, 66 | 78, 93 | 524, 331.
    // fp32 outputs stay with the split kernel, which rounds neither keys nor
    // values and has two parts of the weights, to where a call is a prompt.
    // Short prompts too, up to 2048 pairs of a tile and a block of 16 rows in all
    // (prompts of 50 tokens 15 us against 26, of 100 18, 28; of 200, 2432 pairs, 28,
    // 31; five of 30 tokens after 270 rows, 2440, 38, 35).  The lengths are on the
    // device, so the pairs are those that the tables have room for.
    const int64_t pairs = ((int64_t)d->n_tok * a.qg / 16 + d->B) * d->n_kv * a.tile_cap;
    if (rows > (a.out_bf16 ? VX27_Q4_SPLIT_ROWS : VX27_Q4_SPLIT_ROWS_F32) && pairs > VX27_Q4_SPLIT_TILES) return rows_launch<true>(who, ctx, d, a, rows, 0);
    // (decoding tokens of 6 heads: 8 rows a block)
    a.block_rows = rows <= 8 ? 8 : 16;
    const int nb = (rows + a.block_rows - 1) / a.block_rows;
    a.min_tiles = 4;                             // (a tile a wave)
    // A list that may be past 2^31 units goes to the tile kernel: those of max_T tokens of every sequence, or, where
    // paged_units adds them up, of n_tok tokens in all.
    const int64_t tiles = ((int64_t)a.tile_cap + a.min_tiles - 1) / a.min_tiles * a.min_tiles * d->n_kv, units = tiles * d->B * nb;
    const bool listed = units < MOST_UNITS || (d->B > 64 && ((int64_t)d->n_tok * a.qg / a.block_rows + d->B) * tiles < MOST_UNITS);
    if (!listed) return rows_launch<true>(who, ctx, d, a, rows, 0);
    const int grid = (int)std::min<int64_t>((units + a.min_tiles - 1) / a.min_tiles, 2 * ctx->n_cu);
    a.part_rows = std::min(rows, a.block_rows);
    const size_t n_part = (size_t)2 * grid * a.part_rows;
    const size_t o_bytes = n_part * HDG * 4, ml_bytes = (n_part * sizeof(float2) + 255) / 256 * 256;
    const size_t before_bytes = d->B > 64 ? ((size_t)d->B + 1) * sizeof(int) : 0;
    void *scr;
    if (vx_ctx_scratch(ctx, o_bytes + ml_bytes + before_bytes, &scr)) return -1;
    a.part_o = (float *)scr;
    a.part_ml = (float2 *)((char *)scr + o_bytes);
    a.before = d->B > 64 ? (int *)((char *)scr + o_bytes + ml_bytes) : nullptr;
    if (a.before && units < MOST_UNITS) VX_LAUNCH_NAMED(ctx, "paged_units", (paged_units<true, false>), dim3(1), dim3(1024), a);
    else if (a.before) VX_LAUNCH_NAMED(ctx, "paged_units", (paged_units<true, true>), dim3(1), dim3(1024), a);
    if (a.block_rows == 16) VX_LAUNCH_NAMED(ctx, "paged_q4_split", (paged_q4_split<16, false>), dim3(grid), dim3(256), a);
    else if (a.out_bf16) VX_LAUNCH_NAMED(ctx, "paged_q4_split", (paged_q4_split<8, true>), dim3(grid), dim3(256), a);
    else VX_LAUNCH_NAMED(ctx, "paged_q4_split", (paged_q4_split<8, false>), dim3(grid), dim3(256), a);
    VX_LAUNCH_NAMED(ctx, "paged_join", (paged_join<true>), dim3(d->n_kv * nb, a.part_rows, d->B), dim3(256), a, grid);
    return 0;
}
