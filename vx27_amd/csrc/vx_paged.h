// Internal interface of the paged KV cache kernels: geometry, what a token
// sees, and the clamps that keep every device-side index inside its buffer.
#pragma once
#include "vx_gqa.h"

constexpr int VX_PG_TILE = VX_GQA_VBLK;   // rows per key tile (a V block): page_size is a multiple

// The pages and sequences of a call.
struct vx_paged {
    int B, n_kv, page_size, n_pages, max_pages;
    int log2_page;               // log2(page_size), or -1 where it is no power of two
    const int *table, *len, *q_start;
    int n_tok, max_T;
    int *err_flag;
};

// One sequence's new tokens and rows; token t's row is row0 + t (negative:
// the token has no row and sees nothing).
struct vx_pseq {
    int start, T, len, row0;
};

// A word of a table that no kernel of the call writes: through the constant
// address space, so that it may be loaded once, early and by the scalar unit
// (the kernels' own stores would otherwise order every use).
__host__ __device__ __forceinline__ int vx_table_word(const int *p) {
#ifdef __HIP_DEVICE_COMPILE__
    return *(const __attribute__((address_space(4))) int *)(uintptr_t)p;
#else
    return *p;
#endif
}

__host__ __device__ __forceinline__ vx_pseq vx_paged_seq(const vx_paged &p, int b) {
    vx_pseq s;
    const int cap = p.max_pages * p.page_size;
    const int n = vx_table_word(p.len + b);
    s.len = min(max(n, 0), cap);
    bool bad = s.len != n;
    if (p.q_start) {
        const int s0 = vx_table_word(p.q_start + b), s1 = vx_table_word(p.q_start + b + 1);
        s.start = min(max(s0, 0), p.n_tok);
        s.T = min(max(s1, s.start), p.n_tok) - s.start;
        bad |= s.start != s0 || s.start + s.T != s1 || s.T > p.max_T;
        s.T = min(s.T, p.max_T);
    } else {
        s.start = b;
        s.T = 1;
    }
    s.row0 = s.len - s.T;
    if (bad) *p.err_flag = 1;
    return s;
}

// Page of row r of sequence b (clamped into the pool and flagged).
__host__ __device__ __forceinline__ int vx_page_checked(const vx_paged &p, int pg) {
    const int c = min(max(pg, 0), p.n_pages - 1);
    if (c != pg) *p.err_flag = 1;
    return c;
}
__host__ __device__ __forceinline__ int vx_page_slot(const vx_paged &p, int r) {
    return p.log2_page >= 0 ? r >> p.log2_page : r / p.page_size;
}
__host__ __device__ __forceinline__ int vx_paged_page(const vx_paged &p, int b, int r) {
    return vx_page_checked(p, vx_table_word(p.table + (size_t)b * p.max_pages + vx_page_slot(p, r)));
}

template <int CTRL, int ROW_MASK>
__device__ __forceinline__ int vx_dpp_i(int x) { return __builtin_amdgcn_update_dpp(0, x, CTRL, ROW_MASK, 0xF, true); }
// Sum over lanes 0 .. l (the VALU's DPP paths: no LDS round trips).
__device__ __forceinline__ int vx_wave_scan(int v) {
    v += vx_dpp_i<0x111, 0xF>(v);   // row_shr:1
    v += vx_dpp_i<0x112, 0xF>(v);
    v += vx_dpp_i<0x114, 0xF>(v);
    v += vx_dpp_i<0x118, 0xF>(v);
    v += vx_dpp_i<0x142, 0xA>(v);   // row_bcast:15 into rows 1 and 3
    v += vx_dpp_i<0x143, 0xC>(v);   // row_bcast:31 into rows 2 and 3
    return v;
}

// The bits of rows key0 .. key0 + 31 that lie below row n.
__host__ __device__ __forceinline__ uint32_t vx_below(int n, int key0) {
    if (n <= key0) return 0u;
    return n - key0 >= 32 ? 0xffffffffu : (1u << (n - key0)) - 1u;
}

// What a token at row i sees: row j <= i if j >= lo (the window's first row)
// or j < sink.  i = -1: nothing.
struct vx_sight {
    int i, lo, sink;
    __host__ __device__ __forceinline__ bool sees(int j) const { return j <= i && (j >= lo || j < sink); }
    // bits of rows key0 .. key0 + 31 (key0 >= 0)
    __host__ __device__ __forceinline__ uint32_t block(int key0) const {
        return vx_below(i + 1, key0) & (~vx_below(lo, key0) | vx_below(sink, key0));
    }
};
__host__ __device__ __forceinline__ vx_sight vx_paged_sight(const vx_pseq &s, int t, int window, int n_sink) {
    vx_sight v;
    v.i = t < s.T ? (s.row0 + t > -1 ? s.row0 + t : -1) : -1;
    v.lo = window ? v.i - window + 1 : 0;
    v.sink = n_sink;
    return v;
}

// The key tiles of which tokens t0 .. t1 of a sequence see a row: tiles
// 0 .. st-1 (sinks that the window has left), then fm, fm+1, ...; nt in all.
struct vx_tiles {
    int st, fm, nt;
    __host__ __device__ __forceinline__ int at(int i) const { return i < st ? i : fm + i - st; }
};
__host__ __device__ __forceinline__ vx_tiles vx_paged_tiles(const vx_pseq &s, int t0, int t1, int window, int n_sink) {
    vx_tiles t = {0, 0, 0};
    const int last = s.row0 + t1;
    if (t1 < t0 || last < 0) return t;
    const int first = s.row0 + t0 > 0 ? s.row0 + t0 : 0;
    const int lo = window && first >= window ? first - window + 1 : 0;
    t.st = ((n_sink < lo ? n_sink : lo) + VX_PG_TILE - 1) / VX_PG_TILE;
    t.fm = lo / VX_PG_TILE;
    if (t.fm <= t.st) t.st = t.fm = 0;
    t.nt = t.st + last / VX_PG_TILE + 1 - t.fm;
    return t;
}

// Host checks shared by the entry points; fills the geometry (not err_flag).
int vx_paged_fill(const char *who, vx_paged &p, int B, int n_kv, int hd, int page_size, int n_pages,
                  int max_pages, const int *table, const int *len);
// The ragged token ranges (q_start may be NULL: one token a sequence).
int vx_paged_tokens(const char *who, vx_paged &p, const int *q_start, int n_tok, int max_T);
