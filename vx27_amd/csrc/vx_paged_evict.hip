// Eviction from a paged KV cache by accumulated attention weight, gfx950.
//
// A sequence past its budget keeps, per KV head, its first n_sink rows, its
// last n_recent rows and the heaviest of the others, ties to the lowest row;
// the kept rows move, in row order, to the pages of another table.
//
//   paged_select  one workgroup per (sequence, KV head): the weight of the
//                 last row kept is found digit by digit (a radix select over
//                 the weights' bits, 8 at a time), then the kept rows are
//                 written in order by prefix sums.
//   paged_move    copies the kept rows' K, V and weights.
#include "vx_paged.h"

namespace {

constexpr int HDG = VX_GQA_HD, VB = VX_GQA_VBLK;

struct EvictArgs {
    vx_paged p;
    int budget, n_sink, n_recent;
    const float *acc;
    size_t acc_stride;
    uint16_t *k_pages, *v_pages;
    const int *dst_table;
    int dst_max_pages;
    int *dst_len;
    float *acc_out;
    size_t acc_out_stride;
    int *kept;          // [B][n_kv][budget] (the caller's or scratch)
};

__device__ __forceinline__ int seq_len(const EvictArgs &a, int b) {
    const int n = a.p.len[b], c = min(max(n, 0), a.p.max_pages * a.p.page_size);
    if (c != n) *a.p.err_flag = 1;
    return c;
}
// Order of a weight as an unsigned number; NaN above everything, -0 as 0.
__device__ __forceinline__ uint32_t rank_of(float w) {
    if (w != w) return 0xffffffffu;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int SEL = 1024;
__global__ __launch_bounds__(SEL) void paged_select(EvictArgs a) {
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = seq_len(a, b), keep = min(n, a.budget);
    int *kept = a.kept + ((size_t)b * a.p.n_kv + h) * a.budget;
    if (h == 0 && tid == 0) a.dst_len[b] = keep;
    if (n <= a.budget) {
        for (int i = tid; i < n; i += SEL) kept[i] = i;
        return;
    }
    const float *w = a.acc + ((size_t)b * a.p.n_kv + h) * a.acc_stride;
    const int lo = a.n_sink, hi = n - a.n_recent;     // the rows that compete
    int want = a.budget - a.n_sink - a.n_recent;      // how many of them stay
    __shared__ int hist[256];
    __shared__ int s_digit, s_want, wsum[SEL / 64], weq[SEL / 64];
    uint32_t prefix = 0, mask = 0;
    for (int shift = 24; shift >= 0 && want > 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        for (int i = lo + tid; i < hi; i += SEL) {
            const uint32_t r = rank_of(w[i]);
            if ((r & mask) == prefix) atomicAdd(&hist[(r >> shift) & 255], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int left = want, dgt = 255;
            while (hist[dgt] < left) left -= hist[dgt--];   // (at least `want` rows match the prefix)
            s_digit = dgt;
            s_want = left;
        }
        __syncthreads();
        prefix |= (uint32_t)s_digit << shift;
        mask |= 0xffu << shift;
        want = s_want;
        __syncthreads();
    }
    // rows above `prefix` stay, and the first `want` equal to it; none where want started at 0
    const bool none = a.budget == a.n_sink + a.n_recent;
    int out = 0, eq_seen = 0;
    for (int i0 = 0; i0 < n; i0 += SEL) {
        const int i = i0 + tid;
        bool forced = false, above = false, eq = false;
        if (i < n) {
            forced = i < lo || i >= hi;
            if (!forced && !none) {
                const uint32_t r = rank_of(w[i]);
                above = r > prefix;
                eq = r == prefix;
            }
        }
        const uint64_t below = lane ? (~0ull >> (64 - lane)) : 0;
        const uint64_t be = __ballot(eq);
        if (lane == 0) weq[wave] = __popcll(be);
        __syncthreads();
        int e = eq_seen + __popcll(be & below), etot = eq_seen;
        for (int k = 0; k < SEL / 64; k++) {
            if (k < wave) e += weq[k];
            etot += weq[k];
        }
        const bool stay = forced || above || (eq && e < want);
        const uint64_t bs = __ballot(stay);
        if (lane == 0) wsum[wave] = __popcll(bs);
        __syncthreads();
        int at = out + __popcll(bs & below), tot = out;
        for (int k = 0; k < SEL / 64; k++) {
            if (k < wave) at += wsum[k];
            tot += wsum[k];
        }
        if (stay) kept[at] = i;
        out = tot;
        eq_seen = etot;
        __syncthreads();
    }
}

// grid (32-row blocks of the destination, n_kv, B), block 256: wave w moves
// K rows w, w + 4, ...; thread d gathers dim d of the block's V rows.
__global__ __launch_bounds__(256) void paged_move(EvictArgs a) {
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int n = seq_len(a, b), keep = min(n, a.budget), d0 = blockIdx.x * VB;
    if (d0 >= keep) return;
    const int cnt = min(VB, keep - d0);
    __shared__ int s_row[VB], s_page[VB];
    const int *kept = a.kept + ((size_t)b * a.p.n_kv + h) * a.budget;
    if (tid < VB) {
        const int r = kept[d0 + min(tid, cnt - 1)];
        s_row[tid] = r;
        s_page[tid] = vx_paged_page(a.p, b, r);
        if (a.acc_out && tid < cnt)
            a.acc_out[((size_t)b * a.p.n_kv + h) * a.acc_out_stride + d0 + tid] = a.acc[((size_t)b * a.p.n_kv + h) * a.acc_stride + r];
    }
    __syncthreads();
    const int P = a.p.page_size;
    const int dpage = vx_page_checked(a.p, a.dst_table[(size_t)b * a.dst_max_pages + d0 / P]), dat = d0 % P;
    for (int j = wave; j < cnt; j += 4) {
        const uint2 u = *(const uint2 *)(a.k_pages + vx_k_index(a.p.n_kv, P, s_page[j], h, s_row[j] % P, 4 * lane));
        *(uint2 *)(a.k_pages + vx_k_index(a.p.n_kv, P, dpage, h, dat + j, 4 * lane)) = u;
    }
    uint16_t v[VB];
#pragma unroll
    for (int j = 0; j < VB; j++) v[j] = a.v_pages[vx_v_index(a.p.n_kv, P, s_page[j], h, s_row[j] % P, tid)];
    uint16_t *dst = a.v_pages + vx_v_index(a.p.n_kv, P, dpage, h, dat, tid);
    if (cnt == VB) {
#pragma unroll
        for (int c = 0; c < 4; c++) {
            uint32_t u[4];
#pragma unroll
            for (int k = 0; k < 4; k++) u[k] = v[8 * c + 2 * k] | ((uint32_t)v[8 * c + 2 * k + 1] << 16);
            *(uint4 *)(dst + 8 * c) = make_uint4(u[0], u[1], u[2], u[3]);
        }
    } else {
#pragma unroll
        for (int j = 0; j < VB; j++)
            if (j < cnt) dst[j] = v[j];
    }
}

bool overlap(const void *x, size_t nx, const void *y, size_t ny) {
    const uintptr_t a = (uintptr_t)x, b = (uintptr_t)y;
    return a < b + ny && b < a + nx;
}

}  // namespace

extern "C" int vx27_hip_paged_evict(vx27_hip_ctx *ctx, const vx27_paged_evict_desc *d) {
    static const char who[] = "vx27_hip_paged_evict";
    VX_REQUIRE(d != nullptr, "%s: null descriptor", who);
    EvictArgs a = {};
    if (vx_paged_fill(who, a.p, d->B, d->n_kv, d->hd, d->page_size, d->n_pages, d->max_pages, d->table, d->len)) return -1;
    const int64_t cap = (int64_t)d->max_pages * d->page_size;
    VX_REQUIRE(d->budget >= 1 && d->n_sink >= 0 && d->n_recent >= 0 && (int64_t)d->n_sink + d->n_recent <= d->budget,
               "%s: need budget >= 1 and 0 <= n_sink + n_recent <= budget (got %d, %d, %d)", who, d->budget, d->n_sink, d->n_recent);
    VX_REQUIRE(d->acc && d->k_pages && d->v_pages && d->dst_table && d->dst_len, "%s: null pointer in descriptor", who);
    VX_REQUIRE((int64_t)d->acc_stride >= cap && (!d->acc_out || d->acc_out_stride >= (size_t)d->budget),
               "%s: need acc_stride >= max_pages * page_size and acc_out_stride >= budget (got %zu, %zu)", who, d->acc_stride, d->acc_out_stride);
    VX_REQUIRE(d->dst_max_pages >= 1 && (int64_t)d->dst_max_pages * d->page_size >= (d->budget < cap ? d->budget : cap),
               "%s: dst_max_pages * page_size must hold the kept rows (got %d * %d for %d)", who, d->dst_max_pages, d->page_size, d->budget);
    VX_REQUIRE((((uintptr_t)d->k_pages | (uintptr_t)d->v_pages) & 15) == 0, "%s: the pages must be 16-byte aligned", who);
    const size_t pairs = (size_t)d->B * d->n_kv;
    VX_REQUIRE(!d->acc_out || !overlap(d->acc, pairs * d->acc_stride * 4, d->acc_out, pairs * d->acc_out_stride * 4),
               "%s: acc_out must not overlap acc", who);
    VX_REQUIRE(!overlap(d->len, (size_t)d->B * 4, d->dst_len, (size_t)d->B * 4), "%s: dst_len must not overlap len", who);
    VX_REQUIRE(!overlap(d->table, (size_t)d->B * d->max_pages * 4, d->dst_len, (size_t)d->B * 4), "%s: dst_len must not overlap table", who);
    if (vx_ctx_enter(ctx)) return -1;
    a.p.err_flag = ctx->err_flag;
    a.budget = d->budget; a.n_sink = d->n_sink; a.n_recent = d->n_recent;
    a.acc = d->acc; a.acc_stride = d->acc_stride; a.k_pages = d->k_pages; a.v_pages = d->v_pages;
    a.dst_table = d->dst_table; a.dst_max_pages = d->dst_max_pages; a.dst_len = d->dst_len;
    a.acc_out = d->acc_out; a.acc_out_stride = d->acc_out_stride;
    a.kept = d->kept;
    if (!a.kept) {
        void *scr;
        if (vx_ctx_scratch(ctx, pairs * d->budget * sizeof(int), &scr)) return -1;
        a.kept = (int *)scr;
    }
    const int64_t most = cap < d->budget ? cap : d->budget;
    VX_LAUNCH(ctx, paged_select, dim3(d->n_kv, d->B), dim3(SEL), a);
    VX_LAUNCH(ctx, paged_move, dim3((unsigned)((most + VB - 1) / VB), d->n_kv, d->B), dim3(256), a);
    return 0;
}
