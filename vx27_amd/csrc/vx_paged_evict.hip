// Eviction from a paged KV cache by accumulated attention weight, gfx950.
//
// A sequence past its budget keeps, per KV head, its first n_sink rows, its
// last n_recent rows and the heaviest of the others, ties to the lowest row;
// the kept rows move, in row order, to the pages of another table.
//
//   paged_select  one workgroup per (sequence, KV head): the weight of the
//                 last row kept is found digit by digit (a radix select over
//                 the weights' bits: 11, 11 and 10), then the kept rows are
//                 written in order by prefix sums.
//   paged_move    copies the kept rows' K, V and weights.
#include "vx_lds.h"
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
    int *kept;          // [B][n_kv][kept_stride] (the caller's or scratch)
    size_t kept_stride;
    int blk0;           // paged_move: first 32-row block of the launch
};

__device__ __forceinline__ int seq_len(const EvictArgs &a, int b) {
    const int n = vx_table_word(a.p.len + b), c = min(max(n, 0), a.p.max_pages * a.p.page_size);
    if (c != n) *a.p.err_flag = 1;
    return c;
}
// Order of a weight as an unsigned number; NaN above every other, -0 as 0.
// Between OUT (no row) and KEPT (a row that stays whatever its weight).
constexpr uint32_t OUT = 0, KEPT = 0xffffffffu;
__device__ __forceinline__ uint32_t rank_of(float w) {
    if (w != w) return KEPT - 1;
    const uint32_t u = __float_as_uint(w + 0.0f);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// how many of a ballot's lanes lie below this one
__device__ __forceinline__ int lanes_below(uint64_t x) { return __builtin_amdgcn_mbcnt_hi((uint32_t)(x >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)x, 0)); }

// Wave w owns rows [w seg, (w+1) seg) and reads them 64 at a time, CH of
// these per chunk; a sequence of up to 16 * 64 * CH rows is one chunk a wave,
// read once and held in registers through all passes.  Sinks and recent rows
// have the highest rank, so that the budget counts them like all others.
// Attention weights are alike in their exponents: 64 lanes at one bin of a
// histogram would be added one by one, so there are eight of it side by side,
// each for every eighth lane (8 x 32768 rows: 35 us, with one histogram 54).
// Two buffers: a pass clears the next one's.  One workgroup a pair has the
// whole of its weights at hand; a launch and three passes' latencies are 12 us.
constexpr int SEL = 1024, NW = SEL / 64, CH = 32, BINS = 2048, COPY = 8, HROW = BINS + 4;   // (copies four banks apart)
__global__ __launch_bounds__(SEL) void paged_select(EvictArgs a) {
    const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = seq_len(a, b), keep = min(n, a.budget);
    int *kept = a.kept + ((size_t)b * a.p.n_kv + h) * a.kept_stride;
    if (h == 0 && tid == 0) a.dst_len[b] = keep;
    if (n <= a.budget) {
        for (int i = tid; i < n; i += SEL) kept[i] = i;
        return;
    }
    const float *w = a.acc + ((size_t)b * a.p.n_kv + h) * a.acc_stride;
    const int lo = a.n_sink, hi = n - a.n_recent;     // the rows that compete
    int want = a.budget;                              // rows of the ranks not yet decided that stay
    __shared__ __attribute__((aligned(16))) int hist[2][COPY][HROW];
    __shared__ int s_sum[NW], s_eq[NW], s_found[2];
    const int seg = ((n + NW - 1) / NW + 63) / 64 * 64, w0 = wave * seg, w1 = min(w0 + seg, n);
    uint32_t r[CH];
    auto load = [&](int base) {
#pragma unroll
        for (int k = 0; k < CH; k++)
            if (base + 64 * k < w1) {   // (uniform)
                const int i = base + 64 * k + lane;
                r[k] = rank_of(w[min(i, n - 1)]);
                if (i < lo || i >= hi) r[k] = KEPT;
                if (i >= w1) r[k] = OUT;
            }
    };
    const bool once = seg <= CH * 64;
    load(w0);
    auto clear = [&](int buf) {
        for (int i = tid; i < COPY * HROW / 4; i += SEL) ((int4 *)hist[buf])[i] = make_int4(0, 0, 0, 0);
    };
    clear(0);
    __syncthreads();
    uint32_t prefix = 0, mask = 0;
#pragma unroll 1
    for (int pass = 0; pass < 3; pass++) {
        const int bits = pass < 2 ? 11 : 10, shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = 1 << bits;
        int (*hp)[HROW] = hist[pass & 1];
        if (pass < 2) clear(~pass & 1);
        for (int base = w0; base < w1; base += CH * 64) {
            if (!once) load(base);
#pragma unroll
            for (int k = 0; k < CH; k++) {
                if (base + 64 * k >= w1) continue;
                if (((r[k] ^ prefix) & mask) == 0) atomicAdd(&hp[lane & (COPY - 1)][(r[k] >> shift) & (bins - 1)], 1);
            }
        }
        __syncthreads();
        // the bin of the want-th heaviest: thread t takes bins 2 t and 2 t + 1
        // (from the top), suffix sums over the threads
        int c[2] = {0, 0};
        const int low = BINS - 2 - 2 * tid;
        if (low < bins) {
#pragma unroll
            for (int q = 0; q < COPY; q++) {
                const int2 x = *(const int2 *)&hp[q][low];
                c[0] += x.y;
                c[1] += x.x;
            }
        }
        const int mine = c[0] + c[1];
        int x = vx_wave_scan(mine);
        if (lane == 63) s_sum[wave] = x;
        __syncthreads();
        const int waves = vx_wave_scan(lane < NW ? s_sum[lane & (NW - 1)] : 0);
        x += (wave ? __builtin_amdgcn_readlane(waves, wave - 1) : 0) - mine;
        if (x < want && x + mine >= want) {   // one thread (more than `want` rows match the prefix)
            const int q = x + c[0] >= want ? 0 : 1;
            s_found[0] = BINS - 1 - (2 * tid + q);
            s_found[1] = want - x - (q ? c[0] : 0);
        }
        __syncthreads();
        prefix |= (uint32_t)s_found[0] << shift;
        mask |= (uint32_t)(bins - 1) << shift;
        want = s_found[1];
    }
    // Rows above `prefix` stay, and the first `want` equal to it: each wave
    // counts its own of both kinds, then writes them behind those of the
    // waves before it.
    int nsure = 0, neq = 0;
    for (int base = w0; base < w1; base += CH * 64) {
        if (!once) load(base);
#pragma unroll
        for (int k = 0; k < CH; k++) {
            if (base + 64 * k >= w1) continue;
            nsure += __popcll(__ballot(r[k] > prefix));
            neq += __popcll(__ballot(r[k] == prefix));
        }
    }
    if (lane == 0) {
        s_sum[wave] = nsure;
        s_eq[wave] = neq;
    }
    __syncthreads();
    const int sures = vx_wave_scan(lane < NW ? s_sum[lane & (NW - 1)] : 0), equals = vx_wave_scan(lane < NW ? s_eq[lane & (NW - 1)] : 0);
    int at = wave ? __builtin_amdgcn_readlane(sures, wave - 1) : 0, eqs = wave ? __builtin_amdgcn_readlane(equals, wave - 1) : 0;
    at += min(eqs, want);
    for (int base = w0; base < w1; base += CH * 64) {
        if (!once) load(base);
#pragma unroll
        for (int k = 0; k < CH; k++) {
            if (base + 64 * k >= w1) continue;
            const uint64_t be = __ballot(r[k] == prefix);
            const bool stay = r[k] > prefix || (r[k] == prefix && eqs + lanes_below(be) < want);
            const uint64_t bs = __ballot(stay);
            // (never past `keep`, whatever a changing acc would count)
            if (stay && at + lanes_below(bs) < keep) kept[at + lanes_below(bs)] = base + 64 * k + lane;
            at += __popcll(bs);
            eqs += __popcll(be);
        }
    }
}

// grid (32-row blocks of the destination from blk0 on, n_kv, B), block 256.  K: wave w
// moves rows w, w + 4, ..., 512 bytes each.  V: a destination block's rows
// come from a few source blocks, each read whole (a kept row has two bytes in
// every 64-byte line of its block) into LDS, dim by dim 68 bytes apart, so
// that thread d's reads of dim d fall on distinct banks.  Bound by bytes: where
// one row in four stays nearly every V block is read: 145 us for 8 ragged
// sequences of up to 32768 rows that keep 8192, up to 940 MB.
constexpr int VROW = VB + 2;   // elements from dim to dim in LDS
__global__ __launch_bounds__(256) void paged_move(EvictArgs a) {
    const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = seq_len(a, b), keep = min(n, a.budget), d0 = (a.blk0 + (int)blockIdx.x) * VB;
    if (d0 >= keep) return;
    const int cnt = min(VB, keep - d0), P = a.p.page_size;
    __shared__ int s_row[VB];
    __shared__ size_t s_blk[VB];   // element offset of the row's V block
    __shared__ uint16_t sv[HDG * VROW];
    const int *kept = a.kept + ((size_t)b * a.p.n_kv + h) * a.kept_stride;
    const int dpage = vx_page_checked(a.p, vx_table_word(a.dst_table + (size_t)b * a.dst_max_pages + d0 / P)), dat = d0 % P;
    if (tid < VB) {
        const int r = min(max(kept[d0 + min(tid, cnt - 1)], 0), n - 1);   // (a row, whatever `kept` shares memory with)
        s_row[tid] = r;
        s_blk[tid] = vx_v_index(a.p.n_kv, P, vx_paged_page(a.p, b, r), h, r % P / VB * VB, 0);
        if (a.acc_out && tid < cnt)
            a.acc_out[((size_t)b * a.p.n_kv + h) * a.acc_out_stride + d0 + tid] = a.acc[((size_t)b * a.p.n_kv + h) * a.acc_stride + r];
    }
    __syncthreads();
    // K rows: all loads, then all stores (a V block is as large as its 32 K
    // rows, so a row's K lies at the same offset)
    uint2 kr[VB / 4];
#pragma unroll
    for (int j = 0; j < VB / 4; j++) {
        const int q = min(wave + 4 * j, cnt - 1);
        kr[j] = *(const uint2 *)(a.k_pages + s_blk[q] + (size_t)(s_row[q] % VB) * HDG + 4 * lane);
    }
    // the first row of each source block's (the rows are in order)
    const int sl = lane & (VB - 1);
    uint32_t starts = (uint32_t)__ballot(sl < cnt && (sl == 0 || s_blk[sl] != s_blk[sl - 1]));
    uint16_t v[VB];
    uint4 u[2][4];
    auto fetch = [&](int j, uint4 (&x)[4]) {
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = *(const uint4 *)(a.v_pages + s_blk[j] + (size_t)(tid + 256 * i) * 8);
    };
    // a source block through LDS, with the next one's loads in flight
    auto take = [&](int buf) {
        const int j = __builtin_ctz(starts);
        starts &= starts - 1;
        const int e = starts ? __builtin_ctz(starts) : cnt;
        if (starts) fetch(e, u[buf ^ 1]);
        if (j) vx_lds_barrier();
#pragma unroll
        for (int i = 0; i < 4; i++) {   // unit tid + 256 i: dim unit / 4, rows 8 (unit % 4) ..
            uint32_t *d = (uint32_t *)&sv[((tid >> 2) + 64 * i) * VROW + (tid & 3) * 8];
            d[0] = u[buf][i].x; d[1] = u[buf][i].y; d[2] = u[buf][i].z; d[3] = u[buf][i].w;
        }
        vx_lds_barrier();
#pragma unroll
        for (int q = 0; q < VB; q++)
            if (q >= j && q < e) v[q] = sv[tid * VROW + s_row[q] % VB];   // (uniform)
    };
    fetch(0, u[0]);
    while (starts) {
        take(0);
        if (starts) take(1);
    }
#pragma unroll
    for (int j = 0; j < VB / 4; j++)
        if (wave + 4 * j < cnt) *(uint2 *)(a.k_pages + vx_k_index(a.p.n_kv, P, dpage, h, dat + wave + 4 * j, 4 * lane)) = kr[j];
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

struct Span {
    const char *name;
    const void *p;
    size_t bytes;
};
bool overlap(const Span &x, const Span &y) {
    const uintptr_t a = (uintptr_t)x.p, b = (uintptr_t)y.p;
    return a < b + y.bytes && b < a + x.bytes;
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
    // what a workgroup of paged_select or paged_move writes must not be what another still reads
    const Span acc = {"acc", d->acc, pairs * d->acc_stride * 4}, len = {"len", d->len, (size_t)d->B * 4},
               table = {"table", d->table, (size_t)d->B * d->max_pages * 4}, dst_table = {"dst_table", d->dst_table, (size_t)d->B * d->dst_max_pages * 4},
               dst_len = {"dst_len", d->dst_len, (size_t)d->B * 4}, kept = {"kept", d->kept, pairs * (size_t)d->budget * 4},
               acc_out = {"acc_out", d->acc_out, pairs * d->acc_out_stride * 4};
    const Span apart[][2] = {{acc_out, acc}, {dst_len, len}, {dst_len, table}, {acc_out, len}, {acc_out, table}, {acc_out, dst_table},
                             {acc_out, dst_len}, {acc_out, kept}, {dst_len, dst_table}, {dst_len, kept}, {dst_len, acc}};
    for (const auto &x : apart)
        VX_REQUIRE(!x[0].p || !x[1].p || !overlap(x[0], x[1]), "%s: %s must not overlap %s", who, x[0].name, x[1].name);
    if (vx_ctx_enter(ctx)) return -1;
    a.p.err_flag = ctx->err_flag;
    a.budget = d->budget; a.n_sink = d->n_sink; a.n_recent = d->n_recent;
    a.acc = d->acc; a.acc_stride = d->acc_stride; a.k_pages = d->k_pages; a.v_pages = d->v_pages;
    a.dst_table = d->dst_table; a.dst_max_pages = d->dst_max_pages; a.dst_len = d->dst_len;
    a.acc_out = d->acc_out; a.acc_out_stride = d->acc_out_stride;
    const int64_t most = cap < d->budget ? cap : d->budget;   // rows a sequence keeps at most
    a.kept = d->kept;
    a.kept_stride = d->budget;
    if (!a.kept) {
        void *scr;
        a.kept_stride = most;
        if (vx_ctx_scratch(ctx, pairs * most * sizeof(int), &scr)) return -1;
        a.kept = (int *)scr;
    }
    VX_LAUNCH(ctx, paged_select, dim3(d->n_kv, d->B), dim3(SEL), a);
    // (a launch holds 2^32 threads a dimension; kept rows past 2^28 take another)
    constexpr int PER = 1 << 23;
    for (int64_t left = (most + VB - 1) / VB; left > 0; left -= PER, a.blk0 += PER)
        VX_LAUNCH(ctx, paged_move, dim3((unsigned)(left < PER ? left : PER), d->n_kv, d->B), dim3(256), a);
    return 0;
}
