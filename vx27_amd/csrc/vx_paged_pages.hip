// The paged KV cache's pages on gfx950: rows and pages of a step planned on
// the device, and the values of 4-bit rows read by slot.
//
// The plan is prefix sums over the sequences: pages given back, pages wanted
// (which sequences can be served), tokens (which fit the call), and of those
// that remain the pages and tokens before each.  Everything else follows from
// these: token i's sequence is the last with at most i tokens before it, the
// k-th page taken is entry total - 1 - k of the free pages with the released
// ones on top.  Latencies bound it: 13 sequences 4.5 us, a launch and two
// dependent loads (8.7 with a scan each by shuffles, and lengths read again in
// each pass); 2000 sequences with 330000 tokens 18.4 (20.8 with a search a lane).
#include <limits.h>

#include <algorithm>

#include "vx_paged_q4.h"

namespace {

struct PlanArgs {
    int B, page_size, n_pages, max_pages, n_tok, log2_page;
    const int *new_tok, *ended, *len, *next_pos, *n_free;
    int *table, *free_pages;
    int *took, *q_start, *len_out, *next_pos_out, *n_free_out, *slot, *pos, *seq;
    int *err_flag;
    // scratch: pages given back and pages taken before each sequence, and in all (index B); free pages before the call
    int *back, *grown, *was_free;
};

// What the second half of a plan reads: q_start, back and grown, global or in LDS.
struct PlanSums {
    const int *start, *back, *grown;
    int was_free, released, taken;
};

__device__ __forceinline__ int plan_ceil(const PlanArgs &a, int n) {   // pages of n rows
    return a.log2_page >= 0 ? (int)(((uint32_t)n + (uint32_t)a.page_size - 1) >> a.log2_page) : (n + a.page_size - 1) / a.page_size;
}
// The last b in [0, n) with at[b] <= x (at[0] = 0 <= x).
__device__ __forceinline__ int last_le(const int *at, int n, int x) {
    int lo = 0;
    while (n > 1) {
        const int h = n >> 1;
        if (at[lo + h] <= x) lo += h, n -= h;
        else n = h;
    }
    return lo;
}
__device__ __forceinline__ int checked_page(const PlanArgs &a, int pg) {
    const int c = min(max(pg, 0), a.n_pages - 1);
    if (c != pg) *a.err_flag = 1;
    return c;
}
// last_le for every lane of a wave (n entries), whose x do not fall (DOWN: do not
// rise) from lane to lane.
struct LaneFind {            // each by itself: arrays in LDS
    int n;
    template <bool DOWN>
    __device__ __forceinline__ int find(const int *at, int x, bool need) const { return need ? last_le(at, n, x) : 0; }
};
struct WaveFind {            // the least x by all lanes, then on from there
    int n;
    template <bool DOWN>
    __device__ __forceinline__ int find(const int *at, int x, bool need) const {
        const uint64_t who = __ballot(need);
        if (!who) return 0;
        const int lane = threadIdx.x & 63, head = __builtin_ctzll(who), tail = 63 - __builtin_clzll(who);
        const int least = __builtin_amdgcn_readlane(x, DOWN ? tail : head), most = __builtin_amdgcn_readlane(x, DOWN ? head : tail);
        int lo = 0;
        for (int m = n; m > 1;) {
            const int step = (m + 63) / 64, k = 63 - __builtin_clzll(__ballot(lane == 0 || (lane * step < m && at[lo + min(lane * step, m - 1)] <= least)));
            lo += k * step;
            m = min(step, m - k * step);
        }
        const int next = lo + 1 + lane < n ? at[lo + 1 + lane] : INT_MAX;
        int b = lo;
        for (int k = 0; k < 64; k++) {
            const int v = __builtin_amdgcn_readlane(next, k);
            if (v > most) return b;
            b += x >= v;
        }
        return need ? lo + last_le(at + lo, n - lo, x) : 0;   // (more than 64 of them among the lanes' x)
    }
};
// Entry i of the free pages with the released ones on top.
template <bool DOWN, typename FIND>
__device__ __forceinline__ int stack_page(const PlanArgs &a, const PlanSums &p, const FIND &f, int i, bool need) {
    const bool back = need && i >= p.was_free;
    const int j = i - p.was_free, b = f.template find<DOWN>(p.back, j, back);
    if (!need) return 0;
    return checked_page(a, back ? a.table[(size_t)b * a.max_pages + (j - p.back[b])] : a.free_pages[i]);
}
// A plan's second half, for all lanes of a wave: token t's slot, position and
// sequence.  from(b, row0, pos0): row and position of the first token that
// sequence b got.
template <typename FIND, typename FROM>
__device__ __forceinline__ void plan_token(const PlanArgs &a, const PlanSums &p, const FIND &f, FROM from, int t, int tokens) {
    const bool live = t < tokens;
    const int b = f.template find<false>(p.start, t, live);
    int row = 0, pg = 0, pos = -1, taken = 0;
    bool fresh = false;
    if (live) {
        int row0, pos0;
        from(b, row0, pos0);
        const int k = t - p.start[b];
        row = row0 + k;
        pos = (int)((uint32_t)pos0 + (uint32_t)k);
        pg = a.log2_page >= 0 ? row >> a.log2_page : row / a.page_size;
        const int held = plan_ceil(a, row0);
        fresh = pg >= held;
        taken = p.grown[b] + pg - held;
    }
    const int mine = stack_page<true>(a, p, f, p.was_free + p.released - 1 - taken, fresh);
    const int page = fresh ? mine : live ? checked_page(a, a.table[(size_t)b * a.max_pages + pg]) : 0;
    if (t >= a.n_tok) return;
    if (a.slot) a.slot[t] = live ? page * a.page_size + (row - pg * a.page_size) : -1;
    if (a.pos) a.pos[t] = pos;
    if (a.seq) a.seq[t] = live ? b : -1;
}
// Page k of those taken into its table.
template <typename FIND, typename FROM>
__device__ __forceinline__ void plan_taken(const PlanArgs &a, const PlanSums &p, const FIND &f, FROM from, int k) {
    const bool live = k < p.taken;
    const int b = f.template find<false>(p.grown, k, live), page = stack_page<true>(a, p, f, p.was_free + p.released - 1 - k, live);
    if (!live) return;
    int row0, pos0;
    from(b, row0, pos0);
    a.table[(size_t)b * a.max_pages + plan_ceil(a, row0) + k - p.grown[b]] = page;
}
// Released page k, counted from the lowest, onto the free ones: it was not taken.
template <typename FIND>
__device__ __forceinline__ void plan_freed(const PlanArgs &a, const PlanSums &p, const FIND &f, int k) {
    const bool live = k < p.released - p.taken;
    const int page = stack_page<false>(a, p, f, p.was_free + k, live);
    if (live) a.free_pages[p.was_free + k] = page;
}

constexpr int PLAN_THREADS = 1024, PLAN_WAVES = PLAN_THREADS / 64;
template <int CTRL, int ROW_MASK>
__device__ __forceinline__ int64_t add_dpp(int64_t x) {
    const uint64_t u = (uint64_t)x;
    return x + (int64_t)((uint64_t)(uint32_t)vx_dpp_i<CTRL, ROW_MASK>((int)(u >> 32)) << 32 | (uint32_t)vx_dpp_i<CTRL, ROW_MASK>((int)(uint32_t)u));
}
// Sums over lanes 0 .. l.
__device__ __forceinline__ int64_t wave_scan64(int64_t x) {
    x = add_dpp<0x111, 0xF>(x);   // row_shr:1
    x = add_dpp<0x112, 0xF>(x);
    x = add_dpp<0x114, 0xF>(x);
    x = add_dpp<0x118, 0xF>(x);
    x = add_dpp<0x142, 0xA>(x);   // row_bcast:15 into rows 1 and 3
    return add_dpp<0x143, 0xC>(x);   // row_bcast:31 into rows 2 and 3
}
// Sums of v[i] over the threads before this one (into v), and in all.  waves:
// those that have any; sums: [N][PLAN_WAVES], of this call alone.
template <int N>
__device__ __forceinline__ void block_scan(int64_t (&v)[N], int64_t (&all)[N], int64_t *sums, int waves) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t x[N];
#pragma unroll
    for (int i = 0; i < N; i++) {
        x[i] = wave_scan64(v[i]);
        if (lane == 63) sums[i * PLAN_WAVES + wave] = x[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; i++) {
        int64_t before = 0;
        all[i] = 0;
        for (int w = 0; w < waves; w++) {
            const int64_t s = sums[i * PLAN_WAVES + w];
            before += w < wave ? s : 0;
            all[i] += s;
        }
        v[i] = before + x[i] - v[i];
    }
}

// grid 1, block 1024: the sums; ALL (at most 1024 sequences): the rest as well,
// from LDS, in the same launch.
template <bool ALL>
__global__ __launch_bounds__(PLAN_THREADS) void pages_plan(PlanArgs a) {
    __shared__ int64_t sums[5 * PLAN_WAVES];
    constexpr int L = ALL ? PLAN_THREADS + 1 : 1;
    __shared__ int l_start[L], l_back[L], l_grown[L], l_row0[L], l_pos0[L];
    const int tid = threadIdx.x, per = (a.B + PLAN_THREADS - 1) / PLAN_THREADS, waves = min((a.B + per - 1) / per + 63, PLAN_THREADS) / 64;
    const int b0 = min(tid * per, a.B), b1 = min(b0 + per, a.B);
    const int cap = a.max_pages * a.page_size;
    const int free_in = *a.n_free, was_free = min(max(free_in, 0), a.n_pages);
    bool bad = was_free != free_in;
    // a sequence as it comes: rows (0 once it ended), its pages to give back, tokens and pages wanted
    struct Seq {
        int rows, back, want, need;
        bool over;
    };
    auto read = [&](int b) {
        Seq s;
        const int len = a.len[b], n = a.new_tok[b];
        s.over = a.ended && a.ended[b] != 0;
        s.rows = min(max(len, 0), cap);
        s.want = max(n, 0);
        bad |= s.rows != len || s.want != n;
        s.back = s.over ? plan_ceil(a, s.rows) : 0;
        if (s.over) s.rows = s.want = 0;
        if (s.want > cap - s.rows) s.want = 0;
        s.need = plan_ceil(a, s.rows + s.want) - plan_ceil(a, s.rows);
        return s;
    };
    // f(b, sequence b) for a thread's sequences: up to KEPT of them are read once
    constexpr int KEPT = ALL ? 1 : 4;
    Seq kept[KEPT];
    if (per <= KEPT) {
#pragma unroll
        for (int k = 0; k < KEPT; k++)
            if (b0 + k < b1) kept[k] = read(b0 + k);
    }
    auto each = [&](auto f) {
        if (per <= KEPT) {
#pragma unroll
            for (int k = 0; k < KEPT; k++)
                if (b0 + k < b1) f(b0 + k, kept[k]);
        } else {
            for (int b = b0; b < b1; b++) f(b, read(b));
        }
    };
    int64_t first[2] = {0, 0}, all2[2], tok[1] = {0}, all1[1], last[2] = {0, 0}, given[2];
    each([&](int, const Seq &s) {
        first[0] += s.back;
        first[1] += s.need;
    });
    block_scan<2>(first, all2, sums, waves);
    int64_t released = all2[0];
    if (was_free + released > a.n_pages) {   // (pages given back twice, or not of this pool)
        bad = true;
        released = a.n_pages - was_free;
    }
    const int64_t total = was_free + released;
    auto served = [&](int64_t &needs, const Seq &s) {
        needs += s.need;
        return s.need == 0 || needs <= total ? s.want : 0;
    };
    int64_t x = first[1];
    each([&](int, const Seq &s) { tok[0] += served(x, s); });
    block_scan<1>(tok, all1, sums + 2 * PLAN_WAVES, waves);
    auto took_of = [&](int64_t &needs, int64_t &toks, const Seq &s) {
        const int t = served(needs, s);
        toks += t;
        return toks <= a.n_tok ? t : 0;
    };
    int64_t y = tok[0];
    x = first[1];
    each([&](int, const Seq &s) {
        const int t = took_of(x, y, s);
        last[0] += t;
        last[1] += t ? s.need : 0;
    });
    block_scan<2>(last, given, sums + 3 * PLAN_WAVES, waves);
    const int64_t tokens = given[0], taken = given[1];
    y = tok[0];
    x = first[1];
    each([&](int b, const Seq &s) {
        const int t = took_of(x, y, s);
        const int at = (int)last[0], gr = (int)last[1], bk = (int)min(first[0], released);
        const int pos = a.next_pos && !s.over ? a.next_pos[b] : 0;
        if (ALL) l_start[b] = at, l_grown[b] = gr, l_back[b] = bk, l_row0[b] = s.rows, l_pos0[b] = a.next_pos ? pos : s.rows;
        else a.grown[b] = gr, a.back[b] = bk;
        a.q_start[b] = at;
        a.took[b] = t;
        a.len_out[b] = s.rows + t;
        if (a.next_pos) a.next_pos_out[b] = (int)((uint32_t)pos + (uint32_t)t);
        last[0] += t;
        last[1] += t ? s.need : 0;
        first[0] += s.back;
    });
    if (tid == 0) {
        a.q_start[a.B] = (int)tokens;
        if (!ALL) a.was_free[0] = was_free, a.was_free[1] = (int)released, a.was_free[2] = (int)taken;
    }
    if (bad) *a.err_flag = 1;
    __syncthreads();                         // (every thread has read n_free, which n_free_out may be)
    if (tid == 0) *a.n_free_out = (int)(total - taken);
    if constexpr (ALL) {
        const PlanSums p = {l_start, l_back, l_grown, was_free, (int)released, (int)taken};
        const LaneFind f = {a.B};
        auto from = [&](int b, int &row0, int &pos0) { row0 = l_row0[b], pos0 = l_pos0[b]; };
        for (int t = tid; t < a.n_tok; t += PLAN_THREADS) plan_token(a, p, f, from, t, (int)tokens);
        for (int k = tid; k < p.taken; k += PLAN_THREADS) plan_taken(a, p, f, from, k);
        for (int k = tid; k < p.released - p.taken; k += PLAN_THREADS) plan_freed(a, p, f, k);
    }
}

// grid any, block 256: the second half from the sums in memory, 64 items a wave
// at a time.
__global__ __launch_bounds__(256) void pages_fill(PlanArgs a) {
    const PlanSums p = {a.q_start, a.back, a.grown, a.was_free[0], a.was_free[1], a.was_free[2]};
    const WaveFind f = {a.B};
    auto from = [&](int b, int &row0, int &pos0) {
        const int took = a.q_start[b + 1] - a.q_start[b];
        row0 = a.len_out[b] - took;
        pos0 = a.next_pos ? (int)((uint32_t)a.next_pos_out[b] - (uint32_t)took) : row0;
    };
    const int tokens = a.q_start[a.B], lane = threadIdx.x & 63;
    auto groups = [](int n) { return n > 0 ? (n - 1) / 64 + 1 : 0; };
    const int g1 = groups(a.n_tok), g2 = g1 + groups(p.taken), g3 = g2 + groups(p.released - p.taken);
    for (int g = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); g < g3; g += gridDim.x * 4) {
        if (g < g1) plan_token(a, p, f, from, 64 * g + lane, tokens);
        else if (g < g2) plan_taken(a, p, f, from, 64 * (g - g1) + lane);
        else plan_freed(a, p, f, 64 * (g - g2) + lane);
    }
}

// ------------------------------------------------------------------- read
struct ReadArgs {
    int n_kv, page_size, n_pages, n_rows, bf16, log2_page;
    const int *slots;
    const char *k_pages, *v_pages;
    void *k_out, *v_out;
    int *err_flag;
};
__device__ __forceinline__ uint32_t bf16x2(float x, float y) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    const bf16x2_t v = (bf16x2_t){(__bf16)x, (__bf16)y};
    return __builtin_bit_cast(uint32_t, v);
}

// Of 4 lanes that have 4 words each, lane t gets the words t of all, in order.
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
    const uint32_t t = threadIdx.x & 3;
    uint32_t x[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t y = (uint32_t)vx_dpp_i<0xB1, 0xF>((int)w[i ^ 1]);   // of lane ^ 1 (all lanes take part)
        x[i] = (t ^ i) & 1 ? y : w[i];
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t y = (uint32_t)vx_dpp_i<0x4E, 0xF>((int)x[i ^ 2]);   // of lane ^ 2
        w[i] = (t ^ i) & 2 ? y : x[i];
    }
}
__device__ __forceinline__ void put_values(const ReadArgs &a, void *out, size_t at, const float (&x)[4]) {
    if (a.bf16) *(uint2 *)((uint16_t *)out + at) = make_uint2(bf16x2(x[0], x[1]), bf16x2(x[2], x[3]));
    else *(float4 *)((float *)out + at) = make_float4(x[0], x[1], x[2], x[3]);
}

// 8 rows of K or of V a wave, whose loads are in flight together (the slots'
// checks and the conversions come behind them: between the loads they made each
// row wait for its own).  Eight rows of a block that share V's units, as a
// sequence read in order has them, are one load of codes and up to three of s
// and m; any other rows three loads each.  (Loads and stores, 16 cycles each,
// bound the second form.)  32768 rows of 4 heads in order 37 us in bf16 (the
// copy rate: 33) and 79 in fp32, in random order 56; 77 rows 3.2.
constexpr int READ_ROWS = 8;
template <bool V>
__device__ __forceinline__ void read_rows(const ReadArgs &a, int i0, int h, const char *pages, void *out) {
    const int lane = threadIdx.x & 63, g = lane >> 4;
    const int mine = a.slots[min(i0 + min(lane, READ_ROWS - 1), a.n_rows - 1)];
    const bool in = mine >= 0 && mine < a.n_pages * a.page_size;
    const int place = in ? mine : 0;
    const int page = a.log2_page >= 0 ? place >> a.log2_page : place / a.page_size, at = place - page * a.page_size;
    const int block = (int)(((uint32_t)page * (uint32_t)a.n_kv + (uint32_t)h) * (uint32_t)(a.page_size / VX_PG_TILE) + (uint32_t)(at / VX_PG_TILE));
    auto block_of = [&](int k) { return pages + (size_t)(uint32_t)__builtin_amdgcn_readlane(block, k) * VX_Q4_BLOCK; };
    auto row_of = [&](int k) { return __builtin_amdgcn_readlane(at, k) % VX_PG_TILE; };
    auto out_at = [&](int k) { return ((size_t)(i0 + k) * a.n_kv + h) * VX_GQA_HD; };
    const int first = __builtin_amdgcn_readfirstlane(mine);
    if (first >= 0 && first % READ_ROWS == 0 && i0 + READ_ROWS <= a.n_rows && __all(in && mine == first + min(lane, READ_ROWS - 1))) {
        const char *blk = block_of(0);
        const int r0 = row_of(0);
        if constexpr (V) {   // lane (j,n): a unit, dims 64 j + 16 i + n of the 8 rows; then dims 64 j + 16 (n % 4) + 4 (n / 4) + e
            const int n = lane & 15;
            const uint4 c = *(const uint4 *)(blk + (64 * g + 2 * r0 + n) * 16);
            const uint4 s4 = *(const uint4 *)(blk + VX_Q4_S + g * 64 + r0 * 2), m4 = *(const uint4 *)(blk + VX_Q4_M + g * 64 + r0 * 2);
            float s[8], m[8];
            vx_q4_f32(s4, s);
            vx_q4_f32(m4, m);
            uint32_t w[4] = {c.x, c.y, c.z, c.w};
            transpose4(w);
#pragma unroll
            for (int k = 0; k < READ_ROWS; k++) {
                float x[4];
#pragma unroll
                for (int e = 0; e < 4; e++) x[e] = __builtin_fmaf((float)((w[e] >> (8 * (k & 3) + (k & 4))) & 15), s[k], m[k]);
                put_values(a, out, out_at(k) + 64 * g + 16 * (n & 3) + 4 * (n >> 2), x);
            }
        } else {             // lane (half, k, g, r): a unit, dims 128 k + 32 i + 8 g .. + 7 of row 4 half + r
            const int kh = (lane >> 4) & 1, gd = (lane >> 2) & 3, r = 4 * (lane >> 5) + (lane & 3);
            const uint4 c = *(const uint4 *)(blk + vx_q4_k_unit(r0 + r, 128 * kh + 8 * gd) * 16);
            const uint32_t m2 = *(const uint32_t *)(blk + VX_Q4_M + (r0 + r) * 8 + kh * 4);
            uint16_t s2[2];
#pragma unroll
            for (int e = 0; e < 2; e++) s2[e] = *(const uint16_t *)(blk + VX_Q4_S + (2 * kh + e) * 64 + (r0 + r) * 2);
            const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float s = vx_bf16_to_f32(s2[i >> 1]), m = __uint_as_float(i >> 1 ? m2 & 0xffff0000u : m2 << 16);
                const size_t o = out_at(r) + 128 * kh + 32 * i;
                if (a.bf16) {
                    float x[8];
                    vx_q4_codes_f32(w[i], x);
#pragma unroll
                    for (int e = 0; e < 8; e++) x[e] = __builtin_fmaf(x[e], s, m);
                    *(uint4 *)((uint16_t *)out + o + 8 * gd) = make_uint4(bf16x2(x[0], x[1]), bf16x2(x[2], x[3]), bf16x2(x[4], x[5]), bf16x2(x[6], x[7]));
                    continue;
                }
                // fp32: four lanes' 16 bytes side by side, dims 4 gd .. + 3 of 16 (32 bytes a lane: 8192 rows 19.9 us, so 17.7)
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const uint32_t y = (uint32_t)__shfl((int)w[i], (lane & ~12) + 8 * t + 4 * (gd >> 1), 64), z = (gd & 1 ? y >> 4 : y) & 0x0f0f0f0fu;
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] = __builtin_fmaf((float)((z >> (8 * e)) & 255), s, m);
                    put_values(a, out, o + 16 * t + 4 * gd, x);
                }
            }
        }
        return;
    }
    // row by row: lane L has dims 4L .. 4L + 3 of K, and of V as above
    const uint32_t c_at = V ? g * 1024 + (lane & 15) * 16 : vx_q4_k_unit(0, 4 * lane) * 16 + ((lane >> 3) & 3) * 4;
    const uint32_t s_at = VX_Q4_S + g * 64, m_at = VX_Q4_M + g * (V ? 64 : 2);
    uint32_t c[READ_ROWS][V ? 4 : 1];
    uint16_t s[READ_ROWS], m[READ_ROWS];
#pragma unroll
    for (int k = 0; k < READ_ROWS; k++) {
        const int r = row_of(k);
        const char *blk = block_of(k), *codes = blk + (V ? (r >> 3) * 256 : vx_q4_k_unit(r, 0) * 16);
        if constexpr (V) {
            const uint4 x = *(const uint4 *)(codes + c_at);
            c[k][0] = x.x; c[k][1] = x.y; c[k][2] = x.z; c[k][3] = x.w;
        } else {
            c[k][0] = *(const uint32_t *)(codes + c_at);
        }
        s[k] = *(const uint16_t *)(blk + r * 2 + s_at);
        m[k] = *(const uint16_t *)(blk + r * (V ? 2 : 8) + m_at);
    }
    if (!in && mine != -1) *a.err_flag = 1;
    const uint64_t live = __ballot(in);
#pragma unroll
    for (int k = 0; k < READ_ROWS; k++) {
        if (i0 + k >= a.n_rows) return;
        if (!((live >> k) & 1)) continue;
        const int r = row_of(k);
        const float sc = vx_bf16_to_f32(s[k]), mn = vx_bf16_to_f32(m[k]);
        float x[4];
        size_t o = out_at(k);
        if constexpr (V) {
            const int shift = 8 * (r & 3) + (r & 4);
            transpose4(c[k]);
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = __builtin_fmaf((float)((c[k][e] >> shift) & 15), sc, mn);
            o += 64 * g + 16 * (lane & 3) + 4 * ((lane >> 2) & 3);
        } else {
            const uint32_t w = (lane & 1 ? c[k][0] >> 4 : c[k][0]) & 0x0f0f0f0fu;
#pragma unroll
            for (int e = 0; e < 4; e++) x[e] = __builtin_fmaf((float)((w >> (8 * e)) & 255), sc, mn);
            o += 4 * lane;
        }
        put_values(a, out, o, x);
    }
}

// grid (n_rows / (4 READ_ROWS), n_kv, 2), block 256: z 0 reads K, 1 V.
__global__ __launch_bounds__(256) void paged_read_q4(ReadArgs a) {
    const int i0 = (blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6)) * READ_ROWS;
    if (i0 >= a.n_rows) return;
    if (blockIdx.z == 0) {
        if (a.k_out) read_rows<false>(a, i0, blockIdx.y, a.k_pages, a.k_out);
    } else {
        if (a.v_out) read_rows<true>(a, i0, blockIdx.y, a.v_pages, a.v_out);
    }
}

}  // namespace

extern "C" int vx27_hip_paged_plan(vx27_hip_ctx *ctx, const vx27_paged_plan_desc *d) {
    static const char who[] = "vx27_hip_paged_plan";
    VX_REQUIRE(d != nullptr, "%s: null descriptor", who);
    VX_REQUIRE(d->B >= 1 && d->B <= 65535, "%s: need 1 <= B <= 65535 (B=%d)", who, d->B);
    VX_REQUIRE(d->page_size >= VX_PG_TILE && d->page_size % VX_PG_TILE == 0, "%s: page_size must be a positive multiple of %d (got %d)",
               who, VX_PG_TILE, d->page_size);
    VX_REQUIRE(d->n_pages >= 1 && d->max_pages >= 1 && d->n_tok >= 0, "%s: need n_pages and max_pages >= 1 and n_tok >= 0 (got %d, %d, %d)", who,
               d->n_pages, d->max_pages, d->n_tok);
    VX_REQUIRE((int64_t)d->max_pages * d->page_size <= (1 << 30), "%s: max_pages * page_size is past 2^30 rows (%d * %d)", who,
               d->max_pages, d->page_size);
    VX_REQUIRE((int64_t)d->n_pages * d->page_size < (1ll << 31), "%s: n_pages * page_size is past 2^31 rows (%d * %d)", who, d->n_pages,
               d->page_size);
    VX_REQUIRE(d->new_tok && d->len && d->table && d->free_pages && d->n_free && d->took && d->q_start && d->len_out && d->n_free_out,
               "%s: null pointer in descriptor", who);
    VX_REQUIRE(!d->next_pos == !d->next_pos_out, "%s: next_pos and next_pos_out go together", who);
    // Tokens and pages are looked up in what the call writes: an output may be
    // its input's own array, and overlap nothing else.
    struct Span {
        const char *name;
        const void *p;
        size_t bytes;
        int in_place;   // index of the input that it may be
    };
    const size_t nb = (size_t)d->B * 4, nt = (size_t)d->n_tok * 4;
    const Span in[] = {{"new_tok", d->new_tok, nb, 0}, {"ended", d->ended, nb, 0}, {"len", d->len, nb, 0}, {"next_pos", d->next_pos, nb, 0},
                       {"n_free", d->n_free, 4, 0}};
    const Span out[] = {{"len_out", d->len_out, nb, 2}, {"next_pos_out", d->next_pos_out, nb, 3}, {"n_free_out", d->n_free_out, 4, 4},
                        {"took", d->took, nb, -1}, {"q_start", d->q_start, nb + 4, -1}, {"table", d->table, nb * d->max_pages, -1},
                        {"free_pages", d->free_pages, (size_t)d->n_pages * 4, -1}, {"slot", d->slot, nt, -1}, {"pos", d->pos, nt, -1},
                        {"seq", d->seq, nt, -1}};
    auto apart = [](const Span &x, const Span &y) {
        const uintptr_t a0 = (uintptr_t)x.p, b0 = (uintptr_t)y.p;
        return !x.p || !y.p || !x.bytes || !y.bytes || a0 + x.bytes <= b0 || b0 + y.bytes <= a0;
    };
    for (int i = 0; i < 10; i++) {
        for (int j = 0; j < 5; j++)
            VX_REQUIRE(apart(out[i], in[j]) || (out[i].in_place == j && out[i].p == in[j].p), "%s: %s must not overlap %s", who, out[i].name, in[j].name);
        for (int j = 0; j < i; j++) VX_REQUIRE(apart(out[i], out[j]), "%s: %s must not overlap %s", who, out[i].name, out[j].name);
    }
    if (vx_ctx_enter(ctx)) return -1;
    PlanArgs a = {};
    a.B = d->B; a.page_size = d->page_size; a.n_pages = d->n_pages; a.max_pages = d->max_pages; a.n_tok = d->n_tok;
    a.log2_page = (d->page_size & (d->page_size - 1)) == 0 ? __builtin_ctz(d->page_size) : -1;
    a.new_tok = d->new_tok; a.ended = d->ended; a.len = d->len; a.next_pos = d->next_pos; a.n_free = d->n_free;
    a.table = d->table; a.free_pages = d->free_pages; a.took = d->took; a.q_start = d->q_start; a.len_out = d->len_out;
    a.next_pos_out = d->next_pos_out; a.n_free_out = d->n_free_out; a.slot = d->slot; a.pos = d->pos; a.seq = d->seq;
    a.err_flag = ctx->err_flag;
    if (d->B <= PLAN_THREADS && d->n_tok <= 4 * PLAN_THREADS) {
        VX_LAUNCH_NAMED(ctx, "pages_plan", (pages_plan<true>), dim3(1), dim3(PLAN_THREADS), a);
        return 0;
    }
    void *scr;
    if (vx_ctx_scratch(ctx, ((size_t)2 * d->B + 3) * sizeof(int), &scr)) return -1;
    a.back = (int *)scr; a.grown = a.back + d->B; a.was_free = a.grown + d->B;
    VX_LAUNCH_NAMED(ctx, "pages_plan", (pages_plan<false>), dim3(1), dim3(PLAN_THREADS), a);
    const int64_t most = (int64_t)d->n_tok + d->n_pages;
    VX_LAUNCH(ctx, pages_fill, dim3((unsigned)std::min<int64_t>((most + 255) / 256, 8 * ctx->n_cu)), dim3(256), a);
    return 0;
}

extern "C" int vx27_hip_paged_read_q4(vx27_hip_ctx *ctx, const vx27_paged_read_desc *d) {
    static const char who[] = "vx27_hip_paged_read_q4";
    VX_REQUIRE(d != nullptr, "%s: null descriptor", who);
    VX_REQUIRE(d->hd == VX_GQA_HD, "%s: hd must be 256 (got %d)", who, d->hd);
    VX_REQUIRE(d->n_kv >= 1 && d->n_kv <= 1024, "%s: need 1 <= n_kv <= 1024 (n_kv=%d)", who, d->n_kv);
    VX_REQUIRE(d->page_size >= VX_PG_TILE && d->page_size % VX_PG_TILE == 0, "%s: page_size must be a positive multiple of %d (got %d)",
               who, VX_PG_TILE, d->page_size);
    VX_REQUIRE(d->n_pages >= 1 && (int64_t)d->n_pages * d->page_size < (1ll << 31), "%s: need n_pages >= 1 and n_pages * page_size below 2^31 (%d * %d)",
               who, d->n_pages, d->page_size);
    if (vx_q4_fits(who, d->n_pages, d->n_kv, d->page_size)) return -1;
    VX_REQUIRE(d->n_rows >= 0 && d->n_rows <= (1 << 25), "%s: need 0 <= n_rows <= 2^25 (got %d)", who, d->n_rows);
    VX_REQUIRE(d->out_dtype == VX27_F32 || d->out_dtype == VX27_BF16, "%s: out_dtype must be VX27_F32 or VX27_BF16 (got %d)", who, d->out_dtype);
    VX_REQUIRE(d->slots && (d->k_pages || !d->k_out) && (d->v_pages || !d->v_out), "%s: null pointer in descriptor", who);
    VX_REQUIRE((((uintptr_t)d->k_pages | (uintptr_t)d->v_pages | (uintptr_t)d->k_out | (uintptr_t)d->v_out) & 15) == 0,
               "%s: pages and outputs must be 16-byte aligned", who);
    if (vx_ctx_enter(ctx)) return -1;
    if (d->n_rows == 0 || (!d->k_out && !d->v_out)) return 0;
    const ReadArgs a = {d->n_kv, d->page_size, d->n_pages, d->n_rows, d->out_dtype == VX27_BF16,
                        (d->page_size & (d->page_size - 1)) == 0 ? __builtin_ctz(d->page_size) : -1, d->slots,
                        (const char *)d->k_pages, (const char *)d->v_pages, d->k_out, d->v_out, ctx->err_flag};
    VX_LAUNCH(ctx, paged_read_q4, dim3((d->n_rows + 4 * READ_ROWS - 1) / (4 * READ_ROWS), d->n_kv, 2), dim3(256), a);
    return 0;
}
