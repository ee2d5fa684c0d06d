// Append to a paged KV cache on gfx950: the new tokens' q and k are normed
// and rotated, k and v rounded to bf16 into their pages, q to bf16 for the
// attention.
//
// Per head (vx27_qfwd.c:172-186): s = 1/sqrt(mean(x^2) + 1e-6), y = x s (1+w)
// (or x s w), the first rope_dim dims rotated as NeoX halves by the angle
// (pos / yarn) * freq_i (fp32, as every kernel of this library forms it).
#include "vx_paged.h"

int vx_paged_fill(const char *who, vx_paged &p, int B, int n_kv, int hd, int page_size, int n_pages,
                  int max_pages, const int *table, const int *len) {
    VX_REQUIRE(hd == VX_GQA_HD, "%s: hd must be 256 (got %d)", who, hd);
    VX_REQUIRE(B >= 1 && B <= 65535 && n_kv >= 1 && n_kv <= 1024, "%s: need 1 <= B <= 65535 and 1 <= n_kv <= 1024 (B=%d n_kv=%d)", who,
               B, n_kv);
    VX_REQUIRE(page_size >= VX_PG_TILE && page_size % VX_PG_TILE == 0, "%s: page_size must be a positive multiple of %d (got %d)",
               who, VX_PG_TILE, page_size);
    VX_REQUIRE(n_pages >= 1 && max_pages >= 1, "%s: need n_pages and max_pages >= 1 (got %d, %d)", who, n_pages, max_pages);
    VX_REQUIRE((int64_t)max_pages * page_size <= (1 << 30), "%s: max_pages * page_size is past 2^30 rows (%d * %d)", who,
               max_pages, page_size);
    VX_REQUIRE(table && len, "%s: null page table or lengths", who);
    p.B = B; p.n_kv = n_kv; p.page_size = page_size; p.n_pages = n_pages; p.max_pages = max_pages;
    p.log2_page = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
    p.table = table; p.len = len;
    p.q_start = nullptr; p.n_tok = 0; p.max_T = 0;
    p.err_flag = nullptr;
    return 0;
}

int vx_paged_tokens(const char *who, vx_paged &p, const int *q_start, int n_tok, int max_T) {
    VX_REQUIRE(n_tok >= 0 && max_T >= 0 && max_T <= n_tok, "%s: need 0 <= max_T <= n_tok (max_T=%d n_tok=%d)", who, max_T, n_tok);
    VX_REQUIRE(n_tok == 0 || max_T >= 1, "%s: max_T must be at least 1", who);
    VX_REQUIRE(q_start || (n_tok == p.B && max_T == 1), "%s: q_start may be NULL only for one token a sequence (n_tok=%d B=%d max_T=%d)",
               who, n_tok, p.B, max_T);
    p.q_start = q_start; p.n_tok = n_tok; p.max_T = max_T;
    return 0;
}

namespace {

constexpr int HDG = VX_GQA_HD, VB = VX_GQA_VBLK, MAXR = VX_ROPE_MAXH;

struct AppendArgs {
    vx_paged p;
    int n_q, rope_dim, bf16;
    unsigned flags;
    float yarn;
    const int *pos;
    const void *q, *k, *v;
    size_t q_ts, q_hs, kv_ts;
    const float *q_norm_w, *k_norm_w;
    uint16_t *q_out, *k_pages, *v_pages;
    vx_rope_tab rope;
};

__device__ __forceinline__ float4 load4(const void *base, size_t at, int bf16) {
    if (!bf16) return *(const float4 *)((const float *)base + at);
    const uint2 u = *(const uint2 *)((const uint16_t *)base + at);
    return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                       __uint_as_float(u.y & 0xffff0000u));
}
__device__ __forceinline__ uint2 pack4(float a, float b, float c, float d) {
    return make_uint2((uint32_t)vx_f32_to_bf16(a) | ((uint32_t)vx_f32_to_bf16(b) << 16),
                      (uint32_t)vx_f32_to_bf16(c) | ((uint32_t)vx_f32_to_bf16(d) << 16));
}

// grid (32-row blocks a sequence's tokens can touch, n_kv, B), block 256: one
// workgroup per V block of one KV head, with the query heads of its group.
// The block's cos and sin once; then wave w takes the (token, head) rows w,
// w + 4, ... (query heads, then the key), four at a time so that their loads
// are in flight together, lane l dims 4l..4l+3; v goes through LDS into the
// dim-major block, element by element at its ends so that other rows keep
// their contents.  HALFS: most angles a token has.
template <int HALFS>
__global__ __launch_bounds__(256) void paged_append(AppendArgs a) {
    constexpr int NR = 4;
    const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    __shared__ float2 csn[VB][HALFS];
    __shared__ float row[4][NR][HDG];
    __shared__ __attribute__((aligned(16))) uint16_t vt[VB][HDG];
    const vx_pseq s = vx_paged_seq(a.p, b);
    if (s.row0 < 0 && tid == 0 && hk == 0 && blockIdx.x == 0) *a.p.err_flag = 1;
    const int first = max(s.row0, 0);
    const int p0 = (first / VB + (int)blockIdx.x) * VB;   // first row of the block
    const int lo = max(p0, first), hi = min(p0 + VB, s.len);
    if (lo >= hi) return;
    const int n = hi - lo, tok0 = s.start + (lo - s.row0), half = a.rope_dim / 2;
    const int qg = a.q ? a.n_q / a.p.n_kv : 0, rows = n * (qg + 1);
    const int page = vx_paged_page(a.p, b, p0), at = p0 % a.p.page_size;

    // row r of the block's (token, head) rows; past the last: the last again
    float4 x4[NR];
    auto load_rows = [&](int r0) {
#pragma unroll
        for (int k = 0; k < NR; k++) {
            const int r = min(r0 + 4 * k, rows - 1), j = r / (qg + 1), h = r % (qg + 1);   // h == qg: the key
            const size_t src = h == qg ? (size_t)(tok0 + j) * a.kv_ts + (size_t)hk * HDG
                                       : (size_t)(tok0 + j) * a.q_ts + (size_t)(hk * qg + h) * a.q_hs;
            x4[k] = load4(h == qg ? a.k : a.q, src + 4 * lane, a.bf16);
        }
    };
    load_rows(wave);
    const float4 wk = ((const float4 *)a.k_norm_w)[lane], wq = a.q ? ((const float4 *)a.q_norm_w)[lane] : wk;
    const float one = (a.flags & VX27_GQA_NORM_W) ? 0.0f : 1.0f;
    for (int e = tid; e < n * half; e += 256) {
        const int j = e / half, i = e % half;
        csn[j][i] = vx_rope_cs(a.rope, a.pos ? a.pos[tok0 + j] : lo + j, a.yarn, i);
    }
#pragma unroll 4
    for (int e = tid; e < n * (HDG / 4); e += 256) {
        const int j = e / (HDG / 4), c = e % (HDG / 4);
        const float4 x = load4(a.v, (size_t)(tok0 + j) * a.kv_ts + (size_t)hk * HDG + 4 * c, a.bf16);
        *(uint2 *)&vt[j][4 * c] = pack4(x.x, x.y, x.z, x.w);
    }
    __syncthreads();

    // the V block first: its stores drain while the rows are worked on
    uint16_t *vb = a.v_pages + vx_v_index(a.p.n_kv, a.p.page_size, page, hk, at, 0);
    for (int e = tid; e < HDG * (VB / 8); e += 256) {
        const int d = e / (VB / 8), c = e % (VB / 8), r0 = p0 + 8 * c;
        if (r0 >= lo && r0 + 8 <= hi) {
            uint32_t u[4];
#pragma unroll
            for (int k = 0; k < 4; k++) u[k] = vt[r0 - lo + 2 * k][d] | ((uint32_t)vt[r0 - lo + 2 * k + 1][d] << 16);
            *(uint4 *)(vb + (size_t)d * VB + 8 * c) = make_uint4(u[0], u[1], u[2], u[3]);
        } else {
            for (int k = 0; k < 8; k++)
                if (r0 + k >= lo && r0 + k < hi) vb[(size_t)d * VB + 8 * c + k] = vt[r0 + k - lo][d];
        }
    }

    for (int r0 = wave; r0 < rows; r0 += 4 * NR) {
        float y[NR][4];
        double ss[NR];
#pragma unroll
        for (int k = 0; k < NR; k++) {
            y[k][0] = x4[k].x; y[k][1] = x4[k].y; y[k][2] = x4[k].z; y[k][3] = x4[k].w;
            ss[k] = 0.0;
#pragma unroll
            for (int e = 0; e < 4; e++) ss[k] += (double)y[k][e] * (double)y[k][e];
        }
        if (r0 + 4 * NR < rows) load_rows(r0 + 4 * NR);
#pragma unroll
        for (int k = 0; k < NR; k++) ss[k] = vx_wave_sum_f64_dpp(ss[k]);
#pragma unroll
        for (int k = 0; k < NR; k++) {
            const bool is_k = min(r0 + 4 * k, rows - 1) % (qg + 1) == qg;
            const float w[4] = {is_k ? wk.x : wq.x, is_k ? wk.y : wq.y, is_k ? wk.z : wq.z, is_k ? wk.w : wq.w};
            const float sc = 1.0f / sqrtf((float)(ss[k] / HDG) + 1e-6f);
#pragma unroll
            for (int e = 0; e < 4; e++) y[k][e] = (y[k][e] * sc) * (w[e] + one);
            *(float4 *)&row[wave][k][4 * lane] = make_float4(y[k][0], y[k][1], y[k][2], y[k][3]);
        }
        __builtin_amdgcn_wave_barrier();   // (one wave's LDS operations complete in order)
#pragma unroll
        for (int k = 0; k < NR; k++) {
            const int r = r0 + 4 * k;
            if (r >= rows) break;
            const int j = r / (qg + 1), h = r % (qg + 1);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = 4 * lane + e;
                if (i < half) {
                    const float2 c = csn[j][i];
                    y[k][e] = y[k][e] * c.x - row[wave][k][i + half] * c.y;
                } else if (i < 2 * half) {
                    const float2 c = csn[j][i - half];
                    y[k][e] = row[wave][k][i - half] * c.y + y[k][e] * c.x;
                }
            }
            uint16_t *dst = h == qg ? a.k_pages + vx_k_index(a.p.n_kv, a.p.page_size, page, hk, at + (lo - p0) + j, 4 * lane)
                                    : a.q_out + ((size_t)(tok0 + j) * a.n_q + hk * qg + h) * HDG + 4 * lane;
            *(uint2 *)dst = pack4(y[k][0], y[k][1], y[k][2], y[k][3]);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

}  // namespace

extern "C" int vx27_hip_paged_append(vx27_hip_ctx *ctx, const vx27_paged_append_desc *d) {
    static const char who[] = "vx27_hip_paged_append";
    VX_REQUIRE(d != nullptr, "%s: null descriptor", who);
    AppendArgs a = {};
    if (vx_paged_fill(who, a.p, d->B, d->n_kv, d->hd, d->page_size, d->n_pages, d->max_pages, d->table, d->len)) return -1;
    if (vx_paged_tokens(who, a.p, d->q_start, d->n_tok, d->max_T)) return -1;
    VX_REQUIRE(d->in_dtype == VX27_F32 || d->in_dtype == VX27_BF16, "%s: in_dtype must be VX27_F32 or VX27_BF16 (got %d)", who, d->in_dtype);
    VX_REQUIRE(!d->q || (d->n_q >= d->n_kv && d->n_q % d->n_kv == 0), "%s: need n_q = k*n_kv (n_q=%d n_kv=%d)", who, d->n_q, d->n_kv);
    VX_REQUIRE(d->k_new && d->v_new && d->k_norm_w && d->k_pages && d->v_pages && (!d->q || (d->q_norm_w && d->q_out)),
               "%s: null pointer in descriptor", who);
    if (d->rope_dim != 0) {
        VX_REQUIRE(d->rope_dim >= 2 && d->rope_dim <= HDG && d->rope_dim % 2 == 0, "%s: rope_dim must be even and at most %d (got %d)", who,
                   HDG, d->rope_dim);
        if (vx_rope_fill(a.rope, d->rope_dim, d->rope_theta)) return -1;
    }
    a.q_hs = d->q_head_stride ? d->q_head_stride : HDG;
    a.q_ts = d->q_tok_stride ? d->q_tok_stride : (size_t)d->n_q * HDG;
    a.kv_ts = d->kv_tok_stride ? d->kv_tok_stride : (size_t)d->n_kv * HDG;
    const uintptr_t al = d->in_dtype == VX27_BF16 ? 7 : 15;
    VX_REQUIRE((((uintptr_t)d->q | (uintptr_t)d->k_new | (uintptr_t)d->v_new) & al) == 0 && ((a.q_hs | a.q_ts | a.kv_ts) & 3) == 0,
               "%s: q, k_new and v_new must be %d-byte aligned with strides multiples of 4 elements", who, (int)al + 1);
    VX_REQUIRE((((uintptr_t)d->q_norm_w | (uintptr_t)d->k_norm_w | (uintptr_t)d->q_out | (uintptr_t)d->k_pages | (uintptr_t)d->v_pages) & 15) == 0,
               "%s: q_norm_w, k_norm_w, q_out and the pages must be 16-byte aligned", who);
    if (vx_ctx_enter(ctx)) return -1;
    if (d->n_tok == 0) return 0;
    a.p.err_flag = ctx->err_flag;
    a.n_q = d->n_q; a.rope_dim = d->rope_dim; a.bf16 = d->in_dtype == VX27_BF16; a.flags = d->flags;
    a.yarn = d->rope_yarn < 1.0f ? 1.0f : d->rope_yarn;
    a.pos = d->pos; a.q = d->q; a.k = d->k_new; a.v = d->v_new;
    a.q_norm_w = d->q_norm_w; a.k_norm_w = d->k_norm_w;
    a.q_out = d->q_out; a.k_pages = d->k_pages; a.v_pages = d->v_pages;
    const dim3 grid((d->max_T + VB - 2) / VB + 1, d->n_kv, d->B);
    // (32 angles a token take 8 KiB of LDS, 128 take 32: two workgroups fewer a CU)
    if (d->rope_dim <= 64) VX_LAUNCH_NAMED(ctx, "paged_append", (paged_append<32>), grid, dim3(256), a);
    else VX_LAUNCH_NAMED(ctx, "paged_append", (paged_append<MAXR>), grid, dim3(256), a);
    return 0;
}
