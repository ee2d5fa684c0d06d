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
    int n_q, qg, rope_dim, bf16;
    uint32_t qg_magic;   // floor(2^32 / qg) + 1, 0 for qg = 1
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
// hardware round-to-nearest-even packs (v_cvt_pk_bf16_f32)
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    const bf16x2_t v = (bf16x2_t){(__bf16)x, (__bf16)y};
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ uint2 pack4(float a, float b, float c, float d) { return make_uint2(pack2(a, b), pack2(c, d)); }

// The values of lane l ^ 16 and, within a row of 16 lanes, of another lane.
__device__ __forceinline__ double xor16_f64(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)u, (uint32_t)u, false, false);
    const auto hi = __builtin_amdgcn_permlane16_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
    const bool up = threadIdx.x & 16;
    return __builtin_bit_cast(double, (uint64_t)(up ? hi[0] : hi[1]) << 32 | (up ? lo[0] : lo[1]));
}
// Four sums over the wave at once: the halves of the wave exchange two of
// them, their 16-lane rows one, so that lane l ends with the sum of s[l / 16]
// (with 7 additions and not 24).
__device__ __forceinline__ double wave_sums4(const double (&s)[4]) {
    const bool h = threadIdx.x & 32, q = threadIdx.x & 16;
    const double a = (h ? s[2] : s[0]) + vx_xor32_f64(h ? s[0] : s[2]);
    const double b = (h ? s[3] : s[1]) + vx_xor32_f64(h ? s[1] : s[3]);
    double v = (q ? b : a) + xor16_f64(q ? a : b);
    v += vx_dpp_f64<0xB1, 0xF>(v);    // quad_perm [1,0,3,2]
    v += vx_dpp_f64<0x4E, 0xF>(v);    // quad_perm [2,3,0,1]
    v += vx_dpp_f64<0x124, 0xF>(v);   // row_ror:4
    v += vx_dpp_f64<0x128, 0xF>(v);   // row_ror:8
    return v;
}

// grid (5 a 32-row block that a sequence's tokens can touch, n_kv, B), block
// 256.  Of a block's five workgroups the first takes one KV head's keys and V
// block, the others the group's query heads of 8 tokens each: a prompt's
// workgroups are then short and many (one workgroup a block took 88 us for
// 4364 tokens of 24 + 4 heads, its waves waiting for one another's loads).
// V first, then the tokens' cos and sin in its place in LDS (side by side they
// leave room for six workgroups a CU, not eight: 50 us); then wave w takes
// rows w, w + 4, ..., four at a time so that their loads are in flight
// together, lane l dims 4l..4l+3.
// 49 us for 143 MB (4096 + 268 bf16 tokens; 38 where the last-level cache holds
// the inputs), the copy rate's 27: a wave's loads, norms and stores follow one
// another; one token for 13 sequences, a launch and its latencies, 6.4 us.  v
// goes through LDS into the dim-major block, element by element at its ends
// so that other rows keep their contents.  HALFS: most angles a token has.
constexpr int QTOK = 8;
template <int HALFS>
__global__ __launch_bounds__(256) void paged_append(AppendArgs a) {
    constexpr int NR = 4;
    const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int blk = blockIdx.x / (1 + VB / QTOK), part = blockIdx.x % (1 + VB / QTOK);
    const bool is_k = part == 0;
    if (!is_k && !a.q) return;
    // v's rows; then the tokens' cos and sin, and a row a wave
    constexpr int CS = VB * HALFS * 4;
    __shared__ __attribute__((aligned(16))) char lds[2 * CS + 4 * HDG * 4 > VB * HDG * 2 ? 2 * CS + 4 * HDG * 4 : VB * HDG * 2];
    float (*cs)[HALFS] = (float (*)[HALFS])lds, (*sn)[HALFS] = (float (*)[HALFS])(lds + CS);
    uint16_t (*vt)[HDG] = (uint16_t (*)[HDG])lds;
    const vx_pseq s = vx_paged_seq(a.p, b);
    if (s.row0 < 0 && tid == 0 && hk == 0 && blockIdx.x == 0) *a.p.err_flag = 1;
    const int first = max(s.row0, 0);
    const int p0 = (first / VB + blk) * VB;               // first row of the block
    const int q0 = is_k ? p0 : p0 + QTOK * (part - 1);    // this workgroup's rows [lo, hi)
    const int lo = max(q0, first), hi = min(q0 + (is_k ? VB : QTOK), s.len);
    if (lo >= hi) return;
    const int n = hi - lo, tok0 = s.start + (lo - s.row0), half = a.rope_dim / 2;
    const int per = is_k ? 1 : a.qg, rows = n * per;      // heads of a token
    const uint32_t magic = is_k ? 0 : a.qg_magic;
    const void *src = is_k ? a.k : a.q;
    const size_t ts = is_k ? a.kv_ts : a.q_ts, hs = is_k ? 0 : a.q_hs;
    const size_t base = is_k ? (size_t)hk * HDG : (size_t)hk * a.qg * a.q_hs;
    // row r (past the last: the last again) is head h of token j
    auto tok_of = [&](int r) { return magic ? (int)__umulhi((uint32_t)r, magic) : r; };
    float4 x4[NR];
    auto load_rows = [&](int r0) {
#pragma unroll
        for (int k = 0; k < NR; k++) {
            const int r = min(r0 + 4 * k, rows - 1), j = tok_of(r);
            x4[k] = load4(src, base + (size_t)(tok0 + j) * ts + (size_t)(r - j * per) * hs + 4 * lane, a.bf16);
        }
    };
    load_rows(wave);
    const float4 w4 = ((const float4 *)(is_k ? a.k_norm_w : a.q_norm_w))[lane];
    const float one = (a.flags & VX27_GQA_NORM_W) ? 0.0f : 1.0f;
    const float w[4] = {w4.x + one, w4.y + one, w4.z + one, w4.w + one};
    int page = 0, at = 0;
    if (is_k) {
        page = vx_paged_page(a.p, b, p0);
        at = p0 - vx_page_slot(a.p, p0) * a.p.page_size;
    }
    if (is_k) {
#pragma unroll 4
        for (int e = tid; e < n * (HDG / 4); e += 256) {
            const int j = e / (HDG / 4), c = e % (HDG / 4);
            const float4 x = load4(a.v, (size_t)(tok0 + j) * a.kv_ts + (size_t)hk * HDG + 4 * c, a.bf16);
            *(uint2 *)&vt[j][4 * c] = pack4(x.x, x.y, x.z, x.w);
        }
        __syncthreads();
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
        __syncthreads();
    }
    for (int e = tid; e < n * half; e += 256) {
        const int j = e / half, i = e % half;
        const float2 c = vx_rope_cs(a.rope, a.pos ? a.pos[tok0 + j] : lo + j, a.yarn, i);
        cs[j][i] = c.x;
        sn[j][i] = c.y;
    }
    __syncthreads();

    // half a power of two from 4 on: a pair's dims i and i + half are in lanes
    // l and l ^ (half / 4), at the same element; any other half goes through LDS
    const bool pairs = half >= 4 && (half & (half - 1)) == 0;
    const bool turns = 4 * lane < 2 * half, second = 4 * lane >= half;
    const int ci = pairs ? (4 * lane) & (half - 1) : 0;
    float *row = (float *)(lds + 2 * CS) + wave * HDG;
    for (int r0 = wave; r0 < rows; r0 += 4 * NR) {
        float y[NR][4];
        double ss[NR];
#pragma unroll
        for (int k = 0; k < NR; k++) {
            y[k][0] = x4[k].x; y[k][1] = x4[k].y; y[k][2] = x4[k].z; y[k][3] = x4[k].w;
            ss[k] = (double)y[k][0] * (double)y[k][0];   // (the products are exact)
#pragma unroll
            for (int e = 1; e < 4; e++) ss[k] = __builtin_fma((double)y[k][e], (double)y[k][e], ss[k]);
        }
        if (r0 + 4 * NR < rows) load_rows(r0 + 4 * NR);
        const float sc4 = 1.0f / sqrtf((float)(wave_sums4(ss) / HDG) + 1e-6f);
#pragma unroll
        for (int k = 0; k < NR; k++) {
            const int r = min(r0 + 4 * k, rows - 1), j = tok_of(r);
            const float sc = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(sc4), 16 * k));
#pragma unroll
            for (int e = 0; e < 4; e++) y[k][e] = (y[k][e] * sc) * w[e];
            if (pairs) {
                const float4 c4 = *(const float4 *)&cs[j][ci], s4 = *(const float4 *)&sn[j][ci];
                const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s_[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float z = __shfl_xor(y[k][e], half / 4, 64), zs = z * s_[e];
                    const float t = y[k][e] * c[e] + (second ? zs : -zs);
                    y[k][e] = turns ? t : y[k][e];
                }
            } else if (half) {
                *(float4 *)(row + 4 * lane) = make_float4(y[k][0], y[k][1], y[k][2], y[k][3]);
                __builtin_amdgcn_wave_barrier();   // (one wave's LDS operations complete in order)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int i = 4 * lane + e;
                    if (i < half) y[k][e] = y[k][e] * cs[j][i] - row[i + half] * sn[j][i];
                    else if (i < 2 * half) y[k][e] = row[i - half] * sn[j][i - half] + y[k][e] * cs[j][i - half];
                }
                __builtin_amdgcn_wave_barrier();
            }
            if (r0 + 4 * k < rows) {
                uint16_t *dst = is_k ? a.k_pages + vx_k_index(a.p.n_kv, a.p.page_size, page, hk, at + (lo - p0) + j, 4 * lane)
                                     : a.q_out + ((size_t)(tok0 + j) * a.n_q + hk * per + r - j * per) * HDG + 4 * lane;
                *(uint2 *)dst = pack4(y[k][0], y[k][1], y[k][2], y[k][3]);
            }
        }
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
    // (a row's token by a high product: exact where 8 tokens' rows times the group stay below 2^32)
    VX_REQUIRE(!d->q || (d->n_q >= d->n_kv && d->n_q % d->n_kv == 0 && d->n_q / d->n_kv <= 4096),
               "%s: need n_q = k*n_kv with k <= 4096 (n_q=%d n_kv=%d)", who, d->n_q, d->n_kv);
    // (five workgroups of 256 a 32-row block: a launch holds 2^32 threads a dimension)
    VX_REQUIRE(d->max_T <= (1 << 26), "%s: max_T is past 2^26 (got %d)", who, d->max_T);
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
    a.n_q = d->n_q; a.qg = d->q ? d->n_q / d->n_kv : 1; a.qg_magic = a.qg == 1 ? 0 : (uint32_t)((1ull << 32) / a.qg + 1);
    a.rope_dim = d->rope_dim; a.bf16 = d->in_dtype == VX27_BF16; a.flags = d->flags;
    a.yarn = d->rope_yarn < 1.0f ? 1.0f : d->rope_yarn;
    a.pos = d->pos; a.q = d->q; a.k = d->k_new; a.v = d->v_new;
    a.q_norm_w = d->q_norm_w; a.k_norm_w = d->k_norm_w;
    a.q_out = d->q_out; a.k_pages = d->k_pages; a.v_pages = d->v_pages;
    const dim3 grid(((d->max_T + VB - 2) / VB + 1) * (1 + VB / QTOK), d->n_kv, d->B);
    // (32 angles a token take 16 KiB of LDS, 128 take 36: the 143 MB prompt takes 49 us with the first, 62 with the second)
    if (d->rope_dim <= 64) VX_LAUNCH_NAMED(ctx, "paged_append", (paged_append<32>), grid, dim3(256), a);
    else VX_LAUNCH_NAMED(ctx, "paged_append", (paged_append<MAXR>), grid, dim3(256), a);
    return 0;
}
