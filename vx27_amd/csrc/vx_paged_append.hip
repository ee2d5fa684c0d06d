// Append to a paged KV cache on gfx950: the new tokens' q and k are normed
// and rotated, k and v rounded to bf16 or to 4 bits into their pages, q to bf16
// for the attention.
//
// Per head (vx27_qfwd.c:172-186): s = 1/sqrt(mean(x^2) + 1e-6), y = x s (1+w)
// (or x s w), the first rope_dim dims rotated as NeoX halves by the angle
// (pos / yarn) * freq_i (fp32, as every kernel of this library forms it).
#include "vx_paged_q4.h"

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

// ---------------------------------------------------------- 4-bit pages
// A row's group is 16 lanes of 4 dims.  Values are taken as they are: v's in
// fp32 (REAL float), k's in fp64.  (k carries errors of the norm's sum, the
// angles and the products, and in fp32 these would move a code now and then,
// one value in 10^6, against another order of the sums; in fp64 the codes are
// those of the exact values.)
constexpr float BF16_MAX = 3.38953139e38f;
template <int CTRL>
__device__ __forceinline__ float dpp_f(float x) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xF, 0xF, false)); }
template <int CTRL>
__device__ __forceinline__ double dpp_f(double x) { return vx_dpp_f64<CTRL, 0xF>(x); }
template <bool MAX, typename REAL>
__device__ __forceinline__ REAL over_group(REAL x) {   // maximum or minimum over 16 lanes
    auto pick = [](REAL u, REAL v) { return MAX ? __builtin_elementwise_max(u, v) : __builtin_elementwise_min(u, v); };
    x = pick(x, dpp_f<0xB1>(x));
    x = pick(x, dpp_f<0x4E>(x));
    x = pick(x, dpp_f<0x124>(x));
    return pick(x, dpp_f<0x128>(x));
}
// The largest bf16 number not above x (|x| at most BF16_MAX), as the bits of an
// fp32 number: the truncated bits, or a step on.
__device__ __forceinline__ uint32_t bf16_below(double x) {
    const uint32_t b = __float_as_uint((float)x) & 0xffff0000u;
    if ((double)__uint_as_float(b) <= x) return b;
    return (b & 0x7fffffffu) == 0 ? 0x80010000u : b & 0x80000000u ? b + 0x10000u : b - 0x10000u;
}
// The codes of a lane's four values as bytes, and its group's s and m (bits 16
// to 31 of each).
template <typename REAL>
__device__ __forceinline__ uint32_t quantise(const REAL (&y)[4], uint32_t &s_bits, uint32_t &m_bits) {
    const int lane = threadIdx.x & 63;
    bool fine = true;
#pragma unroll
    for (int e = 0; e < 4; e++) fine &= __builtin_elementwise_abs(y[e]) <= (REAL)BF16_MAX;
    const uint64_t off = __ballot(!fine);
    if ((off >> (lane & 48)) & 0xffff) {
        s_bits = 0;
        m_bits = 0x7fc00000u;
        return 0;
    }
    REAL lo = y[0], hi = y[0];
#pragma unroll
    for (int e = 1; e < 4; e++) lo = __builtin_elementwise_min(lo, y[e]), hi = __builtin_elementwise_max(hi, y[e]);
    m_bits = bf16_below(over_group<false>(lo));
    const double m = __uint_as_float(m_bits);
    // s: the bf16 number just below range / 15 (a last place of the product may
    // be off), and up while 15 s (exact) is below the range
    const double range = (double)over_group<true>(hi) - m;
    uint32_t b = __float_as_uint((float)(range * (1.0 / 15.0))) & 0xffff0000u;
    if (b) b -= 0x10000u;
#pragma unroll
    for (int i = 0; i < 2; i++)
        if ((double)__uint_as_float(b) * 15.0 < range) b += 0x10000u;
    s_bits = b;
    const float s = __uint_as_float(s_bits), rs = __builtin_amdgcn_rcpf(s);
    if (s_bits == 0) return 0;
    // The nearest code.  In fp32 the quotient is 2^-17 off at most (three
    // roundings of 2^-23 and less of it, 15 and less); where that could decide,
    // by what the code leaves in fp64, where it is exact.
    uint32_t codes = 0;
    float far = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float q = (float)(y[e] - (REAL)m) * rs, c = __builtin_rintf(q);
        far = fmaxf(far, __builtin_fabsf(q - c));
        codes |= (uint32_t)c << (8 * e);
    }
    // (a tiny s: fp32 has no reciprocal of it; a range past fp32: the quotient is infinite)
    const bool sure = far < 0.5f - 0x1p-16f && s > 0x1p-100f && range < 0x1p127;
    if (__all(sure)) return codes;
    codes = 0;
    const double rd = 1.0 / (double)s;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const double d = (double)y[e] - m;
        double c = __builtin_rint(d * rd);
        const double r = 2.0 * __builtin_fma(-c, (double)s, d);
        if (__builtin_fabs(r) > (double)s || (__builtin_fabs(r) == (double)s && ((int)c & 1))) c += r > 0.0 ? 1.0 : -1.0;
        codes |= (uint32_t)min(max((int)c, 0), 15) << (8 * e);
    }
    return codes;
}

// 1 / sqrt(x) of a normal x within 2^-50: two of Newton's steps from the
// hardware's 2^-22 (at the ends of fp32's range by the library).
__device__ __forceinline__ double inv_sqrt(double x) {
    if (!(x < 1e30)) return 1.0 / sqrt(x);      // (x is 1e-6 at least, or NaN)
    double r = __builtin_amdgcn_rsqf((float)x);
#pragma unroll
    for (int i = 0; i < 2; i++) r = __builtin_fma(r * 0.5, __builtin_fma(-x * r, r, 1.0), r);
    return r;
}

// One KV head's new keys or values, rows [lo, hi) of the block at row p0 of
// sequence b: a row a wave, its codes into LDS by bytes; then thread u stores
// 16-byte unit u of the block, or of V, where 8 rows share one, as much of it as
// is new.  4362 tokens of 24 + 4 heads (130 MB, 25 us at the copy rate) take 59
// us, keys and values alone 25; with a block's 32 rows in one workgroup, whose
// waves' rows follow one another, 65, and 4 us more for 64 tokens.  Calls timed
// back to back: 53 us, 8192 tokens 95, 65536 672.
constexpr int Q4_ROWS = 8;                    // rows of a workgroup: those that share V's units
constexpr int CODE_ROW = HDG + 4;             // (rows 8 apart then lie in different banks)
template <bool Q4>
constexpr int KV_GROUPS = Q4 ? 2 * VB / Q4_ROWS : 1;
template <int HALFS>                          // codes, the rows' (cos, sin), a row a wave
constexpr int Q4_LDS = Q4_ROWS * CODE_ROW + Q4_ROWS * HALFS * 16 + 4 * HDG * 8;
template <bool V, int HALFS>
__device__ void append_q4_rows(const AppendArgs &a, int hk, int b, int p0, int q0, int lo, int hi, int tok0, char *lds) {
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = hi - lo, half = a.rope_dim / 2;
    const int page = vx_paged_page(a.p, b, p0), at = p0 - vx_page_slot(a.p, p0) * a.p.page_size;
    const size_t block = (size_t)vx_q4_block(a.p, page, hk, at) * VX_Q4_BLOCK;
    char *codes = lds;
    double2 *cs = (double2 *)(lds + Q4_ROWS * CODE_ROW);
    double *row = (double *)(lds + Q4_ROWS * CODE_ROW + Q4_ROWS * HALFS * 16) + wave * HDG;
    char *blk = (char *)(V ? a.v_pages : a.k_pages) + block;
    auto store = [&](int j, const auto &y) {
        const int r = lo - p0 + j;
        uint32_t s, m;
        *(uint32_t *)(codes + r % Q4_ROWS * CODE_ROW + 4 * lane) = quantise(y, s, m);
        if ((lane & 15) == 0) {
            const int c = lane >> 4;
            *(uint16_t *)(blk + VX_Q4_S + c * 64 + r * 2) = (uint16_t)(s >> 16);
            *(uint16_t *)(blk + VX_Q4_M + (V ? c * 64 + r * 2 : r * 8 + c * 2)) = (uint16_t)(m >> 16);
        }
    };
    // (a wave's next row is loaded while it works on one; rows unrolled or four at a time take the registers of the
    // other workgroups' waves)
    auto load_row = [&](int j) { return load4(V ? a.v : a.k, (size_t)(tok0 + min(j, n - 1)) * a.kv_ts + (size_t)hk * HDG + 4 * lane, a.bf16); };
    float4 x = load_row(wave);
    if constexpr (V) {
#pragma unroll 1
        for (int j = wave; j < n; j += 4) {
            const float y[4] = {x.x, x.y, x.z, x.w};
            x = load_row(j + 4);
            store(j, y);
        }
        __syncthreads();
        if (tid < 64) {      // unit (j, rows' eighth, n): dims 64 j + n + 16 i
            const int dim = 64 * (tid >> 4) + (tid & 15);
            uint32_t fresh = 0;                                  // the new rows of the eight
            for (int k = 0; k < Q4_ROWS; k++) fresh |= q0 + k >= lo && q0 + k < hi ? 1u << k : 0u;
            uint4 *dst = (uint4 *)(blk + (64 * (tid >> 4) + 2 * (q0 - p0) + (tid & 15)) * 16);
            uint32_t u[4] = {0, 0, 0, 0}, mask = 0;
#pragma unroll
            for (int k = 0; k < Q4_ROWS; k++) {
                if (!((fresh >> k) & 1)) continue;
                const int at_bit = 8 * (k & 3) + (k & 4);
                mask |= 15u << at_bit;
#pragma unroll
                for (int i = 0; i < 4; i++) u[i] |= (uint32_t)codes[k * CODE_ROW + dim + 16 * i] << at_bit;
            }
            if (fresh != 255) {
                const uint4 old = *dst;
                u[0] |= old.x & ~mask; u[1] |= old.y & ~mask; u[2] |= old.z & ~mask; u[3] |= old.w & ~mask;
            }
            *dst = make_uint4(u[0], u[1], u[2], u[3]);
        }
        return;
    }
    const float4 wf = ((const float4 *)a.k_norm_w)[lane];
    const double one = (a.flags & VX27_GQA_NORM_W) ? 0.0 : 1.0;
    const double w[4] = {wf.x + one, wf.y + one, wf.z + one, wf.w + one};
    for (int e = tid; e < n * half; e += 256) {
        const int j = e / half, i = e % half;
        double sn, c;
        sincos((double)vx_rope_angle(a.rope.freq[i], a.pos ? a.pos[tok0 + j] : lo + j, a.yarn), &sn, &c);
        cs[e] = make_double2(c, sn);
    }
    __syncthreads();
#pragma unroll 1
    for (int j = wave; j < n; j += 4) {
        double y[4] = {x.x, x.y, x.z, x.w};
        x = load_row(j + 4);
        double ss = y[0] * y[0];
#pragma unroll
        for (int e = 1; e < 4; e++) ss = __builtin_fma(y[e], y[e], ss);
        const double sc = inv_sqrt(vx_wave_sum_f64_dpp(ss) * (1.0 / HDG) + 1e-6);
#pragma unroll
        for (int e = 0; e < 4; e++) y[e] = y[e] * sc * w[e];
        if (half) {
            *(double2 *)(row + 4 * lane) = make_double2(y[0], y[1]);
            *(double2 *)(row + 4 * lane + 2) = make_double2(y[2], y[3]);
            __builtin_amdgcn_wave_barrier();   // (one wave's LDS operations complete in order)
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const int i = 4 * lane + e;
                if (i >= 2 * half) continue;
                const bool second = i >= half;
                const double2 c = cs[j * half + (second ? i - half : i)];
                const double z = row[second ? i - half : i + half] * c.y;
                y[e] = y[e] * c.x + (second ? z : -z);
            }
            __builtin_amdgcn_wave_barrier();
        }
        store(j, y);
    }
    __syncthreads();
    // unit (row, k, g): dims 128 k + 8 g + 32 i .. + 7
    const int r = tid >> 3, dim = 128 * ((tid >> 2) & 1) + 8 * (tid & 3);
    if (tid < 8 * Q4_ROWS && q0 + r >= lo && q0 + r < hi) {
        uint32_t u[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t *c = (const uint32_t *)(codes + r * CODE_ROW + dim + 32 * i);
            u[i] = c[0] | (c[1] << 4);
        }
        *(uint4 *)(blk + vx_q4_k_unit(q0 - p0 + r, dim) * 16) = make_uint4(u[0], u[1], u[2], u[3]);
    }
}

// grid (5, or Q4 12, a 32-row block that a sequence's tokens can touch, n_kv, B),
// block 256.  Of a block's workgroups the first takes one KV head's keys and V
// block (Q4: eight, of eight rows' keys or values each), the others the group's
// query heads of 8 tokens each: a prompt's
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
template <int HALFS, bool Q4>
__global__ __launch_bounds__(256) void paged_append(AppendArgs a) {
    constexpr int NR = 4;
    const int hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    constexpr int KV = KV_GROUPS<Q4>;                     // workgroups of a block's keys and values
    const int blk = blockIdx.x / (KV + VB / QTOK), part = blockIdx.x % (KV + VB / QTOK);
    const bool is_k = part < KV;
    if (!is_k && !a.q) return;
    // v's rows; then the tokens' cos and sin, and a row a wave
    constexpr int CS = VB * HALFS * 4;
    constexpr int ROTATE = 2 * CS + 4 * HDG * 4, OTHER = Q4 ? Q4_LDS<HALFS> : VB * HDG * 2;
    __shared__ __attribute__((aligned(16))) char lds[ROTATE > OTHER ? ROTATE : OTHER];
    float (*cs)[HALFS] = (float (*)[HALFS])lds, (*sn)[HALFS] = (float (*)[HALFS])(lds + CS);
    uint16_t (*vt)[HDG] = (uint16_t (*)[HDG])lds;
    const vx_pseq s = vx_paged_seq(a.p, b);
    if (s.row0 < 0 && tid == 0 && hk == 0 && blockIdx.x == 0) *a.p.err_flag = 1;
    const int first = max(s.row0, 0);
    const int p0 = (first / VB + blk) * VB;               // first row of the block
    const int q0 = !is_k ? p0 + QTOK * (part - KV) : Q4 ? p0 + Q4_ROWS * (part >> 1) : p0;    // this workgroup's rows [lo, hi)
    const int lo = max(q0, first), hi = min(q0 + (is_k ? Q4 ? Q4_ROWS : VB : QTOK), s.len);
    if (lo >= hi) return;
    const int n = hi - lo, tok0 = s.start + (lo - s.row0), half = a.rope_dim / 2;
    if constexpr (Q4) {
        if (is_k) {
            if (part & 1) append_q4_rows<true, HALFS>(a, hk, b, p0, q0, lo, hi, tok0, lds);
            else append_q4_rows<false, HALFS>(a, hk, b, p0, q0, lo, hi, tok0, lds);
            return;
        }
    }
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

namespace {

template <bool Q4>
int append(const char *who, vx27_hip_ctx *ctx, const vx27_paged_append_desc *d) {
    VX_REQUIRE(d != nullptr, "%s: null descriptor", who);
    AppendArgs a = {};
    if (vx_paged_fill(who, a.p, d->B, d->n_kv, d->hd, d->page_size, d->n_pages, d->max_pages, d->table, d->len)) return -1;
    if (vx_paged_tokens(who, a.p, d->q_start, d->n_tok, d->max_T)) return -1;
    VX_REQUIRE(d->in_dtype == VX27_F32 || d->in_dtype == VX27_BF16, "%s: in_dtype must be VX27_F32 or VX27_BF16 (got %d)", who, d->in_dtype);
    // (a row's token by a high product: exact where 8 tokens' rows times the group stay below 2^32)
    VX_REQUIRE(!d->q || (d->n_q >= d->n_kv && d->n_q % d->n_kv == 0 && d->n_q / d->n_kv <= 4096),
               "%s: need n_q = k*n_kv with k <= 4096 (n_q=%d n_kv=%d)", who, d->n_q, d->n_kv);
    // (5 workgroups of 256 a 32-row block, or Q4 12: a launch holds 2^32 threads a dimension)
    VX_REQUIRE(d->max_T <= (1 << (Q4 ? 25 : 26)), "%s: max_T is past 2^%d (got %d)", who, Q4 ? 25 : 26, d->max_T);
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
    if (Q4 && vx_q4_fits(who, d->n_pages, d->n_kv, d->page_size)) return -1;
    if (vx_ctx_enter(ctx)) return -1;
    if (d->n_tok == 0) return 0;
    a.p.err_flag = ctx->err_flag;
    a.n_q = d->n_q; a.qg = d->q ? d->n_q / d->n_kv : 1; a.qg_magic = a.qg == 1 ? 0 : (uint32_t)((1ull << 32) / a.qg + 1);
    a.rope_dim = d->rope_dim; a.bf16 = d->in_dtype == VX27_BF16; a.flags = d->flags;
    a.yarn = d->rope_yarn < 1.0f ? 1.0f : d->rope_yarn;
    a.pos = d->pos; a.q = d->q; a.k = d->k_new; a.v = d->v_new;
    a.q_norm_w = d->q_norm_w; a.k_norm_w = d->k_norm_w;
    a.q_out = d->q_out; a.k_pages = d->k_pages; a.v_pages = d->v_pages;
    const dim3 grid(((d->max_T + VB - 2) / VB + 1) * (KV_GROUPS<Q4> + VB / QTOK), d->n_kv, d->B);
    // (32 angles a token take 16 KiB of LDS, 128 take 36: the 143 MB prompt takes 49 us with the first, 62 with the second)
    if (d->rope_dim <= 64) VX_LAUNCH_NAMED(ctx, Q4 ? "paged_append_q4" : "paged_append", (paged_append<32, Q4>), grid, dim3(256), a);
    else VX_LAUNCH_NAMED(ctx, Q4 ? "paged_append_q4" : "paged_append", (paged_append<MAXR, Q4>), grid, dim3(256), a);
    return 0;
}

}  // namespace

extern "C" int vx27_hip_paged_append(vx27_hip_ctx *ctx, const vx27_paged_append_desc *d) {
    return append<false>("vx27_hip_paged_append", ctx, d);
}

extern "C" int vx27_hip_paged_append_q4(vx27_hip_ctx *ctx, const vx27_paged_append_desc *d) {
    return append<true>("vx27_hip_paged_append_q4", ctx, d);
}
