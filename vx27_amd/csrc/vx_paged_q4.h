// The 4-bit pages of the paged KV cache: layout and decoding.
//
// A block is 32 rows of K or of V of one KV head.  A row's 256 dims are four
// groups of 64; dim d of row r is m + s c, with s and m of (r, d / 64) in bf16
// and c in 0..15.  (m is the largest bf16 number not above the group's values
// and s rounded up, so that all codes fit; s and m cost 1/8 of the codes'
// bytes.  Groups of 32 dims would halve the largest group's error at 9% more
// bytes.)
//
// The codes lie in the order in which a wave's MFMA operands take them: 16
// bytes a lane are four operands of 8 codes.  Of an operand's dword, byte i
// holds code i in its low and code i + 4 in its high half, so that two masks
// give two words of four codes each, and a code's byte is the e4m3 number
// c 2^-9 as it stands: v_cvt_scalef32_pk_bf16_fp8 with a scale of 2^9 makes
// two exact bf16 codes of it.
#pragma once
#include "vx_paged.h"

constexpr int VX_Q4_BLOCK = VX27_Q4_BLOCK_BYTES;    // codes, then s, then m
constexpr int VX_Q4_S = 4096, VX_Q4_M = VX_Q4_S + 256;
constexpr int VX_Q4_GROUP = 64;

// Number of the block that holds row `at` (a multiple of 32) of page `page`,
// KV head h: fits 32 bits where the pool's rows times n_kv do.
__host__ __device__ __forceinline__ uint32_t vx_q4_block(const vx_paged &p, int page, int h, int at) {
    return ((uint32_t)page * (uint32_t)p.n_kv + (uint32_t)h) * (uint32_t)(p.page_size / VX_PG_TILE) + (uint32_t)(at / VX_PG_TILE);
}

// Host check of the pool's size.
inline int vx_q4_fits(const char *who, int n_pages, int n_kv, int page_size) {
    VX_REQUIRE((int64_t)n_pages * n_kv * (page_size / VX_PG_TILE) < (1ll << 32), "%s: more than 2^32 blocks (n_pages=%d n_kv=%d page_size=%d)",
               who, n_pages, n_kv, page_size);
    return 0;
}

// Codes of K: unit u = lane (g,n) of operand quad 2 r + k; its dword i holds
// dims 128 k + 32 i + 8 g .. + 7 of row 8 (n/4) + 4 r + n%4.
__host__ __device__ __forceinline__ int vx_q4_k_unit(int row, int dim) {
    return ((row >> 2) & 1) * 128 + (dim >> 7) * 64 + ((dim >> 3) & 3) * 16 + (row >> 3) * 4 + (row & 3);
}
__host__ __device__ __forceinline__ int vx_q4_k_row(int u) { return ((u >> 2) & 3) * 8 + (u >> 7) * 4 + (u & 3); }
// Codes of V: unit u = lane (g,n) of quad j; its dword i holds dim
// 64 j + 16 i + n of rows 8 g .. 8 g + 7.
// Scales s: [4 groups][32 rows].  Minima m: K [32 rows][4 groups], V [4][32].
// One value of a block of V.
__device__ __forceinline__ float vx_q4_v_value(const char *blk, int row, int dim) {
    const int group = dim / VX_Q4_GROUP;
    const uint32_t c = (uint8_t)blk[group * 1024 + (row >> 3) * 256 + (dim & 15) * 16 + ((dim >> 4) & 3) * 4 + (row & 3)] >> (row & 4);
    auto word = [&](int at) { return vx_bf16_to_f32(*(const uint16_t *)(blk + at + group * 64 + row * 2)); };
    return __builtin_fmaf((float)(c & 15), word(VX_Q4_S), word(VX_Q4_M));
}

typedef __bf16 vx_bf16x8 __attribute__((ext_vector_type(8)));

// Eight codes as bf16 numbers.
__device__ __forceinline__ vx_bf16x8 vx_q4_codes(uint32_t w) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 512.0f, true);
    const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 512.0f, true);
    vx_bf16x8 x;
    x[0] = a[0]; x[1] = a[1]; x[2] = b[0]; x[3] = b[1];
    x[4] = c[0]; x[5] = c[1]; x[6] = d[0]; x[7] = d[1];
    return x;
}
// The same as fp32.
__device__ __forceinline__ void vx_q4_codes_f32(uint32_t w, float (&x)[8]) {
    typedef float floatx2 __attribute__((ext_vector_type(2)));
    const uint32_t lo = w & 0x0f0f0f0fu, hi = (w >> 4) & 0x0f0f0f0fu;
    const floatx2 y[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp8(lo, 512.0f, false), __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(lo, 512.0f, true),
                          __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, 512.0f, false), __builtin_amdgcn_cvt_scalef32_pk_f32_fp8(hi, 512.0f, true)};
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = y[e >> 1][e & 1];
}
// Eight bf16 numbers of 16 bytes.
__device__ __forceinline__ void vx_q4_f32(uint4 w, float (&x)[8]) {
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int k = 0; k < 4; k++) {
        x[2 * k] = __uint_as_float(u[k] << 16);
        x[2 * k + 1] = __uint_as_float(u[k] & 0xffff0000u);
    }
}
