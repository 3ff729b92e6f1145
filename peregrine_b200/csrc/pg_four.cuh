// Numbers of 4 bits with a scale per group: what the products with such weights and the attention over such caches share.
//
// A group's scale is bf16(v / -8), v the value of largest magnitude (the first of equals), and a value w is held as
// q = clamp(rint(w / scale) + 8, 0, 15), standing for scale * (q - 8).  A group with a value that is not finite has the scale
// not-a-number, so that whatever reads it says so too.
#pragma once

#include <cuda_fp16.h>

#include "pg_lm.cuh"

struct pg_linear4 {
    void *mem = nullptr;
    const unsigned char *w = nullptr;   // [experts][tiles][K / 64][record]: 16 rows x 64 k, quants and scales (csrc/pg_linear4.cu)
    const float *row = nullptr;         // [experts][tiles * 16]: 2^row
    int64_t n = 0, k = 0, experts = 1, group = 0, tiles = 0, record = 0, bytes = 0;
    int device = 0;
};

// bytes of 16 positions of a head's keys or values in 4 bits: 8 per column, and 32 of scales per 32 columns (width a multiple of 32)
inline int64_t pg_cache4_tile_bytes(int64_t width) { return width * 9; }

// pg_linear4_gemv.cu: up to 16 rows, or the 16-row blocks of a route
int32_t pgk_linear4_gemv(pg_ctx *ctx, const pg_linear4 *lin, const bf16 *a, int64_t lda, int64_t m, int act, float limit, void *y, int y_dtype, int64_t ldy,
                         const PgRouted *routed, int64_t max_blocks);
size_t pgk_linear4_gemv_workspace(const pg_linear4 *lin);
// pg_linear4_tc.cu: any number of rows, or the 128-row blocks of a route (m: the rows that it can have)
int32_t pgk_linear4_tc(pg_ctx *ctx, const pg_linear4 *lin, const bf16 *a, int64_t lda, int64_t m, int act, float limit, void *y, int y_dtype, int64_t ldy,
                       const PgRouted *routed, const pg_route *route);
size_t pgk_linear4_tc_workspace(const pg_ctx *ctx);

#ifdef __CUDACC__
// scale and quant of a value, with the group's value of largest magnitude
__device__ __forceinline__ float four_scale(float top) { return isfinite(top) ? __bfloat162float(__float2bfloat16_rn(top * -0.125f)) : __uint_as_float(0x7fc00000u); }
__device__ __forceinline__ uint32_t four_quant(float w, float scale)
{
    if (!(scale != 0.0f) || !isfinite(scale)) return 8u;   // (a zero scale stands for zeros whatever the quants)
    return (uint32_t)min(15, max(0, __float2int_rn(__fdiv_rn(w, scale)) + 8));
}
// The same for four values, with a product in place of the quotients: that is off by 2^-18 at most where the scale is in the middle of its range
// (reciprocal 2 units in the last place, product half a one, quotients of up to 8), so what it rounds to is the quotient's integer unless it lies
// within 2^-17 of a half.
__device__ __forceinline__ void four_quants(const float (&w)[4], float scale, uint32_t (&q)[4])
{
    const float inv = __fdividef(1.0f, scale), mag = fabsf(scale);
    bool plain = mag >= 1e-30f && mag <= 1e30f;            // (false for not-a-number)
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const float x = w[e] * inv, n = rintf(x);
        plain = plain && fabsf(fabsf(x - n) - 0.5f) > 0x1p-17f;
        q[e] = (uint32_t)min(15, (int)n + 8);              // (the largest is -8 steps of the scale; bf16's rounding of that adds less than a half)
    }
    if (plain) return;
#pragma unroll
    for (int e = 0; e < 4; e++) q[e] = four_quant(w[e], scale);
}

// ---- quants -> f16 pairs: bits 0-3 / 4-7 of both halves of a word, as q - 8, exact.  1024 + q and 64 + q are f16 numbers that have the quant in
// their bits 0-3 and 4-7: one logical operation, then the offset comes off.  1024 + 16 q gives 16 (q - 8) with one constant less.
__device__ __forceinline__ uint32_t four_lop(uint32_t w, uint32_t mask, uint32_t base)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(base));   // (w & mask) | base
    return r;
}
__device__ __forceinline__ uint32_t four_sub_f16(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
constexpr uint32_t FOUR_LO = 0x000f000fu, FOUR_HI = 0x00f000f0u;
__device__ __forceinline__ uint32_t four_f16_lo(uint32_t w) { return four_sub_f16(four_lop(w, FOUR_LO, 0x64006400u), 0x64086408u); }   // 1024, 1032
__device__ __forceinline__ uint32_t four_f16_hi(uint32_t w) { return four_sub_f16(four_lop(w, FOUR_HI, 0x54005400u), 0x54805480u); }   // 64, 72
__device__ __forceinline__ uint32_t four_f16_hi16(uint32_t w) { return four_sub_f16(four_lop(w, FOUR_HI, 0x64006400u), 0x64806480u); }   // 1024, 1152
// the same as bf16, from bits 0-3: 128 + q, less 136
__device__ __forceinline__ uint32_t four_bf16_lo(uint32_t w)
{
    uint32_t r;
    const uint32_t v = four_lop(w, FOUR_LO, 0x43004300u), off = 0x43084308u;
    asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(v), "r"(off));
    return r;
}
// D[16 x 8] += A[16 x 16] B[16 x 8], f16 operands, f32 sums
__device__ __forceinline__ void four_mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same without sums to add to
__device__ __forceinline__ void four_mma_f16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ uint32_t four_pack_f16(float lo, float hi)
{
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
}
// Powers of two that bring numbers of magnitude up to `top` below 2^15 and back: f16 then holds every bf16 number down to 2^-31 of the
// largest exactly (eight bits, the last of them 2^-24 or more), and smaller ones to 2^-39 of it.  (An infinity stays one, and finite numbers beside it
// stay finite.)
__device__ __forceinline__ void four_range(float top, float &down, float &back)
{
    const int e = max((int)(__float_as_uint(top) >> 23 & 255u), 20);
    down = __uint_as_float((uint32_t)(268 - e) << 23);
    back = __uint_as_float((uint32_t)(e - 14) << 23);
}
#endif
