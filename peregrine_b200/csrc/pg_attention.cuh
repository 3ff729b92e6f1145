// What the two attention files share.
#pragma once

#include <math.h>

#include "pg_four.cuh"
#include "pg_lm.cuh"

struct AttnShape {
    int H, G, rep, D, V, dp, vp, sink;   // dp, vp: row widths of the caches (D and V rounded up to 16)
    int cap;                             // rows of a slot's and head's part of the cache
    int limit;                           // positions of a sequence
    int chunk;                           // 0: a position sees all before it; else those of its chunk, and cap is a multiple of chunk
    float eps, scale, coef, every;
    const float *qn, *kn;                // null: no norm
    const float *slopes;                 // [H], null: no distance bias
    // queries, keys and values in f16 over powers of two (null: in bf16): what a query is multiplied by [rows][H], and the largest
    // magnitudes of a head's keys and values, TOPS of them each
    const float *q_up, *k_top, *v_top;
    // [G][V up to 32 / 32][chunks of a slot]: the first row of a chunk whose values in 32 columns are not numbers, which are zeros where the values lie
    const int *v_bad;
};
constexpr int ATTN_TOPS = 32;
// Probabilities in f16 are 2^7 times those of the row's maximum (2^15 at most where that may fall behind by 2^8): those down to 2^-32 of the largest then
// count in the sums as they do in the denominator.  (From 1 on they ended at 2^-25: behind 131072 positions, 2^-8 of an output.)
constexpr float ATTN_P_UP = 7.0f;

#ifdef __CUDACC__
// A chunked layer keeps whole chunks only, position p in row p mod cap: the rows of a chunk lie next to each other.
__device__ __forceinline__ int attn_low(const AttnShape &s, int pos) { return s.chunk ? pos - pos % s.chunk : 0; }
__device__ __forceinline__ int attn_row(const AttnShape &s, int pos) { return s.chunk ? pos % s.cap : pos; }
__device__ __forceinline__ float attn_temperature(const AttnShape &s, int pos)
{
    if (s.every <= 0.0f) return 1.0f;
    return 1.0f + s.coef * logf(floorf(__fdiv_rn((float)(pos + 1), s.every)) + 1.0f);
}

// One warp: dst = rms_norm(src[0 .. D)) * w * mul, or src * mul where w is null; columns D .. dp are zero (D <= 256).
template <typename TA>
__device__ __forceinline__ void attn_head_norm(const float *src, const float *__restrict__ w, int D, int dp, float eps, float mul, TA *dst, int lane)
{
    float x[8], ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        x[i] = i * 32 + lane < D ? __ldcg(src + i * 32 + lane) : 0.0f;
        ss += x[i] * x[i];
    }
    ss = pg_warp_sum(ss);
    const float inv = w ? __fdiv_rn(1.0f, sqrtf(__fdiv_rn(ss, (float)D) + eps)) : 1.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int c = i * 32 + lane;
        if (c < dp) pg_put(dst + c, c < D ? x[i] * inv * (w ? __ldg(w + c) : 1.0f) * mul : 0.0f);
    }
}

// The powers of two of a head's keys or values, by a whole warp (they are within 2^15 times the first).
__device__ __forceinline__ void attn_range(const float *tops, int g, int lane, float &down, float &up)
{
    float top = __ldcg(tops + g * ATTN_TOPS + lane);
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    four_range(top, down, up);
}
// does a row that ends with position `pos` see values that are not numbers in the 32 columns from c on?
__device__ __forceinline__ bool attn_sees_bad(const AttnShape &s, int g, int c, int pos)
{
    const int row = attn_row(s, pos), chunks = s.chunk ? s.cap / s.chunk : 1;
    return __ldcg(s.v_bad + (g * ((s.V + 31) / 32) + c / 32) * chunks + (s.chunk ? row / s.chunk : 0)) <= row;
}
// operands of matrix instructions, two of them in a word
template <bool HALF>
__device__ __forceinline__ uint32_t attn_pack(float lo, float hi)
{
    return HALF ? four_pack_f16(lo, hi) : pg_pack_bf16(lo, hi);
}
#endif

// pg_attention.cu: the shape of a description; keys and values of prompts on mma.sync (any shape)
AttnShape pgk_attention_shape(const pg_attention *p);
int32_t pgk_attention_prompt(pg_ctx *ctx, const AttnShape &s, const pg_batch *bt, const bf16 *q, const bf16 *kc, const bf16 *vc, bf16 *out, int64_t ldo);
// out [rows][H V] f32; every head's query is a row of s.dp floats
int32_t pgk_attention_f32(pg_ctx *ctx, const AttnShape &s, const pg_batch *bt, const float *q, const float *kc, const float *vc, float *out, int64_t ldo);

// pg_attention_tc.cu
// Keys and values that a latent layer made from its latents for one sequence (csrc/pg_latent.cu): every head has its own, and
// a key has a second part that all heads share and that lies in the layer's cache.
struct AttnSplitKeys {
    const bf16 *q;          // [rows][H][qd]: the part for `k`, zero up to a multiple of 64, then the part for `shared`, the same
    int qd;
    const bf16 *k;          // [positions][H][kd], rows ldk elements apart
    int kd;
    const bf16 *v;          // [positions][H][vd], rows ldk elements apart
    int vd;
    int64_t ldk;
    const bf16 *shared;     // [positions][sd] of the sequence's slot, rows lds elements apart
    int sd;
    int64_t lds;
    const float *gate;      // [rows][H V], rows ldg elements apart: the output is multiplied by its sigmoid
    int64_t ldg;
    int seq, len, positions;   // the sequence, its tokens in this step and its positions with them
};
bool pgk_attention_split_supports(int kd, int sd, int V);
int32_t pgk_attention_split_tc(pg_ctx *ctx, const AttnShape &s, const pg_batch *bt, const AttnSplitKeys &k, bf16 *out, int64_t ldo);

bool pgk_attention_prompt_tc_supports(const AttnShape &s, const pg_batch *bt, int64_t slots, int64_t ldo, const void *out);
int32_t pgk_attention_prompt_tc(pg_ctx *ctx, const AttnShape &s, const pg_batch *bt, int64_t slots, const bf16 *q, const bf16 *kc, const bf16 *vc, bf16 *out,
                                int64_t ldo);
