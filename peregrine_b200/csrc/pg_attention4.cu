// Causal attention over a cache of keys and values in 4 bits (csrc/pg_four.cuh): a scale per 32 columns of a position, whose values are those of
// its positions as they are held, a step's own among them.  What a layer may have besides is that of csrc/pg_attention.cu.
//
// A head's part of a cache comes in tiles of 16 positions, so that a tile is one bulk copy: the quants of 32 columns after those of 32 columns, 256
// bytes each, then for the eight pairs of positions the scales of every 32 columns, both positions side by side.
//   keys    position 8 n + r, column 16 s + 4 t + 2 i + h of its 32 -> byte [r][t][s][2 h + n], low half for i = 0
//   values  position 8 i + 2 t + h, column 16 s + 8 n + r of its 32 -> byte [r][t][s][2 h + i], low half for n = 0
// Those are operands of mma.sync m16n8k16 once the quants are numbers: keys the B side of S = Q K^T (16 rows of queries), values the A side of
// O^T = V^T P^T, so that a lane's probabilities are the B operand as they come.  A byte belongs to one position: appending is byte stores.
//
//   few tokens of a sequence    attn4_few_kernel: streams the cache once, a block of 16 (token, head of the group) rows per CTA, the context in slices.
//                               Keys as f16 (exact: a quant as the low bits of an f16 number) times the query as f16 over a power of two (11 bits down to
//                               2^-24 of the row's largest), sums of 32 columns scaled in f32; values as bf16 integers (exact) times
//                               bf16(probability * scale).  One token per sequence
//                               (FUSED): the CTA with the newest position quantises and appends it.  The last CTA of a (sequence, rows) to finish
//                               merges the slices.  What bounds it, 32 + 8 heads of 128: instructions, 300 to a tile of 16 positions and 128 + 128
//                               columns, of which 64 take the quants apart (four bits at a time, the integer pipe at half rate); 4 contexts of 30000 to
//                               60000 71 us, 3.1 TB/s of 6.5, 16 of 2048 to 4096 31 us.  One of 2000: 10 us, a launch and seven dependent trips to
//                               memory (positions, tiles, slices' sums, tickets, the merge).
//   longer portions             attn4_append_kernel, then per sequence attn4_unfold_kernel and the kernels that prompts over a bf16 cache run through, on
//                               f16: keys and values over a power of two of their head, which is exact, queries over one of their own, probabilities
//                               times 2^7 (ATTN_P_UP).  The sequences go one after the other, each with its context unfolded into the same workspace.
#include <algorithm>
#include <type_traits>

#include "pg_async.cuh"
#include "pg_attention.cuh"
#include "pg_four.cuh"

namespace {

constexpr float LOG2E = 1.4426950408889634f;

// what the 4-bit form has beyond AttnShape: groups of 32 columns, bytes of a tile
struct Four {
    int gk, gv;                // groups of a key and of a value
    int kb, vb;                // bytes of a tile
    int64_t kh, vh;            // bytes of a head's part of a slot
};

// ---- quantising and placing a position (one warp) -----------------------------------------------------------------------
// x[i]: columns 32 i + lane; quants (a byte each) and scales to shared memory
__device__ __forceinline__ void quantise_row(const float (&x)[8], int groups, uint8_t *quants, bf16 *scales, int lane)
{
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if (i >= groups) break;
        const uint32_t mag = __float_as_uint(fabsf(x[i])), most = __reduce_max_sync(0xffffffffu, mag);   // (magnitudes order as integers; not-a-numbers are the largest)
        const int first = __ffs(__ballot_sync(0xffffffffu, mag == most)) - 1;
        const float scale = four_scale(__shfl_sync(0xffffffffu, x[i], first));
        quants[32 * i + lane] = (uint8_t)four_quant(x[i], scale);
        if (lane == 0) scales[i] = __float2bfloat16_rn(scale);
    }
    __syncwarp();
}
// into row `row` (0 .. 15) of a tile, in global or shared memory
__device__ __forceinline__ void put_scales(unsigned char *tile, const bf16 *scales, int row, int groups, int lane)
{
    if (lane < groups) *reinterpret_cast<bf16 *>(tile + groups * 256 + (((row >> 1) * groups + lane) * 2 + (row & 1)) * 2) = scales[lane];
}
__device__ __forceinline__ void put_key(unsigned char *tile, const uint8_t *q, const bf16 *scales, int row, int groups, int lane)
{
    const int n = row >> 3, r = row & 7;
    for (int i = lane; i < groups * 8; i += 32) {
        const int g = i >> 3, t = i >> 1 & 3, s = i & 1, c = 32 * g + 16 * s + 4 * t;
        unsigned char *at = tile + g * 256 + ((r * 4 + t) * 2 + s) * 4;
        at[n] = q[c] | q[c + 2] << 4;
        at[2 + n] = q[c + 1] | q[c + 3] << 4;
    }
    put_scales(tile, scales, row, groups, lane);
}
__device__ __forceinline__ void put_value(unsigned char *tile, const uint8_t *q, const bf16 *scales, int row, int groups, int lane)
{
    const int i8 = row >> 3, t = (row & 7) >> 1, h = row & 1;
    for (int i = lane; i < groups * 16; i += 32) {
        const int g = i >> 4, r = i >> 1 & 7, s = i & 1, c = 32 * g + 16 * s + r;
        tile[g * 256 + ((r * 4 + t) * 2 + s) * 4 + 2 * h + i8] = q[c] | q[c + 8] << 4;
    }
    put_scales(tile, scales, row, groups, lane);
}
// a head's row of the projection: x[i] = column 32 i + lane, normalised where w is there; zero behind `width`
__device__ __forceinline__ void load_row(const float *src, const float *__restrict__ w, int width, float eps, float (&x)[8], int lane)
{
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        x[i] = 32 * i + lane < width ? __ldcg(src + 32 * i + lane) : 0.0f;
        ss += x[i] * x[i];
    }
    if (!w) return;
    const float inv = __fdiv_rn(1.0f, sqrtf(__fdiv_rn(pg_warp_sum(ss), (float)width) + eps));
#pragma unroll
    for (int i = 0; i < 8; i++)
        if (32 * i + lane < width) x[i] *= inv * __ldg(w + 32 * i + lane);
}

// ---- append: a CTA per token, a warp per key or value head; with q: the queries too, for pg_attention4_prompt ----------------------
// A lane has four columns of every 128: 32 columns are those of eight lanes, so that the largest magnitudes of all groups are found together.
// The next row is on its way while one is worked on.  2000 tokens of 32 + 8 + 8 heads of 128: 23 us
// (49 MB of rows at 2.1 TB/s; instructions bound it, 160 to a row, three quarters of them the quants' and the queries' conversions).
constexpr int AP_WARPS = 8;
template <int NV, bool WIDE>                              // blocks of 128 columns; rows of 16-byte words
__global__ void __launch_bounds__(AP_WARPS * 32, NV == 1 ? 6 : 4)
    attn4_append_kernel(const AttnShape s, const Four f, const pg_batch bt, const float *__restrict__ proj, int64_t ldp, __half *__restrict__ q, float *__restrict__ q_up,
                        unsigned char *kc, unsigned char *vc, int32_t *status)
{
    pg_pdl_begin();
    const int m = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int pos = __ldcg(bt.d_pos + m);
    const int64_t slot = __ldcg(bt.d_seq_slot + __ldcg(bt.d_row_seq + m));
    if ((unsigned)pos >= (unsigned)s.limit) {   // outside the cache: record it, touch nothing
        if (threadIdx.x == 0) atomicExch(status, (int32_t)PG_ERR_INVALID);
        return;
    }
    const float *row = proj + (int64_t)m * ldp;
    const int at = attn_row(s, pos), items = q ? 2 * s.G + s.H : 2 * s.G;
    // item i: key heads, value heads, queries
    auto load = [&](int i, float4 (&x)[NV]) {
        const bool value = i >= s.G && i < 2 * s.G;
        const int width = value ? s.V : s.D;
        const float *src = row + (i < s.G ? (int64_t)(s.H + i) * s.D : value ? (int64_t)(s.H + s.G) * s.D + (int64_t)(i - s.G) * s.V : (int64_t)(i - 2 * s.G) * s.D);
#pragma unroll
        for (int v = 0; v < NV; v++) {
            const int c = 128 * v + 4 * lane;
            x[v] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (i >= items) continue;
            if (WIDE) {
                if (c < width) x[v] = __ldcg(reinterpret_cast<const float4 *>(src + c));
            } else {
                if (c < width) x[v].x = __ldcg(src + c);
                if (c + 1 < width) x[v].y = __ldcg(src + c + 1);
                if (c + 2 < width) x[v].z = __ldcg(src + c + 2);
                if (c + 3 < width) x[v].w = __ldcg(src + c + 3);
            }
        }
    };
    float4 ahead[NV];
    load(warp, ahead);
    const float mul = attn_temperature(s, pos);
    for (int i = warp; i < items; i += AP_WARPS) {
        float x[NV][4];
#pragma unroll
        for (int v = 0; v < NV; v++) x[v][0] = ahead[v].x, x[v][1] = ahead[v].y, x[v][2] = ahead[v].z, x[v][3] = ahead[v].w;
        load(i + AP_WARPS, ahead);
        const bool key = i < s.G, query = i >= 2 * s.G;
        const float *w = key ? s.kn : query ? s.qn : nullptr;
        if (w) {
            float ss = 0.0f;
#pragma unroll
            for (int v = 0; v < NV; v++) ss += x[v][0] * x[v][0] + x[v][1] * x[v][1] + x[v][2] * x[v][2] + x[v][3] * x[v][3];
            const float inv = __fdiv_rn(1.0f, sqrtf(__fdiv_rn(pg_warp_sum(ss), (float)s.D) + s.eps));
#pragma unroll
            for (int v = 0; v < NV; v++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int c = 128 * v + 4 * lane + e;
                    if (c < s.D) x[v][e] *= inv * __ldg(w + c);
                }
        }
        if (query) {
            // f16 over a power of two of the row's own
            float top = 0.0f;
#pragma unroll
            for (int v = 0; v < NV; v++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    x[v][e] *= mul;
                    top = fmaxf(top, fabsf(x[v][e]));
                }
            top = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(top)));
            float down, up;
            four_range(top, down, up);
            const int64_t to = (int64_t)m * s.H + i - 2 * s.G;
            if (lane == 0) q_up[to] = up;
#pragma unroll
            for (int v = 0; v < NV; v++) {
                const int c = 128 * v + 4 * lane;
                if (c < s.dp)
                    *reinterpret_cast<uint2 *>(q + to * s.dp + c) = make_uint2(four_pack_f16(x[v][0] * down, x[v][1] * down), four_pack_f16(x[v][2] * down, x[v][3] * down));
            }
            continue;
        }
        const int groups = key ? f.gk : f.gv;
        unsigned char *tile = key ? kc + (slot * s.G + i) * f.kh + (int64_t)(at >> 4) * f.kb : vc + (slot * s.G + i - s.G) * f.vh + (int64_t)(at >> 4) * f.vb;
        const int p = at & 15;
#pragma unroll
        for (int v = 0; v < NV; v++) {
            // (magnitudes order as integers; not-a-numbers are the largest)
            uint32_t most = 0;
            float mine = x[v][0];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const uint32_t mag = __float_as_uint(fabsf(x[v][e]));
                if (mag > most) most = mag, mine = x[v][e];
            }
            const uint32_t own = most;
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
            const uint32_t has = __ballot_sync(0xffffffffu, own == most) >> (lane & 24) & 255u;
            const float scale = four_scale(__shfl_sync(0xffffffffu, mine, (lane & 24) + __ffs(has) - 1));
            uint32_t n[4], all = 0;
            four_quants(x[v], scale, n);
#pragma unroll
            for (int e = 0; e < 4; e++) all |= n[e] << (8 * e);
            const uint32_t across = __shfl_xor_sync(0xffffffffu, all, 2);   // eight columns on (or back)
            const int g = 4 * v + (lane >> 3), half = lane >> 2 & 1;
            if (g < groups) {
                if (key) {
                    unsigned char *to = tile + g * 256 + (((p & 7) * 4 + (lane & 3)) * 2 + half) * 4 + (p >> 3);
                    to[0] = (unsigned char)(n[0] | n[2] << 4);
                    to[2] = (unsigned char)(n[1] | n[3] << 4);
                } else {
                    // columns r = 4 (lane & 1) + e of the first and the second eight in a byte: the lanes of the first write e = 0, 1
                    const bool second = lane >> 1 & 1;
                    const uint32_t both = second ? across | all << 4 : all | across << 4;
                    const int e = second ? 2 : 0, r = 4 * (lane & 1) + e;
                    unsigned char *to = tile + g * 256 + ((r * 4 + ((p & 7) >> 1)) * 2 + half) * 4 + 2 * (p & 1) + (p >> 3);
                    to[0] = (unsigned char)(both >> (8 * e));
                    to[32] = (unsigned char)(both >> (8 * e + 8));
                }
                if ((lane & 7) == 0) *reinterpret_cast<bf16 *>(tile + groups * 256 + (((p >> 1) * groups + g) * 2 + (p & 1)) * 2) = __float2bfloat16_rn(scale);
            }
        }
    }
}

// ---- a cache as numbers -------------------------------------------------------------------------------------------------
// quant of a tile: position p of 16, column c
template <bool VALUES>
__device__ __forceinline__ int quant_of(const unsigned char *tile, int p, int c)
{
    const int g = c >> 5, s = c >> 4 & 1;
    if (VALUES) return tile[g * 256 + (((c & 7) * 4 + ((p & 7) >> 1)) * 2 + s) * 4 + 2 * (p & 1) + (p >> 3)] >> (4 * (c >> 3 & 1)) & 15;
    return tile[g * 256 + (((p & 7) * 4 + (c >> 2 & 3)) * 2 + s) * 4 + 2 * (c & 1) + (p >> 3)] >> (4 * (c >> 1 & 1)) & 15;
}
__device__ __forceinline__ float scale_of(const unsigned char *tile, int groups, int p, int g)
{
    return __bfloat162float(*reinterpret_cast<const bf16 *>(tile + groups * 256 + (((p >> 1) * groups + g) * 2 + (p & 1)) * 2));
}

// grid (tiles, parts): f32 [parts][rows][32 groups]
template <bool VALUES>
__global__ void __launch_bounds__(128) attn4_read_kernel(const unsigned char *__restrict__ cache, int groups, int tile_bytes, int64_t head_bytes, int rows, float *__restrict__ out)
{
    pg_pdl_begin();
    const unsigned char *tile = cache + (int64_t)blockIdx.y * head_bytes + (int64_t)blockIdx.x * tile_bytes;
    const int first = (int)blockIdx.x * 16, width = groups * 32;
    float *dst = out + ((int64_t)blockIdx.y * rows + first) * width;
    for (int i = threadIdx.x; i < min(16, rows - first) * width; i += 128) {
        const int p = i / width, c = i - p * width;
        dst[i] = scale_of(tile, groups, p, c >> 5) * (float)(quant_of<VALUES>(tile, p, c) - 8);
    }
}

// grid (ATTN_TOPS, G, keys and values): no value of a head's rows [0, rows) is larger than the largest of its tops.  (Scales that are not numbers
// do not count: what lies beside them keeps its digits.)  Marks no row's values as bad.  A batch that is not the one the host was told of (a recorded
// call's may have changed) is reported.
__global__ void __launch_bounds__(128) attn4_tops_kernel(const unsigned char *__restrict__ kc, const unsigned char *__restrict__ vc, const Four f, int rows, int bad,
                                                         float *__restrict__ k_top, float *__restrict__ v_top, int *__restrict__ v_bad, const pg_batch bt, int seq, int len,
                                                         int positions, int slot, int32_t *status)
{
    __shared__ float tops[4];
    pg_pdl_begin();
    if (blockIdx.x == 0 && blockIdx.y == 0 && blockIdx.z == 0 && threadIdx.x == 0) {
        const int row0 = __ldcg(bt.d_seq_row0 + seq);
        if (__ldcg(bt.d_seq_row0 + seq + 1) - row0 != len || __ldcg(bt.d_pos + row0) + len != positions || __ldcg(bt.d_seq_slot + seq) != slot)
            atomicExch(status, (int32_t)PG_ERR_INVALID);
    }
    const bool values = blockIdx.z == 1;
    const int groups = values ? f.gv : f.gk, bytes = values ? f.vb : f.kb, part = blockIdx.x, words = groups * 8, tiles = (rows + 15) / 16;
    const unsigned char *head = values ? vc + blockIdx.y * f.vh : kc + blockIdx.y * f.kh;
    float top = 0.0f;
    for (int i = threadIdx.x; i < (tiles - part + ATTN_TOPS - 1) / ATTN_TOPS * words; i += 128) {
        const int tile = part + i / words * ATTN_TOPS, at = i % words, p = tile * 16 + at / groups * 2;
        if (tile >= tiles) break;
        const uint32_t two = __ldcg(reinterpret_cast<const uint32_t *>(head + (int64_t)tile * bytes + groups * 256) + at);
        const float s0 = fabsf(pg_bf16_lo(two)), s1 = fabsf(pg_bf16_hi(two));
        if (p < rows && isfinite(s0)) top = fmaxf(top, s0);
        if (p + 1 < rows && isfinite(s1)) top = fmaxf(top, s1);
    }
#pragma unroll
    for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x == 0) (values ? v_top : k_top)[blockIdx.y * ATTN_TOPS + part] = 8.0f * fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    if (values)
        for (int i = part * 128 + threadIdx.x; i < bad; i += ATTN_TOPS * 128) v_bad[blockIdx.y * (int64_t)bad + i] = 0x7fffffff;
}

// grid (tiles of 16 positions, G, keys and values): rows [0, rows) of a slot in f16 over the head's power of two, zeros up to row `padded`.  A scale of
// eight bits times a quant has eleven, so that f16 holds it as it is, down to 2^-29 of the head's largest.
// 3000 positions of 8 heads of 128: 9.3 us, 12.3 MB written; the pass over the scales in front of it 4.5 us.
__global__ void __launch_bounds__(128)
    attn4_unfold_kernel(const AttnShape s, const Four f, const unsigned char *__restrict__ kc, const unsigned char *__restrict__ vc, int rows, int padded,
                        __half *__restrict__ k, __half *__restrict__ v, int *__restrict__ v_bad)
{
    __shared__ __align__(16) unsigned char tile[8 * 288];
    __shared__ __align__(16) __half numbers[16][256 + 8];
    pg_pdl_begin();
    const bool values = blockIdx.z == 1;
    const int groups = values ? f.gv : f.gk, bytes = values ? f.vb : f.kb, width = values ? s.vp : s.dp, lane = threadIdx.x & 31;
    const uint4 *src = reinterpret_cast<const uint4 *>((values ? vc + blockIdx.y * f.vh : kc + blockIdx.y * f.kh) + (int64_t)blockIdx.x * bytes);
    for (int i = threadIdx.x; i < bytes / 16; i += 128) reinterpret_cast<uint4 *>(tile)[i] = __ldcg(src + i);
    float down, up;
    attn_range(values ? s.v_top : s.k_top, blockIdx.y, lane, down, up);
    __syncthreads();
    const int first = (int)blockIdx.x * 16, left = min(16, padded - first);
    const int r = lane >> 2, t = lane & 3;
    for (int g = threadIdx.x >> 5; g < groups; g += 4) {
        const uint2 two = *reinterpret_cast<const uint2 *>(tile + g * 256 + lane * 8);
        const uint32_t w[2] = {two.x, two.y};
        if (values) {
#pragma unroll
            for (int b = 0; b < 4; b++) {                 // byte 2 h + i
                const int p = 8 * (b & 1) + 2 * t + (b >> 1);
                float scale = scale_of(tile, groups, p, g);
                if (!isfinite(scale)) {
                    // a row that sees them has to say so, the others must not
                    const int row = first + p, chunks = s.chunk ? s.cap / s.chunk : 1;
                    if (r == 0 && row < rows) atomicMin(v_bad + (blockIdx.y * groups + g) * chunks + (s.chunk ? row / s.chunk : 0), row);
                    scale = 0.0f;
                }
                scale = first + p < rows ? scale * down : 0.0f;
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int n = 0; n < 2; n++) numbers[p][32 * g + 16 * e + 8 * n + r] = __float2half_rn(scale * (float)((int)(w[e] >> (8 * b + 4 * n) & 15u) - 8));
            }
        } else {
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const int p = 8 * n + r;
                const float scale = first + p < rows ? scale_of(tile, groups, p, g) * down : 0.0f;
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float x[4];                           // column 2 i + h: byte 2 h + n, half i
#pragma unroll
                    for (int c = 0; c < 4; c++) x[c] = first + p < rows ? scale * (float)((int)(w[e] >> (16 * (c & 1) + 8 * n + 4 * (c >> 1)) & 15u) - 8) : 0.0f;
                    *reinterpret_cast<uint2 *>(&numbers[p][32 * g + 16 * e + 4 * t]) = make_uint2(four_pack_f16(x[0], x[1]), four_pack_f16(x[2], x[3]));
                }
            }
        }
    }
    __syncthreads();
    __half *dst = (values ? v : k) + ((int64_t)blockIdx.y * s.cap + first) * width;
    const int eights = width / 8;
    for (int i = threadIdx.x; i < left * eights; i += 128) {
        const int p = i / eights, c = (i - p * eights) * 8;
        *reinterpret_cast<uint4 *>(dst + (int64_t)p * width + c) = *reinterpret_cast<const uint4 *>(&numbers[p][c]);
    }
}

// D[16 x 8] = C + A[16 x 16] B[16 x 8], f16 operands
__device__ __forceinline__ void mma_from(float (&d)[4], const float4 &c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c.x), "f"(c.y), "f"(c.z), "f"(c.w));
}

// the scales of a pair of positions, all groups'
template <int N, bool EXACT>
__device__ __forceinline__ void load_scales(uint32_t (&v)[N], uint32_t at, int groups)
{
    if (EXACT && N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]) : "r"(at + i * 4));
    } else if (EXACT && N == 2) {
        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(at));
    } else {
#pragma unroll
        for (int i = 0; i < N; i++)
            if (i < groups) asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[i]) : "r"(at + i * 4));
    }
}

// ---- few tokens: grid (slices of all sequences, G * blocks of 16 rows) --------------------------------------------------------------------
constexpr int A4_WARPS = 8, A4_STAGES = 3, A4_SLICES = 64, A4_FILL = 2;   // most fills in flight of a warp; most slices of a context; tiles of a fill

// CTAs to an SM.  More than eight rows of heads wider than 64: one with 255 registers a lane, as two with 128 spill (32 + 8 heads of 128, 16 x 4 tokens at
// 4096: 36.7 us instead of 64).  Up to eight rows keep two: one is slower in long contexts (4 at 60000: 85 instead of 75), faster in short ones (2000: 8.3, 9.3).
// Heads wider than 128 with more than eight rows spill some 490 bytes even so.
__host__ __device__ constexpr int a4_per_sm(int gk, int gv, bool hi) { return gk > 4 || gv > 4 || (hi && gk + gv > 4) ? 1 : 2; }

// part [blocks of rows][slices][16][vs + 4]: sums, then maximum (log 2 units) and denominator of each row
// EXACT: GK and GV are the groups of the layer, else at least as many
template <int GK, int GV, bool HI, bool FUSED, bool EXACT>
__global__ void __launch_bounds__(A4_WARPS * 32, a4_per_sm(GK, GV, HI))
    attn4_few_kernel(const AttnShape s, const Four f, const pg_batch bt, int few, int per, int stages, const float *__restrict__ proj, int64_t ldp, unsigned char *kc, unsigned char *vc,
                     float *part, int32_t *tickets, bf16 *__restrict__ out, int64_t ldo, int32_t *status, unsigned long long limit_ns)
{
    constexpr int NT = HI ? 2 : 1, JT = HI ? 1 : 2;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) uint64_t bars[A4_WARPS * A4_STAGES];
    __shared__ float weight[16][A4_SLICES];
    __shared__ float denom[16], back[16];
    __shared__ __align__(16) float4 offset[8][8];         // of rows r, r, r + 8, r + 8
    __shared__ int last_in;
    __shared__ volatile int abort_flag;
    __shared__ uint8_t new_q[2][256];
    __shared__ bf16 new_s[2][8];
    __shared__ volatile int kept[4];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int S = gridDim.x, g = blockIdx.y % s.G, block = blockIdx.y / s.G;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = lane >> 2, t = lane & 3;
    const int gk = EXACT ? GK : f.gk, gv = EXACT ? GV : f.gv, kbytes = gk * 288, vbytes = gv * 288, stage = A4_FILL * (kbytes + vbytes), vs = gv * 32;
    const uint32_t ring = pg_smem(smem) + (uint32_t)(warp * stages) * stage, bar = pg_smem(bars) + (uint32_t)warp * A4_STAGES * 8;
    const int qs = gk * 32 + 8;                                       // f16 elements between the rows of queries
    __half *qrow = reinterpret_cast<__half *>(smem + A4_WARPS * stages * stage);
    float *mg = reinterpret_cast<float *>(smem);                      // the merge reuses the rings
    if (threadIdx.x == 0) {
        for (int i = 0; i < A4_WARPS * A4_STAGES; i++) pg_mbar_init(pg_smem(bars) + 8 * i, 1);
        abort_flag = 0;
        pg_mbar_fence();
    }
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // A sequence's part of this block: count rows (token, head) = (block * 16 + c) / rep, % rep; the cache's rows x0 .. x1 - 1 hold the positions
    // low .. of them (in a chunked layer T is 1, and a chunk's rows lie together), a0 is the first row of the first fill.
    struct Seq {
        int row0 = 0, count = 0, pos0 = 0, low = 0, x0 = 0, x1 = 0, a0 = 0;
    };
    auto look = [&](int i, Seq &q) {
        q.row0 = __ldcg(bt.d_seq_row0 + i);
        const int T = __ldcg(bt.d_seq_row0 + i + 1) - q.row0;
        q.count = min(16, T * s.rep - block * 16);
        if (T > few || q.count <= 0) return false;
        q.pos0 = __ldcg(bt.d_pos + q.row0);
        if (q.pos0 < 0 || q.pos0 + T > s.limit) {                     // outside the cache: record it, touch nothing (all CTAs of the sequence leave)
            atomicExch(status, (int32_t)PG_ERR_INVALID);
            return false;
        }
        q.low = attn_low(s, q.pos0), q.x0 = attn_row(s, q.low), q.x1 = q.x0 + (q.pos0 + (block * 16 + q.count - 1) / s.rep) + 1 - q.low;
        q.a0 = q.x0 & ~31;
        return true;
    };
    // per > 0: so many slices to every context, in whole fills of all warps (256 rows).  per == 0, single tokens of 2 to 32 sequences: slices of one length,
    // the shortest of which there are no more than CTAs, found by every warp for itself, a lane to a sequence.  (32 + 8 heads of 128, contexts of 16 sequences
    // anywhere up to 4096: 27.2 us with equal numbers, 18.8 dealt out; all of 4096: 31.1 both.)
    int seq, split, used, chunk;
    int64_t slot = 0;
    Seq me;
    if (!FUSED || per) {
        seq = blockIdx.x / per, split = blockIdx.x - seq * per;
        slot = __ldcg(bt.d_seq_slot + seq);
        if (!look(seq, me)) return;
        chunk = ((me.x1 - me.a0 + per - 1) / per + 255) & ~255;
        used = (me.x1 - me.a0 + chunk - 1) / chunk;
        if (split >= used) return;
    } else {
        int own = 0;
        if (lane < bt.seqs) {
            slot = __ldcg(bt.d_seq_slot + lane);
            own = look(lane, me) ? (me.x1 - me.a0 + 255) / 256 : 0;
        }
        const int all = __reduce_add_sync(0xffffffffu, own), most = __reduce_max_sync(0xffffffffu, own);
        uint32_t lo = max(1, max((all + S - 1) / S, (most + A4_SLICES - 1) / A4_SLICES)), hi = max((int)lo, most);
        for (uint32_t mid = lo; lo < hi; mid = (lo + hi) / 2) {       // (the shortest that could be is tried first)
            if (__reduce_add_sync(0xffffffffu, (own + mid - 1) / mid) <= (uint32_t)S)
                hi = mid;
            else
                lo = mid + 1;
        }
        chunk = (int)lo * 256;
        // this CTA's sequence: the one whose slices hold the CTA's number
        const int n = (own + lo - 1) / lo;
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, upto > (int)blockIdx.x);
        if (!past) return;
        seq = __ffs(past) - 1;
        used = __shfl_sync(0xffffffffu, n, seq);
        split = (int)blockIdx.x - __shfl_sync(0xffffffffu, upto - n, seq);
        slot = __shfl_sync(0xffffffffu, slot, seq);
        me.row0 = __shfl_sync(0xffffffffu, me.row0, seq), me.count = __shfl_sync(0xffffffffu, me.count, seq);
        me.pos0 = __shfl_sync(0xffffffffu, me.pos0, seq), me.low = __shfl_sync(0xffffffffu, me.low, seq);
        me.x0 = __shfl_sync(0xffffffffu, me.x0, seq), me.x1 = __shfl_sync(0xffffffffu, me.x1, seq), me.a0 = __shfl_sync(0xffffffffu, me.a0, seq);
    }
    const int row0 = me.row0, count = me.count, pos0 = me.pos0, low = me.low, x0 = me.x0, x1 = me.x1;
    const int t0 = me.a0 + split * chunk, t1 = min(x1, t0 + chunk);
    if (threadIdx.x == 0) kept[0] = split, kept[1] = used, kept[2] = row0, kept[3] = count;   // (for the end: registers are short in between)
    const bool newest = FUSED && t1 == x1;
    unsigned char *kb = kc + (slot * s.G + g) * f.kh, *vb = vc + (slot * s.G + g) * f.vh;

    const int nfills = (t1 - t0 + 31) / 32, mine = nfills > warp ? (nfills - warp + A4_WARPS - 1) / A4_WARPS : 0;
    const int tiles = (s.cap + 15) / 16;                              // of a head's part
    auto fetch = [&](int i, int to) {
        if (lane == 0) {
            const uint32_t at = ring + (uint32_t)(to) * stage, on = bar + (uint32_t)(to) * 8;
            const int tile = (t0 >> 4) + A4_FILL * (warp + A4_WARPS * i), n = min(A4_FILL, tiles - tile);
            pg_mbar_expect(on, (uint32_t)(n * (kbytes + vbytes)));
            pg_bulk_load(at, kb + (int64_t)tile * kbytes, (uint32_t)(n * kbytes), on);
            pg_bulk_load(at + A4_FILL * kbytes, vb + (int64_t)tile * vbytes, (uint32_t)(n * vbytes), on);
        }
    };
    for (int i = 0; i < stages && i < mine; i++) fetch(i, i);

    // the rows' queries as f16 over a power of two, and what their scores are multiplied by
    const float sl = s.scale * LOG2E;
    for (int c = warp; c < 16; c += A4_WARPS) {
        if (c < count) {
            const int idx = block * 16 + c, token = idx / s.rep, h = g * s.rep + idx % s.rep;
            float x[8], top = 0.0f;
            load_row(proj + (int64_t)(row0 + token) * ldp + (int64_t)h * s.D, s.qn, s.D, s.eps, x, lane);
            const float mul = attn_temperature(s, pos0 + token);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[i] *= mul;
                top = fmaxf(top, fabsf(x[i]));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            float down, up;
            four_range(top, down, up);
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < gk) {
                    const __half v = __float2half_rn(x[i] * down);
                    qrow[c * qs + 32 * i + lane] = v;
                    const float sum = pg_warp_sum(__half2float(v));
                    if (lane < 2) reinterpret_cast<float *>(&offset[c & 7][i])[c / 8 * 2 + lane] = sum * -0x1p-21f;   // (the keys' quants are 8 too large)
                }
            if (lane == 0) back[c] = up * sl * 0x1p12f;   // (half of the 2^24 of the scores' smallest steps, so that neither factor leaves the range)
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < gk) qrow[c * qs + 32 * i + lane] = __float2half_rn(0.0f);
            if (lane < 16) reinterpret_cast<float *>(&offset[c & 7][lane >> 1])[c / 8 * 2 + (lane & 1)] = 0.0f;
            if (lane == 0) back[c] = 0.0f;
        }
    }
    if (newest && warp >= A4_WARPS - 2) {
        // the newest position: warp 6 its key, warp 7 its value
        const bool key = warp == A4_WARPS - 2;
        const float *row = proj + (int64_t)row0 * ldp;
        float x[8];
        load_row(key ? row + (int64_t)(s.H + g) * s.D : row + (int64_t)(s.H + s.G) * s.D + (int64_t)g * s.V, key ? s.kn : nullptr, key ? s.D : s.V, s.eps, x, lane);
        quantise_row(x, key ? gk : gv, new_q[key ? 0 : 1], new_s[key ? 0 : 1], lane);
    }
    __syncthreads();
    if (newest && block == 0 && warp >= A4_WARPS - 2) {
        // appended for later steps; this step takes it from shared memory (below)
        const int at = x1 - 1;
        if (warp == A4_WARPS - 2)
            put_key(kb + (int64_t)(at >> 4) * kbytes, new_q[0], new_s[0], at & 15, gk, lane);
        else
            put_value(vb + (int64_t)(at >> 4) * vbytes, new_q[1], new_s[1], at & 15, gv, lane);
    }
    uint32_t qf[GK][2][HI ? 4 : 2];
#pragma unroll
    for (int i = 0; i < GK; i++) {
        if (i >= gk) break;
#pragma unroll
        for (int e = 0; e < 2; e++) {
            // columns 4 t + {0, 1} and 4 t + {2, 3} of 16; the second pair's keys come 16 times too large
            const uint2 lo = *reinterpret_cast<const uint2 *>(qrow + r * qs + 32 * i + 16 * e + 4 * t);
            const __half2 less = __float2half2_rn(0.0625f);
            __half2 b = __hmul2(*reinterpret_cast<const __half2 *>(&lo.y), less);
            qf[i][e][0] = lo.x;
            qf[i][e][1] = *reinterpret_cast<uint32_t *>(&b);
            if constexpr (HI) {
                const uint2 hi = *reinterpret_cast<const uint2 *>(qrow + (r + 8) * qs + 32 * i + 16 * e + 4 * t);
                b = __hmul2(*reinterpret_cast<const __half2 *>(&hi.y), less);
                qf[i][e][2] = hi.x;
                qf[i][e][3] = *reinterpret_cast<uint32_t *>(&b);
            }
        }
    }
    float o[GV][2][NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int i = 0; i < GV; i++) o[i][0][n][j] = o[i][1][n][j] = 0.0f;
    // of the lane's rows r (and r + 8): factor of the scores, last row of the cache seen, slope
    float fac[NT], m[NT], l[NT], bias[NT];
    int seen[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const int c = r + 8 * n, idx = block * 16 + min(c, count - 1);
        fac[n] = back[c];
        seen[n] = x0 + pos0 + idx / s.rep - low;
        bias[n] = s.slopes ? __ldg(s.slopes + g * s.rep + idx % s.rep) * LOG2E : 0.0f;
        m[n] = -1e30f, l[n] = 0.0f;                       // (finite: exp2(-inf - m) is 0 where a row sees nothing of a slice)
    }
    const int sees_all = x0 + pos0 + block * 16 / s.rep - low;        // of the block's first row: every row sees that far
    bool ok = true;
    int at_stage = 0;
    uint32_t phase = 0;
    for (int i = 0; i < mine; i++) {
        ok = pg_mbar_wait_warp(bar + (uint32_t)at_stage * 8, phase, &abort_flag, status, limit_ns);
        if (!ok) break;
        const int j0 = t0 + 32 * (warp + A4_WARPS * i);
        unsigned char *at = smem + (size_t)(warp * stages + at_stage) * stage;
        if (newest && j0 + 32 >= x1) {
            // the copies brought what the cache held at the newest position: put the new one in its place
            const int row = x1 - 1 - j0;
            put_key(at + (row >> 4) * kbytes, new_q[0], new_s[0], row & 15, gk, lane);
            put_value(at + A4_FILL * kbytes + (row >> 4) * vbytes, new_q[1], new_s[1], row & 15, gv, lane);
            __syncwarp();
        }
        // (the masks have a version of their own: taking them out of the way of all other keys is a fifth of the instructions)
        auto tiles_of = [&](auto masked) {
            constexpr bool edge = decltype(masked)::value;
#pragma unroll
            for (int part = 0; part < A4_FILL; part += JT) {  // as many tiles at once as registers allow
                const int jp = j0 + 16 * part;
                if (jp >= t1) break;                          // (uniform)
                // scores of keys 16 h + 8 n + 2 t and 16 h + 8 n + 2 t + 1 with rows r and r + 8.  A quant as the low bits of an f16 number is that number of
                // its smallest steps, 2^-24; the sums start at what 8 of them in every column make.
                float sc[JT][2][2 * NT];
#pragma unroll
                for (int h = 0; h < JT; h++) {
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int j = 0; j < 2 * NT; j++) sc[h][n][j] = 0.0f;
                    const uint32_t kt = pg_smem(at) + (uint32_t)((part + h) * kbytes);
                    uint32_t ks[2][GK];                   // of keys 8 n + 2 t and 8 n + 2 t + 1
#pragma unroll
                    for (int n = 0; n < 2; n++) load_scales<GK, EXACT>(ks[n], kt + (uint32_t)((gk * 64 + (4 * n + t) * gk) * 4), gk);
#pragma unroll
                    for (int x = 0; x < GK; x++) {
                        if (x >= gk) break;
                        const float4 c4 = offset[r][x];
                        float d[2][4];
                        uint32_t w[2];
                        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(kt + x * 256 + lane * 8));
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const uint32_t w8 = w[e] >> 8, q0 = qf[x][e][0], q1 = HI ? qf[x][e][2 % (HI ? 4 : 2)] : 0u, q2 = qf[x][e][1], q3 = HI ? qf[x][e][3 % (HI ? 4 : 2)] : 0u;
                            if (e == 0) {
                                mma_from(d[0], c4, q0, q1, q2, q3, w[e] & FOUR_LO, w[e] & FOUR_HI);
                                mma_from(d[1], c4, q0, q1, q2, q3, w8 & FOUR_LO, w8 & FOUR_HI);
                            } else {
                                four_mma_f16(d[0], q0, q1, q2, q3, w[e] & FOUR_LO, w[e] & FOUR_HI);
                                four_mma_f16(d[1], q0, q1, q2, q3, w8 & FOUR_LO, w8 & FOUR_HI);
                            }
                        }
#pragma unroll
                        for (int n = 0; n < 2; n++) {
                            const float s0 = pg_bf16_lo(ks[n][x]), s1 = pg_bf16_hi(ks[n][x]);
                            sc[h][n][0] = fmaf(s0, d[n][0], sc[h][n][0]), sc[h][n][1] = fmaf(s1, d[n][1], sc[h][n][1]);
                            if (HI) sc[h][n][2 * NT - 2] = fmaf(s0, d[n][2], sc[h][n][2 * NT - 2]), sc[h][n][2 * NT - 1] = fmaf(s1, d[n][3], sc[h][n][2 * NT - 1]);
                        }
                    }
                }
                // to units of log 2, bias, mask
                float top[NT];
                uint32_t hidden = 0;                      // bit (2 h + n) 2 NT + 2 u + j
#pragma unroll
                for (int u = 0; u < NT; u++) {
                    top[u] = -INFINITY;
                    const float b0 = s.slopes ? bias[u] * (float)(jp + 2 * t - seen[u]) : 0.0f;
#pragma unroll
                    for (int h = 0; h < JT; h++)
#pragma unroll
                        for (int n = 0; n < 2; n++)
#pragma unroll
                            for (int j = 0; j < 2; j++) {
                                float v = sc[h][n][2 * u + j] * 0x1p12f;
                                v = s.slopes ? fmaf(v, fac[u], fmaf(bias[u], (float)(16 * h + 8 * n + j), b0)) : v * fac[u];
                                if (edge) {
                                    const int x = jp + 16 * h + 8 * n + 2 * t + j;
                                    if (x < x0 || x >= t1 || x > seen[u]) v = -INFINITY, hidden |= 1u << ((2 * h + n) * 2 * NT + 2 * u + j);
                                }
                                sc[h][n][2 * u + j] = v;
                                top[u] = fmaxf(top[u], v);
                            }
                }
                // the maximum is replaced where it falls behind by more than 2^8, which is rare behind the first keys
                if (__any_sync(0xffffffffu, top[0] > m[0] + 8.0f || top[NT - 1] > m[NT - 1] + 8.0f)) {
#pragma unroll
                    for (int u = 0; u < NT; u++) {
                        top[u] = fmaxf(top[u], __shfl_xor_sync(0xffffffffu, top[u], 1));
                        top[u] = fmaxf(top[u], __shfl_xor_sync(0xffffffffu, top[u], 2));
                        const float next = fmaxf(m[u], top[u]), corr = pg_ex2(m[u] - next);
                        m[u] = next;
                        // sums lie by row as columns: 2 t and 2 t + 1 of every eight
                        const float c0 = __shfl_sync(0xffffffffu, corr, 8 * t), c1 = __shfl_sync(0xffffffffu, corr, 8 * t + 4);
                        auto less = [&](float (&v)[4]) { v[0] *= c0, v[1] *= c1, v[2] *= c0, v[3] *= c1; };
                        l[u] *= corr;
#pragma unroll
                        for (int x = 0; x < GV; x++) less(o[x][0][u]), less(o[x][1][u]);
                    }
                }
#pragma unroll
                for (int h = 0; h < JT; h++)
#pragma unroll
                    for (int n = 0; n < 2; n++)
#pragma unroll
                        for (int j = 0; j < 2 * NT; j++) {
                            sc[h][n][j] = pg_ex2(sc[h][n][j] - m[j >> 1]);
                            l[j >> 1] += sc[h][n][j];
                        }
                // O^T += V^T P'^T, P' a probability times its value's scale
#pragma unroll
                for (int h = 0; h < JT; h++) {
                    const uint32_t vt = pg_smem(at) + (uint32_t)(A4_FILL * kbytes + (part + h) * vbytes);
                    uint32_t scales[2][GV];
#pragma unroll
                    for (int n = 0; n < 2; n++) load_scales<GV, EXACT>(scales[n], vt + (uint32_t)((gv * 64 + (4 * n + t) * gv) * 4), gv);
#pragma unroll
                    for (int x = 0; x < GV; x++) {
                        if (x >= gv) break;
                        uint32_t b[NT][2];
#pragma unroll
                        for (int n = 0; n < 2; n++) {
#pragma unroll
                            for (int u = 0; u < NT; u++) {
                                float p0 = sc[h][n][2 * u] * pg_bf16_lo(scales[n][x]), p1 = sc[h][n][2 * u + 1] * pg_bf16_hi(scales[n][x]);
                                // (what a row does not see may hold anything; what it sees is not a number whatever its weight, 0 too)
                                if (edge) {
                                    const int bit = (2 * h + n) * 2 * NT + 2 * u;
                                    p0 = hidden >> bit & 1u ? 0.0f : p0, p1 = hidden >> (bit + 1) & 1u ? 0.0f : p1;
                                }
                                b[u][n] = pg_pack_bf16(p0, p1);
                            }
                        }
                        uint32_t w[2];
                        asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(vt + x * 256 + lane * 8));
#pragma unroll
                        for (int e = 0; e < 2; e++) {
                            const uint32_t a0 = four_bf16_lo(w[e]), a1 = four_bf16_lo(w[e] >> 4), a2 = four_bf16_lo(w[e] >> 8), a3 = four_bf16_lo(w[e] >> 12);
#pragma unroll
                            for (int u = 0; u < NT; u++) pg_mma_bf16(o[x][e][u], a0, a1, a2, a3, b[u][0], b[u][1]);
                        }
                    }
                }
            }
        };
        if (j0 < x0 || j0 + 31 > sees_all || j0 + 31 >= t1)   // some row does not see all of these
            tiles_of(std::true_type{});
        else
            tiles_of(std::false_type{});
        __syncwarp();                                     // every lane is done with the stage before it is filled again
        if (i + stages < mine) fetch(i + stages, at_stage);
        if (++at_stage == stages) at_stage = 0, phase ^= 1;
    }
    if (!ok) {
        // copies that are still in flight get a bounded time to land before their shared memory is used again
        const unsigned long long w0 = pg_globaltimer_ns();
        while (pg_globaltimer_ns() - w0 < 2000000ull) {
        }
    }
    __syncthreads();                                      // the rings are free
    // warps meet in shared memory: [warp][16][vs + 4]
    const int ms = vs + 4;
    float *w0 = mg + (size_t)warp * 16 * ms;
#pragma unroll
    for (int x = 0; x < GV; x++) {
        if (x >= gv) break;
#pragma unroll
        for (int u = 0; u < NT; u++) {
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int j = 0; j < 4; j++) w0[(8 * u + 2 * t + (j & 1)) * ms + 32 * x + 16 * e + r + 8 * (j >> 1)] = o[x][e][u][j];
        }
    }
#pragma unroll
    for (int u = 0; u < NT; u++) {
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 1);
        l[u] += __shfl_xor_sync(0xffffffffu, l[u], 2);
        if (t == 0) w0[(r + 8 * u) * ms + vs] = m[u], w0[(r + 8 * u) * ms + vs + 1] = l[u];
    }
    __syncthreads();
    // (a sequence's slices are neighbours)
    const int slices = kept[1], row_at = kept[2], rows = kept[3];
    const int64_t first = (int64_t)blockIdx.y * S + blockIdx.x - kept[0];
    float *mine_part = part + ((int64_t)blockIdx.y * S + blockIdx.x) * 16 * ms;
    const int vq = vs / 4;
    auto put = [&](int c, int col, const float4 &a, float by) {
        const int idx = block * 16 + c;
        bf16 *dst = out + (int64_t)(row_at + idx / s.rep) * ldo + (int64_t)(g * s.rep + idx % s.rep) * s.V + col;
        const float y[4] = {a.x * by, a.y * by, a.z * by, a.w * by};
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (col + i < s.V) pg_put(dst + i, y[i]);
    };
    for (int x = threadIdx.x; x < rows * vq; x += A4_WARPS * 32) {
        const int c = x / vq, col = (x - c * vq) * 4;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < A4_WARPS; w++) top = fmaxf(top, mg[((size_t)w * 16 + c) * ms + vs]);
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < A4_WARPS; w++) {
            const float *from = mg + ((size_t)w * 16 + c) * ms;
            const float by = pg_ex2(from[vs] - top);      // 0 for a warp that saw nothing
            const float4 v = *reinterpret_cast<const float4 *>(from + col);
            a.x = fmaf(by, v.x, a.x), a.y = fmaf(by, v.y, a.y), a.z = fmaf(by, v.z, a.z), a.w = fmaf(by, v.w, a.w);
            sum = fmaf(by, from[vs + 1], sum);
        }
        if (slices == 1) {
            float by = 1.0f;
            if (s.sink) {
                const float mm = fmaxf(top, 0.0f);
                by = pg_ex2(top - mm);
                sum = sum * by + pg_ex2(-mm);
            }
            put(c, col, a, __fdiv_rn(by, sum));
        } else {
            *reinterpret_cast<float4 *>(mine_part + (size_t)c * ms + col) = a;
            if (col == 0) *reinterpret_cast<float2 *>(mine_part + (size_t)c * ms + vs) = make_float2(top, sum);
        }
    }
    if (slices == 1) return;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();
        last_in = atomicAdd(tickets + first, 1) == slices - 1;
    }
    __syncthreads();
    if (!last_in) return;
    __threadfence();
    if (threadIdx.x == 0) tickets[first] = 0;
    // a warp per row: the slices' weights; then all columns, eight slices' loads in flight, the first eight's while the weights are found
    const float *parts = part + first * 16 * ms;
    float4 v[8];
    auto load = [&](int x, int k0) {
        const float *from = parts + (size_t)(x / vq) * ms + (x % vq) * 4;
#pragma unroll
        for (int k = 0; k < 8; k++) v[k] = __ldcg(reinterpret_cast<const float4 *>(from + (size_t)min(k0 + k, slices - 1) * 16 * ms));
    };
    if (threadIdx.x < rows * vq) load(threadIdx.x, 0);
    for (int c = warp; c < rows; c += A4_WARPS) {
        float2 ml[A4_SLICES / 32];
        float top = s.sink ? 0.0f : -INFINITY, sum = 0.0f;
#pragma unroll
        for (int i = 0; i < A4_SLICES / 32; i++) {
            const int k = i * 32 + lane;
            ml[i] = k < slices ? __ldcg(reinterpret_cast<const float2 *>(parts + ((size_t)k * 16 + c) * ms + vs)) : make_float2(-INFINITY, 0.0f);
            top = fmaxf(top, ml[i].x);
        }
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
#pragma unroll
        for (int i = 0; i < A4_SLICES / 32; i++) {
            const float by = pg_ex2(ml[i].x - top);
            weight[c][i * 32 + lane] = by;
            sum = fmaf(by, ml[i].y, sum);
        }
        sum = pg_warp_sum(sum) + (s.sink ? pg_ex2(-top) : 0.0f);
        if (lane == 0) denom[c] = __fdiv_rn(1.0f, sum);
    }
    __syncthreads();
    for (int x = threadIdx.x; x < rows * vq; x += A4_WARPS * 32) {
        const int c = x / vq, col = (x - c * vq) * 4;
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int k0 = 0; k0 < slices; k0 += 8) {            // (behind the last slice its weight is 0)
            if (x != (int)threadIdx.x || k0 > 0) load(x, k0);
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float by = k0 + k < slices ? weight[c][k0 + k] : 0.0f;
                a.x = fmaf(by, v[k].x, a.x), a.y = fmaf(by, v[k].y, a.y), a.z = fmaf(by, v[k].z, a.z), a.w = fmaf(by, v[k].w, a.w);
            }
        }
        put(c, col, a, denom[c]);
    }
}

Four four_of(const AttnShape &s)
{
    Four f;
    f.gk = (s.D + 31) / 32, f.gv = (s.V + 31) / 32;
    f.kb = (int)pg_cache4_tile_bytes(f.gk * 32), f.vb = (int)pg_cache4_tile_bytes(f.gv * 32);
    const int64_t tiles = (s.cap + 15) / 16;
    f.kh = tiles * f.kb, f.vh = tiles * f.vb;
    return f;
}

// Slices of all sequences' contexts: as many CTAs as SMs take at once, none shorter than 256 rows.  per: of every context, 0 where they are dealt out
int slices(const pg_ctx *ctx, int64_t seqs, int64_t rows, const AttnShape &s, int per_sm, bool single, int &per)
{
    const int64_t cap = s.chunk && s.chunk < s.cap ? s.chunk : s.cap;
    const int64_t most = std::min<int64_t>((cap + 31 + 255) / 256, A4_SLICES), at_once = per_sm * (int64_t)ctx->sm_count / std::max<int64_t>(1, rows);   // (a chunk may begin inside a fill)
    const int64_t all = std::min(at_once, seqs * most);
    per = (int)std::max<int64_t>(1, all / std::max<int64_t>(1, seqs));
    if (single && seqs > 1 && seqs <= 32 && all > seqs) {
        per = 0;
        return (int)all;
    }
    return (int)(seqs * per);
}

template <int GK, int GV, bool HI, bool FUSED, bool EXACT>
int32_t run_few(pg_ctx *ctx, const AttnShape &s, const Four &f, const pg_batch *bt, int few, int blocks, const float *proj, int64_t ldp, unsigned char *kc,
                unsigned char *vc, float *part, int32_t *tickets, bf16 *out, int64_t ldo)
{
    auto kern = attn4_few_kernel<GK, GV, HI, FUSED, EXACT>;
    // (two CTAs to an SM where the widths allow)
    const int fill = A4_WARPS * A4_FILL * (f.kb + f.vb), stages = 3 * fill <= 100 * 1024 ? 3 : 2, rings = stages * fill;
    const int smem = std::max(rings + 16 * (f.gk * 32 + 8) * 2, A4_WARPS * 16 * (f.gv * 32 + 4) * 4);
    static std::atomic<uint64_t> set{0};
    PG_CUDA(pg_max_smem_once(kern, 200 * 1024, ctx->device, set));   // (widths of 256: 157 KB)
    int per;
    const int S = slices(ctx, bt->seqs, (int64_t)s.G * blocks, s, a4_per_sm(GK, GV, HI), FUSED, per);
    return launch_pdl(ctx, kern, dim3((unsigned)S, (unsigned)(s.G * blocks)), dim3(A4_WARPS * 32), (size_t)smem, s, f, *bt, few, per, stages, proj, ldp, kc,
                      vc, part, tickets, out, ldo, ctx->d_status, ctx->wait_limit_ns);
}

int32_t check(const pg_attention *p, const pg_batch *batch, const void *kc, const void *vc, const void *out, int32_t dtype, int64_t ldo)
{
    PG_REQUIRE(p && batch && kc && vc && out && p->d_q && p->d_part && p->d_tickets, "attention4: null pointer");
    PG_REQUIRE(dtype == PG_BF16, "attention4: steps are bf16");
    PG_REQUIRE(p->heads > 0 && p->kv_heads > 0 && p->heads % p->kv_heads == 0 && p->dim > 0 && p->dim <= 256 && p->vdim > 0 && p->vdim <= 256 && p->cap > 0 && p->slots > 0,
               "attention4: bad shape (heads %d / %d, dim %d and vdim %d at most 256)", p->heads, p->kv_heads, p->dim, p->vdim);
    PG_REQUIRE(p->chunk >= 0 && (p->chunk == 0 ? p->positions <= p->cap : p->cap % p->chunk == 0), "attention4: a cache of %d rows for %d positions in chunks of %d",
               p->cap, p->positions, p->chunk);
    PG_REQUIRE(p->chunk == 0 || p->positions <= p->cap || ((int64_t)(p->chunk + batch->max_len - 2) / p->chunk + 1) * p->chunk <= p->cap,
               "attention4: a step of %d tokens has more chunks of %d than the cache of %d rows", batch->max_len, p->chunk, p->cap);
    PG_REQUIRE(((uintptr_t)kc & 15) == 0 && ((uintptr_t)vc & 15) == 0, "attention4: caches start on 16-byte boundaries");
    PG_REQUIRE(((uintptr_t)p->d_part & 15) == 0 && ((uintptr_t)out & 1) == 0, "attention4: workspace on no 16-byte boundary, or output not aligned");
    PG_REQUIRE(ldo >= (int64_t)p->heads * p->vdim, "attention4: rows too short");
    PG_REQUIRE(p->kv_heads <= 65535 && batch->rows >= 0 && batch->seqs >= 0 && batch->seqs <= 65535, "attention4: too many heads or sequences");
    return PG_OK;
}

}  // namespace

extern "C" {

PG_API int64_t pg_cache4_bytes(int32_t width, int64_t positions)
{
    return width > 0 && positions > 0 ? pg_up(positions, 16) / 16 * pg_cache4_tile_bytes(pg_up(width, 32)) : 0;
}

PG_API int64_t pg_attention4_part_floats(pg_ctx *ctx, const pg_attention *p)
{
    // (slices only where there are no more CTAs than two per SM)
    return ctx && p && p->vdim > 0 ? (int64_t)2 * ctx->sm_count * 16 * (pg_up(p->vdim, 32) + 4) : 0;
}

PG_API int64_t pg_attention4_tickets(pg_ctx *ctx) { return ctx ? (int64_t)2 * ctx->sm_count + 1 : 0; }

PG_API int64_t pg_attention4_unfold_bytes(const pg_attention *p)
{
    if (!p || p->kv_heads <= 0 || p->cap <= 0 || p->chunk < 0) return 0;
    const int64_t chunks = p->chunk ? std::max(1, p->cap / p->chunk) : 1;
    return (int64_t)p->kv_heads * ((int64_t)p->cap * (pg_up(p->dim, 16) + pg_up(p->vdim, 16)) * 2 + 2 * ATTN_TOPS * 4 + pg_up(p->vdim, 32) / 32 * chunks * 4);
}

PG_API int32_t pg_attention4_run(pg_ctx *ctx, const pg_attention *p, const pg_batch *batch, int64_t few, int64_t short_rows, int64_t short_len, const float *d_proj,
                                 int64_t ldp, void *d_kcache, void *d_vcache, void *d_out, int32_t dtype, int64_t ldo)
{
    PG_ENTER(ctx);
    const int32_t rc = check(p, batch, d_kcache, d_vcache, d_out, dtype, ldo);
    if (rc != PG_OK) return rc;
    const AttnShape s = pgk_attention_shape(p);
    const Four f = four_of(s);
    PG_REQUIRE(d_proj && ldp >= (int64_t)(s.H + s.G) * s.D + (int64_t)s.G * s.V, "attention4: rows too short");
    PG_REQUIRE(((uintptr_t)d_proj & 3) == 0 && (((uintptr_t)p->d_q & 15) == 0 || short_rows == batch->rows), "attention4: rows or queries not aligned");
    PG_REQUIRE(few >= 0 && few <= 4096 && short_rows >= 0 && short_rows <= batch->rows && short_len >= 0 && short_len <= few && (short_len == 0) == (short_rows == 0),
               "attention4: %lld rows of up to %lld tokens among sequences of up to %lld", (long long)short_rows, (long long)short_len, (long long)few);
    PG_REQUIRE(s.chunk == 0 || few <= 1, "attention4: a chunked layer takes one token of a sequence here");
    if (batch->rows == 0) return PG_OK;
    unsigned char *kc = (unsigned char *)d_kcache, *vc = (unsigned char *)d_vcache;
    const bool fused = batch->max_len == 1 && few >= 1;
    if (!fused) {
        __half *q = short_rows < batch->rows ? (__half *)p->d_q : nullptr;
        float *q_up = (float *)((__half *)p->d_q + (int64_t)batch->rows * s.H * s.dp);
        const bool wide = s.D % 4 == 0 && s.V % 4 == 0 && ldp % 4 == 0 && ((uintptr_t)d_proj & 15) == 0;
        auto append = s.D <= 128 && s.V <= 128 ? (wide ? attn4_append_kernel<1, true> : attn4_append_kernel<1, false>)
                                               : (wide ? attn4_append_kernel<2, true> : attn4_append_kernel<2, false>);
        const int32_t ra = launch_pdl(ctx, append, dim3((unsigned)batch->rows), dim3(AP_WARPS * 32), 0, s, f, *batch, d_proj, ldp, q, q_up, kc, vc, ctx->d_status);
        if (ra != PG_OK || short_rows == 0) return ra;
    }
    const int64_t cols = (fused ? 1 : short_len) * s.rep;
    const int blocks = (int)((cols + 15) / 16);
    PG_REQUIRE((int64_t)s.G * blocks <= 65535, "attention4: too many heads");
    const bool hi = cols > 8;
    float *part = p->d_part;
    int32_t *tickets = p->d_tickets;
    bf16 *out = (bf16 *)d_out;
#define PG_A4(GK, GV, HI, EXACT)                                                                                                                              \
    do {                                                                                                                                                      \
        if (fused) return run_few<GK, GV, HI, true, EXACT>(ctx, s, f, batch, (int)few, blocks, d_proj, ldp, kc, vc, part, tickets, out, ldo);                 \
        return run_few<GK, GV, HI, false, EXACT>(ctx, s, f, batch, (int)few, blocks, d_proj, ldp, kc, vc, part, tickets, out, ldo);                           \
    } while (0)
#define PG_A4_HI(GK, GV, EXACT)             \
    do {                                    \
        if (hi) PG_A4(GK, GV, true, EXACT); \
        PG_A4(GK, GV, false, EXACT);        \
    } while (0)
    // (loops of a known length without a way out are half again as fast; the usual widths have them)
    if (f.gk == 2 && f.gv == 2) PG_A4_HI(2, 2, true);
    if (f.gk == 4 && f.gv == 4) PG_A4_HI(4, 4, true);
    if (f.gk <= 2 && f.gv <= 2) PG_A4_HI(2, 2, false);
    if (f.gk <= 4 && f.gv <= 4) PG_A4_HI(4, 4, false);
    PG_A4_HI(8, 8, false);
#undef PG_A4
#undef PG_A4_HI
}

PG_API int32_t pg_attention4_prompt(pg_ctx *ctx, const pg_attention *p, const pg_batch *batch, int64_t seq, int64_t len, int64_t positions, int64_t slot,
                                    const void *d_kcache, const void *d_vcache, void *d_work, void *d_out, int32_t dtype, int64_t ldo)
{
    PG_ENTER(ctx);
    const int32_t rc = check(p, batch, d_kcache, d_vcache, d_out, dtype, ldo);
    if (rc != PG_OK) return rc;
    AttnShape s = pgk_attention_shape(p);
    const Four f = four_of(s);
    PG_REQUIRE(((uintptr_t)p->d_q & 15) == 0, "attention4: queries on no 16-byte boundary");
    PG_REQUIRE(d_work && ((uintptr_t)d_work & 127) == 0, "attention4: no workspace, or not on a 128-byte boundary");
    PG_REQUIRE(seq >= 0 && seq < batch->seqs && len > 0 && len <= batch->max_len && positions >= len && positions <= s.limit && slot >= 0 && slot < p->slots,
               "attention4: sequence %lld with %lld tokens and %lld positions in slot %lld", (long long)seq, (long long)len, (long long)positions, (long long)slot);
    // the slot's rows that hold something, in the order that they have there
    const int rows = (int)std::min<int64_t>(positions, s.cap), padded = (int)std::min<int64_t>(rows + 128, s.cap);   // (a tile of keys may end behind them)
    __half *k = (__half *)d_work, *v = k + (int64_t)s.G * s.cap * s.dp;
    float *k_top = (float *)(v + (int64_t)s.G * s.cap * s.vp), *v_top = k_top + s.G * ATTN_TOPS;
    int *v_bad = (int *)(v_top + s.G * ATTN_TOPS);
    const int bad = f.gv * (s.chunk ? s.cap / s.chunk : 1);
    s.q_up = (const float *)((const __half *)p->d_q + (int64_t)batch->rows * s.H * s.dp), s.k_top = k_top, s.v_top = v_top, s.v_bad = v_bad;
    const unsigned char *kc = (const unsigned char *)d_kcache + slot * s.G * f.kh, *vc = (const unsigned char *)d_vcache + slot * s.G * f.vh;
    int32_t ru = launch_pdl(ctx, attn4_tops_kernel, dim3(ATTN_TOPS, (unsigned)s.G, 2), dim3(128), 0, kc, vc, f, rows, bad, k_top, v_top, v_bad, *batch, (int)seq,
                            (int)len, (int)positions, (int)slot, ctx->d_status);
    if (ru == PG_OK)
        ru = launch_pdl(ctx, attn4_unfold_kernel, dim3((unsigned)((padded + 15) / 16), (unsigned)s.G, 2), dim3(128), 0, s, f, kc, vc, rows, padded, k, v, v_bad);
    if (ru != PG_OK) return ru;
    // the sequence as a batch of its own, its cache in slot 0 (the last ticket is always zero)
    pg_batch one = *batch;
    one.seqs = 1;
    one.max_len = (int32_t)len;
    one.d_seq_row0 += seq;
    one.d_seq_slot = p->d_tickets + 2 * ctx->sm_count;
    bf16 *out = (bf16 *)d_out;
    const bf16 *q = (const bf16 *)p->d_q, *kh = (const bf16 *)k, *vh = (const bf16 *)v;   // (f16, which s says)
    if (pgk_attention_prompt_tc_supports(s, &one, 1, ldo, out)) return pgk_attention_prompt_tc(ctx, s, &one, 1, q, kh, vh, out, ldo);
    return pgk_attention_prompt(ctx, s, &one, q, kh, vh, out, ldo);
}

PG_API int32_t pg_cache4_read(pg_ctx *ctx, const void *d_cache, int32_t values, int32_t width, int64_t cap, int64_t parts, int64_t rows, float *d_out)
{
    PG_ENTER(ctx);
    PG_REQUIRE(d_cache && d_out && ((uintptr_t)d_cache & 15) == 0 && ((uintptr_t)d_out & 3) == 0, "cache4_read: null pointer, or not on a 16-byte boundary");
    PG_REQUIRE(width > 0 && width <= 256 && cap > 0 && parts > 0 && parts <= 65535 && rows > 0 && rows <= cap, "cache4_read: bad shape");
    const int w = (int)pg_up(width, 32), tile = (int)pg_cache4_tile_bytes(w);
    const dim3 grid((unsigned)((rows + 15) / 16), (unsigned)parts);
    const int64_t head = pg_up(cap, 16) / 16 * tile;
    auto kern = values ? attn4_read_kernel<true> : attn4_read_kernel<false>;
    return launch_whole(ctx, kern, grid, dim3(128), 0, (const unsigned char *)d_cache, w / 32, tile, head, (int)rows, d_out);
}

}  // extern "C"
