// Product y = act(a W^T) with weights of 4 bits (csrc/pg_linear4.cu) and many rows, on the 5th-generation tensor cores.
//
//   * The weights are the M side: 128 rows to a tile, their quants unpacked to f16 in TMEM, 64 k at a time, by four warps (a thread per row);
//     the activations are the N side, BN rows of f16 in shared memory by TMA.  scale * (q - 8) is an f16 number exactly (csrc/pg_linear4.cu), and
//     linear4_rows_kernel writes the activations as f16 divided by a power of two per row, which holds bf16 numbers exactly down to 2^-29 of the
//     row's largest: sums are those of the bf16 activations with the weights, in f32.
//   * Warps 0 .. 3 unpack, 4 .. 7 write outputs (lane = weight row, so a store is 32 columns of one row of y), 8 copies, 9 issues the products.
//     Two accumulators, so that outputs are written while the next tile is computed.
//   * Few tiles: K is divided over CTAs; raw sums go to slabs, the last warp of a 32-row band to finish adds them in a fixed order.
//   * ROUTED: BN rows belong to one expert; pieces of a 128-row block without a row are left out.
//
// Every mbarrier wait is bounded (pg_async.cuh).
#include <algorithm>

#include "pg_async.cuh"
#include "pg_four.cuh"
#include "pg_tcgen05.cuh"

namespace {

constexpr int T4_THREADS = 320;
constexpr int BM = 128;                 // weight rows of a tile
constexpr int W_BYTES = 8 * 512;        // quants of a tile and 64 k
constexpr int S_BYTES = 8 * 32 * 2;     // scales of them (groups of 32: two to 64 k)

template <int BN>
struct Cfg {
    static constexpr int X = BN * 128;
    static constexpr int STAGE = X + W_BYTES + 1024;
    static constexpr int ROOM = 227 * 1024 - 1024 - 512;
    static constexpr int STAGES = ROOM / STAGE > 12 ? 12 : ROOM / STAGE;
    static constexpr int A_SLOTS = BN > 128 ? 4 : 8;      // unpacked blocks of 64 k in TMEM, 32 columns each
    static constexpr int A_COL = 2 * BN;                  // behind the two accumulators
    static constexpr size_t SMEM = (size_t)STAGES * STAGE + 1024 + 512;
    static_assert(A_COL + 32 * A_SLOTS <= 512, "TMEM");
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap *tmap, uint32_t bar, int x, int y, int z, int w)
{
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(tmap),
                 "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
                 : "memory");
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// ---- rows of a as f16 over a power of two: a CTA per row ----------------------------------------------------------------
constexpr int RW_T = 256, RW_KEEP = 8;
__global__ void __launch_bounds__(RW_T)
    linear4_rows_kernel(const bf16 *__restrict__ a, int64_t lda, int k, const PgRouted rt, uint4 *__restrict__ out, float *__restrict__ back)
{
    __shared__ float red[8];
    pg_pdl_begin();
    const int64_t m = blockIdx.x;
    int64_t src = m;
    const bool routed = rt.blocks != nullptr;
    if (routed) {
        if (m >= (int64_t)__ldcg(rt.blocks) * PG_ROUTE_BLOCK) return;
        const int p = __ldcg(rt.row_pair + m);
        if (p < 0) {                                       // a row of zeros
            for (int i = threadIdx.x; i < k / 8; i += RW_T) out[m * (k / 8) + i] = make_uint4(0u, 0u, 0u, 0u);
            if (threadIdx.x == 0) back[m] = 1.0f;
            return;
        }
        if (rt.by_token) src = p / rt.top;
    }
    const uint4 *row = reinterpret_cast<const uint4 *>(a + src * lda);
    const int n = k / 8;
    uint4 keep[RW_KEEP];
    float top = 0.0f;
    auto look = [&](const uint4 &v) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; i++) top = fmaxf(top, fmaxf(fabsf(pg_bf16_lo(w[i])), fabsf(pg_bf16_hi(w[i]))));
    };
#pragma unroll
    for (int i = 0; i < RW_KEEP; i++) {
        const int at = threadIdx.x + i * RW_T;
        keep[i] = at < n ? __ldcg(row + at) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < RW_KEEP; i++) look(keep[i]);
    for (int at = threadIdx.x + RW_KEEP * RW_T; at < n; at += RW_T) look(__ldcg(row + at));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; i++) top = fmaxf(top, red[i]);
    float down, up;
    four_range(top, down, up);
    if (threadIdx.x == 0) back[m] = up;
    auto put = [&](int at, const uint4 &v) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = four_pack_f16(pg_bf16_lo(w[i]) * down, pg_bf16_hi(w[i]) * down);
        out[m * n + at] = make_uint4(o[0], o[1], o[2], o[3]);
    };
#pragma unroll
    for (int i = 0; i < RW_KEEP; i++)
        if (threadIdx.x + i * RW_T < n) put(threadIdx.x + i * RW_T, keep[i]);
    for (int at = threadIdx.x + RW_KEEP * RW_T; at < n; at += RW_T) put(at, __ldcg(row + at));
}

// How K is divided: parts of `blocks` 64-element blocks; slab of (unit, quarter): [BN][32 weight rows]
struct KParts {
    int parts, blocks;
    float *slabs;
    unsigned int *tickets;   // one per (tile, quarter), zero between calls
};

template <int BN, int ACT, typename TY>
__global__ void __launch_bounds__(T4_THREADS, 1)
    linear4_tc_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_s,
                      const float *__restrict__ wrow, const float *xback, int M, int N, int K, int group, int wtiles, float limit, TY *__restrict__ y, int64_t ldy,
                      const PgRouted rt, const KParts kp, int32_t *status, unsigned long long limit_ns)
{
    using C = Cfg<BN>;
    constexpr int STAGES = C::STAGES, SLOTS = C::A_SLOTS;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = pg_smem(smem_raw), base = (raw_addr + 1023u) & ~1023u;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem_raw + (base - raw_addr) + (size_t)STAGES * C::STAGE);
    const uint32_t bar_full = pg_smem(bars), bar_empty = bar_full + 8 * STAGES, bar_afull = bar_empty + 8 * STAGES, bar_aempty = bar_afull + 8 * SLOTS,
                   bar_tfull = bar_aempty + 8 * SLOTS, bar_tempty = bar_tfull + 16;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * STAGES + 2 * SLOTS + 4);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    static_assert((2 * STAGES + 2 * SLOTS + 5) * 8 <= 512, "barriers");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) {
            pg_mbar_init(bar_full + 8 * s, 1);
            pg_mbar_init(bar_empty + 8 * s, 1);
        }
        for (int s = 0; s < SLOTS; s++) {
            pg_mbar_init(bar_afull + 8 * s, 4);            // one arrival per unpacking warp
            pg_mbar_init(bar_aempty + 8 * s, 1);
        }
        for (int i = 0; i < 2; i++) {
            pg_mbar_init(bar_tfull + 8 * i, 1);
            pg_mbar_init(bar_tempty + 8 * i, 4);           // one arrival per output warp
        }
        *abort_flag = 0;
        pg_mbar_fence();
    }
    __syncwarp();
    if (warp == 9) tmem_alloc<1>(pg_smem(tmem_slot), 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const bool routed = rt.blocks != nullptr;
    if (routed) asm volatile("griddepcontrol.wait;" ::: "memory");   // the list of tiles comes from the preceding kernels
    const int tiles_m = routed ? __ldcg(rt.blocks) * (PG_ROUTE_BLOCK / BN) : (M + BN - 1) / BN;
    const int tiles_n = (N + BM - 1) / BM;
    const int sp = kp.parts, total = tiles_m * tiles_n * sp;   // unit u: part u % sp of tile u / sp
    const int kblocks = K / 64;
    const int rows = routed ? tiles_m * BN : M;
    auto k_first = [&](int u) { return (u % sp) * kp.blocks; };
    auto k_end = [&](int u) { return min(kblocks, (u % sp + 1) * kp.blocks); };
    // a piece of a route's block that has no row (they are filled from the first on)
    auto nothing = [&](int u) { return routed && __ldcg(rt.row_pair + (int64_t)(u / sp % tiles_m) * BN) < 0; };
    const int gs = group == 32 ? 2 : 1;                    // scales of a row to 64 k
    const uint32_t stage_bytes = (uint32_t)(C::X + W_BYTES + 8 * 32 * gs);

    if (warp == 8) {
        // ---------------------------------------------------------------- copies
        if (lane == 0) {
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            auto weights = [&](uint32_t at, uint32_t bar, int kb, int tile) {
                const int mt = tile % tiles_m, wt = (routed ? __ldcg(rt.block_expert + mt / (PG_ROUTE_BLOCK / BN)) * wtiles : 0) + tile / tiles_m * (BM / 16);
                pg_mbar_expect(bar, stage_bytes);
                tma_load_4d(at + C::X, &map_w, bar, 0, 0, kb, wt);
                tma_load_3d(at + C::X + W_BYTES, &map_s, bar, 0, kb * 64 / group, wt);
            };
            int early = 0;
            if (!routed) {
                if ((int)blockIdx.x < total) {
                    const int u = blockIdx.x, first = k_first(u);
                    early = min(k_end(u) - first, STAGES);
                    for (int i = 0; i < early; i++) weights(base + i * C::STAGE, bar_full + 8 * i, first + i, u / sp);
                }
                asm volatile("griddepcontrol.wait;" ::: "memory");
            }
            for (int u = blockIdx.x; ok && u < total; u += gridDim.x) {
                if (nothing(u)) continue;
                const int tile = u / sp, m0 = tile % tiles_m * BN;
                for (int kb = k_first(u), end = k_end(u); kb < end; kb++) {
                    if (!(ok = pg_mbar_wait(bar_empty + 8 * stage, phase ^ 1, abort_flag, status, limit_ns))) break;
                    const uint32_t at = base + stage * C::STAGE;
                    if (early > 0)
                        early--;
                    else
                        weights(at, bar_full + 8 * stage, kb, tile);
                    tma_load_2d(at, &map_x, bar_full + 8 * stage, kb * 64, m0);
                    if (++stage == STAGES) stage = 0, phase ^= 1;
                }
            }
            if (!ok) {
                // give copies that are still in flight a bounded time to land before the CTA exits
                const unsigned long long t0 = pg_globaltimer_ns();
                while (pg_globaltimer_ns() - t0 < 2000000ull) {
                }
            }
        }
    } else if (warp == 9) {
        // ---------------------------------------------------------------- products (the whole warp; one lane's count)
        const uint32_t on = pg_elect();
        constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);   // f16 operands, f32 sums
        uint32_t stage = 0, phase = 0, slot = 0, aphase = 0, acc = 0, acc_phase = 0;
        bool ok = true;
        for (int u = blockIdx.x; ok && u < total; u += gridDim.x) {
            if (nothing(u)) continue;
            if (!(ok = pg_mbar_wait_warp(bar_tempty + 8 * acc, acc_phase ^ 1, abort_flag, status, limit_ns))) break;
            tc_fence_after();
            const uint32_t d = tmem + acc * BN;
            const int first = k_first(u), end = k_end(u);
            for (int kb = first; kb < end; kb++) {
                if (!(ok = pg_mbar_wait_warp(bar_full + 8 * stage, phase, abort_flag, status, limit_ns))) break;
                if (!(ok = pg_mbar_wait_warp(bar_afull + 8 * slot, aphase, abort_flag, status, limit_ns))) break;
                tc_fence_after();
                const uint64_t db = make_smem_desc(base + stage * C::STAGE);
                const uint32_t ta = tmem + C::A_COL + slot * 32;
#pragma unroll
                for (int j = 0; j < 4; j++) umma_f16_ta(d, ta + j * 8, db + (uint64_t)(j * 2), idesc, kb != first || j != 0 ? 1u : 0u, on);
                umma_commit(bar_empty + 8 * stage, on);
                umma_commit(bar_aempty + 8 * slot, on);
                if (++stage == STAGES) stage = 0, phase ^= 1;
                if (++slot == SLOTS) slot = 0, aphase ^= 1;
            }
            if (!ok) break;
            umma_commit(bar_tfull + 8 * acc, on);
            if (++acc == 2) acc = 0, acc_phase ^= 1;
        }
    } else if (warp < 4) {
        // ---------------------------------------------------------------- quants -> f16 in TMEM: a thread per weight row
        const int ti = 2 * warp + (lane >> 4), rr = lane & 15;
        const uint32_t off = (uint32_t)(ti * 512 + (rr & 7) * 64), swz = (off >> 7 & 7u) << 4;   // (bits 7 .. 9 do not change over the row's 64 bytes)
        const uint32_t mask = rr < 8 ? FOUR_LO : FOUR_HI, sub = rr < 8 ? FOUR_OFF_LO : FOUR_OFF_HI;
        const uint32_t less = rr < 8 ? 0x3c003c00u : 0x2c002c00u;     // 1, and 1 / 16
        uint32_t stage = 0, phase = 0, slot = 0, aphase = 0;
        bool ok = true;
        for (int u = blockIdx.x; ok && u < total; u += gridDim.x) {
            if (nothing(u)) continue;
            for (int kb = k_first(u), end = k_end(u); kb < end; kb++) {
                if (!(ok = pg_mbar_wait_warp(bar_full + 8 * stage, phase, abort_flag, status, limit_ns))) break;
                const uint32_t at = base + stage * C::STAGE + C::X;
                uint4 q[4];
#pragma unroll
                for (int i = 0; i < 4; i++) q[i] = pg_lds128(at + ((off + i * 16) ^ swz));
                uint32_t sc[2];
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    unsigned short h;
                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(at + W_BYTES + (uint32_t)((ti * gs + (gs == 2 ? c : 0)) * 32 + rr * 2)));
                    sc[c] = mul_f16x2((uint32_t)h * 0x10001u, less);
                }
                uint32_t v[32];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const int to = 16 * (j >> 1) + 4 * i + 2 * (j & 1);
                        v[to] = mul_f16x2(four_sub_f16(four_lop(w[j], mask, FOUR_F16), sub), sc[j >> 1]);
                        v[to + 1] = mul_f16x2(four_sub_f16(four_lop(w[j] >> 8, mask, FOUR_F16), sub), sc[j >> 1]);
                    }
                }
                if (!(ok = pg_mbar_wait_warp(bar_aempty + 8 * slot, aphase ^ 1, abort_flag, status, limit_ns))) break;
                tc_fence_after();
                tmem_st32(tmem + ((uint32_t)(warp * 32) << 16) + C::A_COL + slot * 32, v);
                tmem_wait_st();
                tc_fence_before();
                pg_mbar_arrive_warp(bar_afull + 8 * slot, lane);
                if (++stage == STAGES) stage = 0, phase ^= 1;
                if (++slot == SLOTS) slot = 0, aphase ^= 1;
            }
        }
    } else {
        // ---------------------------------------------------------------- outputs
        const int q = warp & 3;
        if (!routed) asm volatile("griddepcontrol.wait;" ::: "memory");   // y may still be read by the predecessor; xback is its work
        uint32_t acc = 0, acc_phase = 0;
        bool ok = true;
        for (int u = blockIdx.x; ok && u < total; u += gridDim.x) {
            if (nothing(u)) continue;
            const int tile = u / sp, mt = tile % tiles_m, m0 = mt * BN, n0 = tile / tiles_m * BM + q * 32;
            const int64_t wt = (routed ? (int64_t)__ldcg(rt.block_expert + mt / (PG_ROUTE_BLOCK / BN)) * wtiles : 0) + n0 / 16;
            const float fac = n0 + lane < wtiles * 16 ? __ldg(wrow + wt * 16 + lane) : 0.0f;
            if (!(ok = pg_mbar_wait_warp(bar_tfull + 8 * acc, acc_phase, abort_flag, status, limit_ns))) break;
            tc_fence_after();
            // sums of weight row n0 + lane with rows m0 + c .. of a
            auto put = [&](const uint32_t (&v)[32], int c) {
                const int m = m0 + c, left = rows - m;
                const float xb = lane < left ? __ldcg(xback + m + lane) : 0.0f;
                if constexpr (ACT != PG_ACT_NONE) {
                    // lanes l and l ^ 8 have a gate and its up: the gate's lane takes the even rows, the other the odd ones
                    const bool up = lane & 8;
                    TY *dst = y + (int64_t)m * ldy + n0 / 2 + (lane >> 4) * 8 + (lane & 7);
#pragma unroll
                    for (int j = 0; j < 32; j += 2) {
                        const float b0 = __shfl_sync(0xffffffffu, xb, j), b1 = __shfl_sync(0xffffffffu, xb, j + 1);
                        const float v0 = __uint_as_float(v[j]) * fac * b0, v1 = __uint_as_float(v[j + 1]) * fac * b1;
                        const float other = __shfl_xor_sync(0xffffffffu, up ? v0 : v1, 8);
                        const float o = up ? pg_glu<ACT>(other, v1, limit) : pg_glu<ACT>(v0, other, limit);
                        const int jj = up ? j + 1 : j;
                        if (jj < left && n0 + lane < N) pg_put(dst + (int64_t)jj * ldy, o);
                    }
                } else {
                    TY *dst = y + (int64_t)m * ldy + n0 + lane;
#pragma unroll
                    for (int j = 0; j < 32; j++) {
                        const float b = __shfl_sync(0xffffffffu, xb, j);
                        if (j < left && n0 + lane < N) pg_put(dst + (int64_t)j * ldy, __uint_as_float(v[j]) * fac * b);
                    }
                }
            };
#pragma unroll 1
            for (int c = 0; c < BN; c += 32) {
                if (m0 + c >= rows || n0 >= N) break;         // uniform over the warp
                uint32_t v[32];
                tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + acc * BN + c, v);
                if (sp > 1) {
                    float *slab = kp.slabs + (((int64_t)u * 4 + q) * BN + c) * 32 + lane;
#pragma unroll
                    for (int j = 0; j < 32; j++) __stcg(slab + j * 32, __uint_as_float(v[j]));
                } else {
                    put(v, c);
                }
            }
            tc_fence_before();
            pg_mbar_arrive_warp(bar_tempty + 8 * acc, lane);
            if (sp > 1 && n0 < N) {
                unsigned int *ticket = kp.tickets + tile * 4 + q;
                __threadfence();
                __syncwarp();
                const unsigned int before = __shfl_sync(0xffffffffu, lane == 0 ? atomicAdd(ticket, 1u) : 0u, 0);
                if (before == (unsigned)(sp - 1)) {
                    __threadfence();
                    if (lane == 0) *ticket = 0;
#pragma unroll 1
                    for (int c = 0; c < BN; c += 32) {
                        if (m0 + c >= rows) break;
                        const float *slab = kp.slabs + (((int64_t)tile * sp * 4 + q) * BN + c) * 32 + lane;
                        float sum[32];
#pragma unroll
                        for (int j = 0; j < 32; j++) sum[j] = __ldcg(slab + j * 32);
                        for (int p = 1; p < sp; p++) {
                            const float *at = slab + (int64_t)p * 4 * BN * 32;
                            float b[32];
#pragma unroll
                            for (int j = 0; j < 32; j++) b[j] = __ldcg(at + j * 32);
#pragma unroll
                            for (int j = 0; j < 32; j++) sum[j] += b[j];
                        }
                        uint32_t v[32];
#pragma unroll
                        for (int j = 0; j < 32; j++) v[j] = __float_as_uint(sum[j]);
                        put(v, c);
                    }
                }
            }
            if (++acc == 2) acc = 0, acc_phase ^= 1;
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc<1>(tmem, 512);
    }
}

// ---------------------------------------------------------------- host side ----
constexpr int SLAB_ROWS = 256;         // rows of slabs (128 weight rows each) per SM, at most

template <int BN, int ACT, typename TY>
int32_t launch(pg_ctx *ctx, const pg_linear4 *lin, const void *x, const float *xback, int64_t m, float limit, TY *y, int64_t ldy, const PgRouted &rt, KParts kp)
{
    using C = Cfg<BN>;
    CUtensorMap mx, mw, ms;
    const cuuint64_t xd[2] = {(cuuint64_t)lin->k, (cuuint64_t)m}, xs[1] = {(cuuint64_t)lin->k * 2};
    const cuuint32_t xb[2] = {64, (cuuint32_t)BN};
    int32_t rc = pg_encode_map(&mx, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, x, 2, xd, xs, xb);
    if (rc) return rc;
    const cuuint64_t tiles = (cuuint64_t)(lin->experts * lin->tiles), kb = (cuuint64_t)(lin->k / 64), kg = (cuuint64_t)(lin->k / lin->group);
    const cuuint64_t wd[4] = {32, 4, kb, tiles}, wst[3] = {128, 512, kb * 512};
    const cuuint32_t wb[4] = {32, 4, 1, 8};
    rc = pg_encode_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT32, lin->q, 4, wd, wst, wb);
    if (rc) return rc;
    const cuuint64_t sd[3] = {16, kg, tiles}, sst[2] = {32, kg * 32};
    const cuuint32_t sb[3] = {16, lin->group == 32 ? 2u : 1u, 8};
    rc = pg_encode_map(&ms, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, lin->s, 3, sd, sst, sb, CU_TENSOR_MAP_SWIZZLE_NONE);
    if (rc) return rc;
    auto kern = linear4_tc_kernel<BN, ACT, TY>;
    static std::atomic<uint64_t> set{0};
    PG_CUDA(pg_max_smem_once(kern, (int)C::SMEM, ctx->device, set));
    const int64_t units = ((m + BN - 1) / BN) * ((lin->n + BM - 1) / BM) * kp.parts;
    PG_REQUIRE(units < (1ll << 31) - 65536, "linear4: too many tiles");
    kp.tickets = reinterpret_cast<unsigned int *>(ctx->splitk);
    kp.slabs = reinterpret_cast<float *>(reinterpret_cast<unsigned char *>(ctx->splitk) + PG_LM_TICKET_BYTES);
    return launch_pdl(ctx, kern, dim3((unsigned)std::min<int64_t>(units, ctx->sm_count)), dim3(T4_THREADS), C::SMEM, mx, mw, ms, lin->row, xback, (int)m, (int)lin->n,
                      (int)lin->k, (int)lin->group, (int)lin->tiles, limit, y, ldy, rt, kp, ctx->d_status, ctx->wait_limit_ns);
}

template <int ACT, typename TY>
int32_t dispatch(pg_ctx *ctx, const pg_linear4 *lin, const void *x, const float *xback, int64_t m, float limit, TY *y, int64_t ldy, const PgRouted &rt, int64_t pairs)
{
    const int kblocks = (int)(lin->k / 64);
    const int64_t tiles_n = (lin->n + BM - 1) / BM;
    KParts kp = {1, kblocks, nullptr, nullptr};
    int bn = 128;
    if (rt.blocks) {
        // rows an expert has on average
        const int64_t rows = (pairs + lin->experts - 1) / lin->experts;
        bn = rows <= 24 ? 32 : rows <= 48 ? 64 : 128;
    } else {
        // cycles of a block of 64 k: its products (2 BN), the unpacking, and its bytes at what L2 gives an SM; of a unit: its outputs
        double best = 1e30;
        for (int cand : {32, 64, 128, 192}) {
            const int64_t tiles = ((m + cand - 1) / cand) * tiles_n;
            const double block = std::max({2.0 * cand, 190.0, (4600.0 + 128.0 * cand) / 60.0});
            for (int parts = 1; parts <= std::min(16, kblocks / 4 > 0 ? kblocks / 4 : 1); parts++) {
                const int blocks = (kblocks + parts - 1) / parts, real = (kblocks + blocks - 1) / blocks;
                if (real != parts) continue;
                if (parts > 1 && (tiles * parts * cand > (int64_t)ctx->sm_count * SLAB_ROWS || tiles > 4096)) break;
                const int64_t rounds = (tiles * parts + ctx->sm_count - 1) / ctx->sm_count;
                const double time = rounds * (blocks * block + (parts > 1 ? 300 + 8.0 * cand : 0)) + 1000 + 20.0 * cand + (parts > 1 ? 1500 + parts * 8.0 * cand : 0);
                if (time < best) {
                    best = time;
                    bn = cand;
                    kp.parts = parts;
                    kp.blocks = blocks;
                }
            }
        }
    }
    if (kp.parts > 1) {
        const int32_t rc = pg_splitk_reserve(ctx, pgk_linear4_tc_workspace(ctx));
        if (rc != PG_OK) return rc;
    }
    if (bn == 192) return launch<192, ACT, TY>(ctx, lin, x, xback, m, limit, y, ldy, rt, kp);
    if (bn == 128) return launch<128, ACT, TY>(ctx, lin, x, xback, m, limit, y, ldy, rt, kp);
    if (bn == 64) return launch<64, ACT, TY>(ctx, lin, x, xback, m, limit, y, ldy, rt, kp);
    return launch<32, ACT, TY>(ctx, lin, x, xback, m, limit, y, ldy, rt, kp);
}

}  // namespace

size_t pgk_linear4_tc_workspace(const pg_ctx *ctx) { return PG_LM_TICKET_BYTES + (size_t)ctx->sm_count * SLAB_ROWS * BM * sizeof(float); }

int32_t pgk_linear4_tc(pg_ctx *ctx, const pg_linear4 *lin, const bf16 *a, int64_t lda, int64_t m, int act, float limit, void *y, int y_dtype, int64_t ldy,
                       const PgRouted *routed, int64_t pairs)
{
    static const PgRouted no_route = {};
    const PgRouted &rt = routed ? *routed : no_route;
    const size_t xbytes = (size_t)m * lin->k * 2;
    int32_t rc = pg_scratch_reserve_recording(ctx, xbytes + (size_t)m * sizeof(float));
    if (rc != PG_OK) return rc;
    float *back = reinterpret_cast<float *>((unsigned char *)ctx->scratch + xbytes);
    rc = launch_pdl(ctx, linear4_rows_kernel, dim3((unsigned)m), dim3(RW_T), 0, a, lda, (int)lin->k, rt, (uint4 *)ctx->scratch, back);
    if (rc != PG_OK) return rc;
    if (act == PG_ACT_GELU_TANH_GLU) return dispatch<PG_ACT_GELU_TANH_GLU, bf16>(ctx, lin, ctx->scratch, back, m, limit, (bf16 *)y, ldy, rt, pairs);
    if (act == PG_ACT_CLAMPED_SWISH_GLU) return dispatch<PG_ACT_CLAMPED_SWISH_GLU, bf16>(ctx, lin, ctx->scratch, back, m, limit, (bf16 *)y, ldy, rt, pairs);
    if (y_dtype == PG_BF16) return dispatch<PG_ACT_NONE, bf16>(ctx, lin, ctx->scratch, back, m, limit, (bf16 *)y, ldy, rt, pairs);
    return dispatch<PG_ACT_NONE, float>(ctx, lin, ctx->scratch, back, m, limit, (float *)y, ldy, rt, pairs);
}
