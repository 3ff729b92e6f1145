// Product y = act(a W^T) with weights of 4 bits (csrc/pg_linear4.cu) and many rows, on the 5th-generation tensor cores.
//
//   * The weights are the M side: a pair of CTAs has 256 rows, each unpacks its 128 to f16 in TMEM, 128 k at a time (a thread per row, two or three
//     teams of four warps that take the blocks in turn, two blocks of TMEM each); the activations are the N side, BN rows of f16 in shared memory by TMA, half in each CTA.
//     scale * (q - 8) is an f16 number exactly (csrc/pg_linear4.cu), and linear4_rows_kernel writes the activations as f16 divided by a power of two
//     per row, which holds bf16 numbers exactly down to 2^-31 of the row's largest: sums are those of the bf16 activations with the weights.
//   * An accumulator sums up 512 k; eight warps add the accumulators up in f32 registers.  (The tensor cores cut sums off: 4096 k in one
//     accumulator were 3.9e-6 off 64 bits, 512 at a time 6e-7.)  They write the outputs: lane = weight row, so a store is 32 columns of one row of y.
//   * Where whole tiles would leave SMs idle, the tiles' blocks of 128 k are divided evenly over the pairs of CTAs; sums of a tile that several share
//     go to slabs, and the last warp to finish adds them in a fixed order.
//   * With a route BN rows belong to one expert; pieces of a 128-row block without a row are left out.
//   * What bounds it: up to some 100 rows the unpacking, 830 cycles for a block of 128 x 128 where its products at BN = 128 are 512 (its steps' latency: more
//     teams were no faster), and what a call costs besides, some 10 us (rows_kernel 3, first weights 3.5, slabs and outputs 3, pair and TMEM 1.5).
//     2048 rows of 28672 x 4096: 430 us, 1.12 PFLOP/s of 1.68, the power cap included.
//
// Every mbarrier wait is bounded (pg_async.cuh).
#include <algorithm>

#include "pg_async.cuh"
#include "pg_four.cuh"
#include "pg_tcgen05.cuh"

namespace {

constexpr int BM = 128;                 // weight rows of a CTA's tile
constexpr int BK = 128;                 // columns of K in a block (the last one may have 64)
constexpr int CHUNK = 4;                // blocks that one accumulator sums up
constexpr int CG = 2;                   // CTAs of a pair
constexpr int W_COPY = 0, W_MMA = 1, W_WEIGHTS = 2, W_UNPACK = 4;   // warps: activations, products, weights (two), then the unpacking ones, eight for the outputs
constexpr int W_BLOCK = 16 * 576;       // bytes of a CTA's weights of a block, at most

template <int BN>
struct Cfg {
    static constexpr int TEAMS = BN > 64 ? 2 : 3;         // of unpacking warps, four warps each; they take the blocks in turn
    static constexpr int SLOTS = 2 * TEAMS;               // blocks in flight: activations in shared memory, unpacked weights in TMEM (64 columns each)
    static constexpr int OUT = W_UNPACK + 4 * TEAMS, THREADS = (OUT + 8) * 32;
    static constexpr int DEPTH = 7;                       // entries of the weights' ring, two blocks each
    static constexpr int RING = DEPTH * 2 * W_BLOCK;
    static constexpr int XT = BN / CG * 128;              // 64 columns of a block of the activations, a CTA's half
    static constexpr int A_COL = 2 * BN;                  // behind the two accumulators
    static constexpr size_t SMEM = (size_t)SLOTS * 2 * XT + RING + 1024 + (2 * SLOTS + 5 + 2 * DEPTH) * 8;
    static constexpr int COLS = BN >= 64 ? BN / 2 : BN;   // accumulator columns of an output warp
    // registers of a lane where the output warps' sums need more than an equal share: 20 x 96 of them, divided
    static constexpr int R_UNPACK = 80, R_OUT = 128, R_REST = 64;
    static constexpr bool SHARES = COLS >= 64;
    static_assert(!SHARES || 4 * TEAMS * R_UNPACK + 8 * R_OUT + 4 * R_REST == (OUT + 8) * 96, "no more registers than there are");
    static_assert(BN % 32 == 0 && BN >= 32 && BN <= 256, "a pair's products with the weights in TMEM take rows in steps of 32");
    static_assert(A_COL + 64 * SLOTS <= 512 && SMEM <= 227 * 1024, "TMEM, shared memory");
};

__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// ---- rows of a as f16 over a power of two: a CTA per row of a.  With a route: to the rows of the token's pairs, or (by_token == 0) per pair; rows
// without a pair keep what is there, and nobody reads their outputs -----------------------------------------------------------------
constexpr int RW_KEEP = 4;
template <int RW_T>
__global__ void __launch_bounds__(RW_T)
    linear4_rows_kernel(const bf16 *__restrict__ a, int64_t lda, int k, const PgRouted rt, const int32_t *pair_row, uint4 *__restrict__ out, float *__restrict__ back)
{
    __shared__ float red[RW_T / 32];
    pg_pdl_begin();
    int64_t src = blockIdx.x, to = src;
    if (pair_row && !rt.by_token) {
        src = to = __ldcg(pair_row + src);
        if (to < 0) return;
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
#pragma unroll 4
    for (int at = threadIdx.x + RW_KEEP * RW_T; at < n; at += RW_T) look(__ldcg(row + at));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < RW_T / 32; i++) top = fmaxf(top, red[i]);
    float down, up;
    four_range(top, down, up);
    auto f16 = [&](const uint4 &v) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        uint32_t o[4];
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = four_pack_f16(pg_bf16_lo(w[i]) * down, pg_bf16_hi(w[i]) * down);
        return make_uint4(o[0], o[1], o[2], o[3]);
    };
#pragma unroll
    for (int i = 0; i < RW_KEEP; i++) keep[i] = f16(keep[i]);
    const int copies = pair_row && rt.by_token ? rt.top : 1;
    for (int c = 0; c < copies; c++) {
        if (pair_row && rt.by_token) to = __ldcg(pair_row + src * rt.top + c);
        if (to < 0) continue;
        if (threadIdx.x == 0) back[to] = up;
#pragma unroll
        for (int i = 0; i < RW_KEEP; i++)
            if (threadIdx.x + i * RW_T < n) out[to * n + threadIdx.x + i * RW_T] = keep[i];
        for (int at = threadIdx.x + RW_KEEP * RW_T; at < n; at += RW_T) out[to * n + at] = f16(__ldcg(row + at));
    }
}

// How the work is divided.  blocks > 0: the tiles' blocks of 64 k, tile after tile, in stretches of `blocks`, one per pair of CTAs; a tile that several
// pairs share is put together from slabs, [COLS][32 weight rows] for every (CTA, whether it is the first or the last of its stretch, output warp).
// blocks == 0: whole tiles in turn.
struct Share {
    int blocks;
    float *slabs;
    unsigned int *tickets;   // one per (tile, CTA of the pair, output warp), zero between calls
};
// a piece of a tile: blocks k0 .. k1 of 64 k
struct Piece {
    int tile, k0, k1, expert;
};
constexpr int LIST = 192;               // pieces of a route that a pair looks up before it begins

// A warp's sums of weight rows n0 + lane with rows m0 .. of a (`left` of them exist) -> outputs
template <int COLS, bool ALL, typename TY>
__device__ __forceinline__ void put_rows(const float (&v)[COLS], float fac, const float (&xback)[COLS / 16], int left, bool in, TY *dst, int64_t ldy)
{
#pragma unroll
    for (int c = 0; c < COLS; c += 16) {
        if (!ALL && c >= left) break;                      // uniform over the warp
        const float xb = xback[c / 16];
#pragma unroll
        for (int j = 0; j < 16; j++) {
            const float o = v[c + j] * fac * __shfl_sync(0xffffffffu, xb, j);
            if ((ALL || c + j < left) && in) pg_put(dst, o);
            dst += ldy;
        }
    }
}
template <int COLS, int ACT, typename TY>
__device__ __forceinline__ void put(const float (&v)[COLS], float fac, const float (&xback)[COLS / 16], int m0, int left, int n0, int N, float limit, TY *y, int64_t ldy,
                                    int lane)
{
    const bool in = n0 + lane < N;
    if constexpr (ACT == PG_ACT_NONE) {
        TY *dst = y + (int64_t)m0 * ldy + n0 + lane;
        if (left >= COLS)
            put_rows<COLS, true>(v, fac, xback, left, in, dst, ldy);
        else
            put_rows<COLS, false>(v, fac, xback, left, in, dst, ldy);
    } else {
        // lanes l and l ^ 8 have a gate and its up: the gate's lane takes the even rows, the other the odd ones
        const bool up = lane & 8;
        TY *dst = y + (int64_t)(m0 + (up ? 1 : 0)) * ldy + n0 / 2 + (lane >> 4) * 8 + (lane & 7);
#pragma unroll
        for (int c = 0; c < COLS; c += 16) {
            if (c >= left) break;                          // uniform over the warp
            const float xb = xback[c / 16];
#pragma unroll
            for (int j = 0; j < 16; j += 2) {
                const float v0 = v[c + j] * fac * __shfl_sync(0xffffffffu, xb, j), v1 = v[c + j + 1] * fac * __shfl_sync(0xffffffffu, xb, j + 1);
                const float other = __shfl_xor_sync(0xffffffffu, up ? v0 : v1, 8);
                const float o = pg_glu<ACT>(up ? other : v0, up ? v1 : other, limit);
                if (c + j + (up ? 1 : 0) < left && in) pg_put(dst, o);
                dst += 2 * ldy;
            }
        }
    }
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]),
          "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
    tmem_wait_ld();
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(v[0]), "r"(v[1]),
                 "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]),
                 "r"(v[15]), "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ uint2 lds64(uint32_t addr)
{
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}
template <int N>
__device__ __forceinline__ void set_regs_less()
{
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void set_regs_more()
{
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

template <int BN, int ACT, typename TY>
__global__ void __launch_bounds__(Cfg<BN>::THREADS, 1)
    linear4_tc_kernel(const __grid_constant__ CUtensorMap map_x, const unsigned char *__restrict__ w, const float *__restrict__ wrow, const float *xback, int M, int N,
                      int K, int record, int wtiles, int alltiles, float limit, TY *__restrict__ y, int64_t ldy, const PgRouted rt, const Share sh, int32_t *status,
                      unsigned long long limit_ns)
{
    using C = Cfg<BN>;
    constexpr int COLS = C::COLS, TEAMS = C::TEAMS, SLOTS = C::SLOTS, DEPTH = C::DEPTH, RING = C::RING, W_OUT = C::OUT;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw_addr = pg_smem(smem_raw), base = (raw_addr + 1023u) & ~1023u;
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem_raw + (base - raw_addr) + SLOTS * 2 * C::XT + RING);
    const uint32_t bar_full = pg_smem(bars), bar_free = bar_full + 8 * SLOTS, bar_tfull = bar_free + 8 * SLOTS, bar_tempty = bar_tfull + 16,
                   bar_w = bar_tempty + 16, bar_read = bar_w + 8 * DEPTH;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * SLOTS + 4 + 2 * DEPTH);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);
    // (a shuffle's result is known to be the same in the whole warp: what follows from it stays in uniform registers)
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31, rank = __shfl_sync(0xffffffffu, (int)pg_cluster_rank(), 0);
    constexpr int OUT_WARPS = BN >= 64 ? 8 : 4;           // that have columns
    if (threadIdx.x == 0) {
        for (int s = 0; s < SLOTS; s++) {
            pg_mbar_init(bar_full + 8 * s, 4 * CG + 1);    // the warps of both CTAs' teams, and the copies of the activations
            pg_mbar_init(bar_free + 8 * s, 1);
        }
        for (int i = 0; i < 2; i++) {
            pg_mbar_init(bar_tfull + 8 * i, 1);
            pg_mbar_init(bar_tempty + 8 * i, OUT_WARPS * CG);
        }
        for (int i = 0; i < DEPTH; i++) {
            pg_mbar_init(bar_w + 8 * i, 1);
            pg_mbar_init(bar_read + 8 * i, 8);             // the warps of a team, for each of two blocks
        }
        *abort_flag = 0;
        pg_mbar_fence();
    }
    // A route's tiles of this pair and their experts, once for all warps.  (Looked up by every role where its tile begins: 777 tokens on 64 experts, gate and
    // up 95.6 us instead of 93.5, down 63.7 instead of 59.9.)
    __shared__ int list_tile[LIST], list_expert[LIST], list_n;
    const bool routed = rt.blocks != nullptr;
    constexpr int PER_BLOCK = PG_ROUTE_BLOCK / BN;
    const int tiles_n = (N + CG * BM - 1) / (CG * BM), unit0 = blockIdx.x / CG, units = gridDim.x / CG;
    if (routed && warp == W_UNPACK) {
        asm volatile("griddepcontrol.wait;" ::: "memory");   // the list of tiles comes from the preceding kernels
        const int across = __ldcg(rt.blocks) * PER_BLOCK, all = across * tiles_n;
        int n = 0;
        for (int64_t at = unit0 + (int64_t)lane * units; __any_sync(0xffffffffu, at < all); at += 32 * (int64_t)units) {
            // a piece of a route's block that has no row is left out (they are filled from the first on)
            const int m = at < all ? (int)(at % across) : 0;
            const bool there = at < all && __ldcg(rt.row_pair + (int64_t)m * BN) >= 0;
            const int e = there ? __ldcg(rt.block_expert + m / PER_BLOCK) : 0;
            const uint32_t which = __ballot_sync(0xffffffffu, there);
            const int to = n + __popc(which & ((1u << lane) - 1u));
            if (there && to < LIST) list_tile[to] = (int)at, list_expert[to] = e;
            n += __popc(which);
        }
        if (lane == 0) list_n = n;
    }
    __syncthreads();
    if (warp == W_MMA) tmem_alloc<CG>(pg_smem(tmem_slot), 512);
    tc_fence_before();
    // (the warps that bring weights need neither the other CTA nor TMEM: they wait at their end)
    const bool early = warp >= W_WEIGHTS && warp < W_UNPACK;
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    if (!early) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    tc_fence_after();
    const uint32_t tmem = early ? 0u : __shfl_sync(0xffffffffu, *tmem_slot, 0);
    if (routed) asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tiles_m = routed ? __shfl_sync(0xffffffffu, __ldcg(rt.blocks), 0) * PER_BLOCK : (M + BN - 1) / BN;
    const int total = tiles_m * tiles_n, kblocks = (K + BK - 1) / BK;
    const int rows = routed ? tiles_m * BN : M;
    const bool listed = routed && list_n <= LIST;
    // (longer lists are read where they are)
    auto nothing = [&](int tile) { return routed && __ldcg(rt.row_pair + (int64_t)(tile % tiles_m) * BN) < 0; };
    // the pieces of this pair, in their order; at: block (or tile, or entry of the list) that comes next
    const int64_t at0 = listed ? 0 : sh.blocks ? (int64_t)unit0 * sh.blocks : unit0;
    const int64_t at_end = listed ? list_n : sh.blocks ? min(at0 + sh.blocks, (int64_t)total * kblocks) : total;
    auto next = [&](int64_t &at, Piece &p) {
        if (listed) {
            if (at >= at_end) return false;
            p = {list_tile[at], 0, kblocks, list_expert[at]};
            at++;
            return true;
        }
        if (sh.blocks) {
            if (at >= at_end) return false;
            p.tile = (int)(at / kblocks), p.expert = 0;
            p.k0 = (int)(at - (int64_t)p.tile * kblocks);
            p.k1 = (int)min((int64_t)kblocks, p.k0 + (at_end - at));
            at += p.k1 - p.k0;
            return true;
        }
        while (at < at_end && nothing((int)at)) at += units;
        if (at >= at_end) return false;
        p = {(int)at, 0, kblocks, routed ? __ldcg(rt.block_expert + (int)at % tiles_m / PER_BLOCK) : 0};
        at += units;
        return true;
    };
    // first of the CTA's 16-row tiles in the weights' layout
    auto w_tile = [&](const Piece &p) { return p.expert * wtiles + (p.tile / tiles_m * CG + rank) * (BM / 16); };
    const bool odd = (K / 64) & 1;                         // the last block has 64 columns

    if (warp < W_UNPACK) {
        if constexpr (C::SHARES) set_regs_less<C::R_REST>();
        if (warp == W_COPY && lane == 0) {
            // ------------------------------------------------------------ activations
            uint32_t slot = 0, phase = 1;
            bool ok = true;
            const uint32_t full_leader = pg_leader<CG>(bar_full);
            if (!routed) asm volatile("griddepcontrol.wait;" ::: "memory");
            Piece p;
            for (int64_t at = at0; ok && next(at, p);) {
                const int m0 = p.tile % tiles_m * BN + rank * (BN / CG);
                for (int kb = p.k0; kb < p.k1; kb++) {
                    if (!(ok = pg_mbar_wait(bar_free + 8 * slot, phase, abort_flag, status, limit_ns))) break;
                    const bool half = odd && kb == kblocks - 1;
                    const uint32_t to = base + slot * (2 * C::XT), bar = full_leader + 8 * slot;
                    if (rank == 0) pg_mbar_expect(bar_full + 8 * slot, half ? BN * 128 : BN * 256);
                    tma_load_2d_to<CG>(to, &map_x, bar, kb * BK, m0);
                    if (!half) tma_load_2d_to<CG>(to + C::XT, &map_x, bar, kb * BK + 64, m0);
                    if (++slot == SLOTS) slot = 0, phase ^= 1;
                }
            }
            if (!ok) {
                // give copies that are still in flight a bounded time to land before the CTA exits
                const unsigned long long t0 = pg_globaltimer_ns();
                while (pg_globaltimer_ns() - t0 < 2000000ull) {
                }
            }
        } else if (warp >= W_WEIGHTS) {
            // ------------------------------------------------------------ weights: every second entry, a 16-row tile's four records by a lane each
            // (A copy's issue takes its lane some 200 cycles whatever its size, and a warp's lanes follow one another.  An entry per block: 2048 rows of
            // 28672 x 4096 449 us instead of 430.  Copied by the warps that unpack, a lane's two copies took 450 cycles of a block's 2700.)
            int64_t at = at0;
            Piece p = {0, 0, 0, 0};
            int e = warp - W_WEIGHTS;                      // the warp's next entry of the piece
            uint32_t entry = (uint32_t)e, phase = 1;
            bool ok = true;
            while (ok) {
                bool more = true;
                for (int n; more && e >= (n = (p.k1 - p.k0 + 1) / 2);) {
                    e -= n;
                    more = next(at, p);
                }
                if (!more) break;
                // (rows behind the last weights repeat the last ones, whose sums are dropped)
                const unsigned char *from = w + (int64_t)min(w_tile(p) + (lane & 7), alltiles - 1) * (K / 64) * record;
                for (; p.k0 + 2 * e < p.k1; e += 2) {
                    if (!(ok = pg_mbar_wait_warp(bar_read + 8 * entry, phase, abort_flag, status, limit_ns))) break;
                    const int kb = p.k0 + 2 * e, end = min(kb + 2, p.k1);
                    const uint32_t bytes = (uint32_t)((2 * (end - kb) - (odd && end == kblocks ? 1 : 0)) * record), bar = bar_w + 8 * entry;
                    if (lane == 0) pg_mbar_expect(bar, 8 * bytes);
                    __syncwarp();
                    if (lane < 8) pg_bulk_load(base + SLOTS * 2 * C::XT + entry * (2 * W_BLOCK) + (uint32_t)lane * 4 * record, from + (int64_t)(2 * kb) * record, bytes, bar);
                    entry += 2;
                    if (entry >= (uint32_t)DEPTH) entry -= DEPTH, phase ^= 1;
                }
            }
            if (!ok) {
                // give copies that are still in flight a bounded time to land before the CTA exits
                const unsigned long long t0 = pg_globaltimer_ns();
                while (pg_globaltimer_ns() - t0 < 2000000ull) {
                }
            }
            __syncwarp();
            asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        } else if (warp == W_MMA && rank == 0) {
            // ------------------------------------------------------------ products (the whole warp; one lane's count)
            // This warp shares its scheduler with four that unpack and two that write: every instruction here counts, so one wait and one
            // commit for 128 k (waits and commits of their own for the activations and for 64 k took 27 us instead of 17 rows x 14336 x 4096's 22).
            const uint32_t on = pg_elect();
            constexpr uint32_t idesc = (1u << 4) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(CG * BM >> 4) << 24);   // f16 operands, f32 sums
            uint32_t slot = 0, phase = 0, acc = 0, acc_phase = 0;
            bool ok = true;
            Piece p;
            for (int64_t at = at0; ok && next(at, p);) {
                int in = 0;
                for (int kb = p.k0; kb < p.k1; kb++) {
                    const uint32_t d = tmem + acc * BN;
                    if (in == 0) {
                        if (!(ok = pg_mbar_wait_warp(bar_tempty + 8 * acc, acc_phase ^ 1, abort_flag, status, limit_ns))) break;
                    }
                    if (!(ok = pg_mbar_wait_warp(bar_full + 8 * slot, phase, abort_flag, status, limit_ns))) break;
                    tc_fence_after();
                    const uint64_t db = make_smem_desc(base + slot * (2 * C::XT));
                    const uint32_t ta = tmem + C::A_COL + slot * 64;
#pragma unroll
                    for (int j = 0; j < 4; j++) umma_f16_ta_of<CG>(d, ta + j * 8, db + (uint64_t)(j * 2), idesc, in != 0 || j != 0 ? 1u : 0u, on);
                    if (!(odd && kb == kblocks - 1)) {
#pragma unroll
                        for (int j = 0; j < 4; j++) umma_f16_ta_of<CG>(d, ta + 32 + j * 8, db + (uint64_t)((C::XT >> 4) + j * 2), idesc, 1u, on);
                    }
                    umma_commit_to<CG>(bar_free + 8 * slot, on);
                    if (++slot == SLOTS) slot = 0, phase ^= 1;
                    if (++in == CHUNK || kb == p.k1 - 1) {
                        umma_commit_to<CG>(bar_tfull + 8 * acc, on);
                        in = 0;
                        if (++acc == 2) acc = 0, acc_phase ^= 1;
                    }
                }
            }
        }
    } else if (warp < W_OUT) {
        // ---------------------------------------------------------------- quants -> f16 in TMEM: a thread per weight row
        if constexpr (C::SHARES) set_regs_less<C::R_UNPACK>();
        const int team = (warp - W_UNPACK) >> 2, quarter = warp & 3, ti = lane >> 4, rr = lane & 15;
        const uint32_t ring = base + SLOTS * 2 * C::XT + (uint32_t)(quarter * 8 * record);
        const uint32_t off = (uint32_t)(ti * 4 * record + (rr & 7) * 64 + (rr >> 3) * 8), swz = (uint32_t)(rr >> 1 & 3) << 4;
        const uint32_t s_off = (uint32_t)(ti * 4 * record + 512 + (rr & 7) * 4 + (rr >> 3) * 2), s_step = record > 544 ? 32u : 0u;
        const uint32_t q_off[4] = {off + swz, off + (16u ^ swz), off + (32u ^ swz), off + (48u ^ swz)};
        const uint32_t a_at = tmem + ((uint32_t)(quarter * 32) << 16) + C::A_COL + team * 64, full = pg_leader<CG>(bar_full) + 8 * team, free_at = bar_free + 8 * team;
        uint32_t turn = 0;                                     // which of the team's two slots
        // the team's blocks of the pieces' blocks, one after the other
        int64_t read_at = at0;
        Piece now = {0, 0, 0, 0};
        int rb = team;
        uint32_t phase = 1, entries = 0;                       // entries: of the pieces in front of this one
        bool ok = true;
#pragma unroll 1
        for (;; rb += TEAMS) {
            while (rb >= now.k1) {
                rb -= now.k1;
                entries += (uint32_t)(now.k1 - now.k0 + 1) >> 1;
                if (!next(read_at, now)) {
                    rb = -1;
                    break;
                }
                rb += now.k0;
            }
            if (rb < 0) break;
            const int halves = odd && rb == kblocks - 1 ? 1 : 2;
            const uint32_t in = (uint32_t)(rb - now.k0), nth = entries + (in >> 1), entry = nth % DEPTH;
            if (!(ok = pg_mbar_wait_warp(bar_w + entry * 8, nth / DEPTH & 1, abort_flag, status, limit_ns))) break;
            uint32_t at = ring + entry * (2 * W_BLOCK) + (in & 1) * 2 * (uint32_t)record, to_tmem = a_at + turn * (64 * TEAMS);
#pragma unroll 1
            for (int c = 0; c < halves; c++) {                 // 64 columns, then 32 at a time: word e of the row's four lanes
                uint2 q[4];
#pragma unroll
                for (int i = 0; i < 4; i++) q[i] = lds64(at + q_off[i]);
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    unsigned short h;
                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(h) : "r"(at + s_off + e * s_step));
                    const uint32_t sc = (uint32_t)h * 0x10001u;
                    uint32_t v[16];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t word = e ? q[i].y : q[i].x, word8 = word >> 8;
                        v[4 * i] = mul_f16x2(four_f16_lo(word), sc);
                        v[4 * i + 1] = mul_f16x2(four_f16_hi(word), sc);
                        v[4 * i + 2] = mul_f16x2(four_f16_lo(word8), sc);
                        v[4 * i + 3] = mul_f16x2(four_f16_hi(word8), sc);
                    }
                    if (e == 0 && c == 0) {
                        if (!(ok = pg_mbar_wait_warp(free_at + turn * (8 * TEAMS), phase, abort_flag, status, limit_ns))) break;
                        tc_fence_after();
                    }
                    tmem_st16(to_tmem + e * 16, v);
                }
                if (!ok) break;
                at += record, to_tmem += 32;
            }
            if (!ok) break;
            pg_mbar_arrive_warp_n(bar_read + entry * 8, lane, (in & 1) == 0 && rb + 1 == now.k1 ? 2u : 1u);
            tmem_wait_st();
            tc_fence_before();
            pg_arrive_leader_warp<CG>(full + turn * (8 * TEAMS), lane);
            phase ^= turn;
            turn ^= 1;
        }
    } else {
        // ---------------------------------------------------------------- outputs: the accumulators' sums added up in registers, then written
        if constexpr (C::SHARES) set_regs_more<C::R_OUT>();
        const int q = warp & 3, half = (warp - W_OUT) >> 2;
        if (!routed) asm volatile("griddepcontrol.wait;" ::: "memory");   // y may still be read by the predecessor; xback is its work
        if (half == 0 || OUT_WARPS == 8) {
            const uint32_t tempty_leader = pg_leader<CG>(bar_tempty);
            uint32_t acc = 0, acc_phase = 0;
            bool ok = true;
            Piece p;
            for (int64_t at = at0; ok && next(at, p);) {
                const int m0 = p.tile % tiles_m * BN + half * COLS, n0 = (p.tile / tiles_m * CG + rank) * BM + q * 32;
                const float fac = n0 + lane < wtiles * 16 ? __ldg(wrow + (int64_t)(w_tile(p) + q * 2) * 16 + lane) : 0.0f;
                float xb[COLS / 16];                           // of rows m0 + 16 c + (lane & 15)
#pragma unroll
                for (int c = 0; c < COLS / 16; c++) xb[c] = m0 + 16 * c + (lane & 15) < rows ? __ldcg(xback + m0 + 16 * c + (lane & 15)) : 0.0f;
                float sum[COLS];
                for (int left = p.k1 - p.k0, first = 1; left > 0; left -= CHUNK, first = 0) {
                    if (!(ok = pg_mbar_wait_warp(bar_tfull + 8 * acc, acc_phase, abort_flag, status, limit_ns))) break;
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < COLS; c += 16) {
                        uint32_t v[16];
                        tmem_ld16(tmem + ((uint32_t)(q * 32) << 16) + acc * BN + half * COLS + c, v);
#pragma unroll
                        for (int j = 0; j < 16; j++) sum[c + j] = first ? __uint_as_float(v[j]) : sum[c + j] + __uint_as_float(v[j]);
                    }
                    tc_fence_before();
                    pg_arrive_leader_warp<CG>(tempty_leader + 8 * acc, lane);
                    if (++acc == 2) acc = 0, acc_phase ^= 1;
                }
                if (!ok) break;
                if (n0 >= N || m0 >= rows) {
                    // (nothing of the warp's piece lies inside y)
                } else if (p.k1 - p.k0 == kblocks) {
                    put<COLS, ACT>(sum, fac, xb, m0, rows - m0, n0, N, limit, y, ldy, lane);
                } else {
                    // the tile's pairs: a pair's piece is the first of its stretch unless that starts at the tile's beginning or in front of it
                    const int64_t b0 = (int64_t)p.tile * kblocks;
                    const int lo = (int)(b0 / sh.blocks), hi = (int)((b0 + kblocks - 1) / sh.blocks);
                    auto slab_of = [&](int pair) {
                        const int64_t last = (int64_t)pair * sh.blocks > b0 ? 0 : 1;
                        return sh.slabs + ((((int64_t)pair * CG + rank) * 2 + last) * OUT_WARPS + (warp - W_OUT)) * (COLS * 32) + lane;
                    };
                    float *mine = slab_of(unit0);
#pragma unroll
                    for (int j = 0; j < COLS; j++) __stcg(mine + j * 32, sum[j]);
                    unsigned int *ticket = sh.tickets + (p.tile * CG + rank) * OUT_WARPS + (warp - W_OUT);
                    __threadfence();
                    __syncwarp();
                    const unsigned int before = __shfl_sync(0xffffffffu, lane == 0 ? atomicAdd(ticket, 1u) : 0u, 0);
                    if (before == (unsigned)(hi - lo)) {
                        // the last one in adds them up in their order
                        __threadfence();
                        if (lane == 0) *ticket = 0;
#pragma unroll
                        for (int c = 0; c < COLS; c += 16) {
                            float a[16];
#pragma unroll
                            for (int j = 0; j < 16; j++) a[j] = 0.0f;
                            // (as many pairs' sums on their way at once as registers allow)
                            constexpr int AHEAD = COLS == 64 ? 3 : 2;
                            for (int pair = lo; pair <= hi; pair += AHEAD) {
                                float b[AHEAD][16];
#pragma unroll
                                for (int u = 0; u < AHEAD; u++) {
                                    const float *from = slab_of(min(pair + u, hi)) + c * 32;
#pragma unroll
                                    for (int j = 0; j < 16; j++) b[u][j] = __ldcg(from + j * 32);
                                }
#pragma unroll
                                for (int u = 0; u < AHEAD; u++)
                                    if (pair + u <= hi) {
#pragma unroll
                                        for (int j = 0; j < 16; j++) a[j] += b[u][j];
                                    }
                            }
#pragma unroll
                            for (int j = 0; j < 16; j++) sum[c + j] = a[j];
                        }
                        put<COLS, ACT>(sum, fac, xb, m0, rows - m0, n0, N, limit, y, ldy, lane);
                    }
                }
            }
        }
    }
    // (neither CTA of a pair may leave while the other can still touch its shared memory, barriers or TMEM)
    __syncwarp();
    tc_fence_before();
    pg_group_sync<CG>();
    if (warp == W_MMA) {
        tc_fence_after();
        tmem_dealloc<CG>(tmem, 512);
    }
}

// ---------------------------------------------------------------- host side ----
template <int BN, int ACT, typename TY>
int32_t launch(pg_ctx *ctx, const pg_linear4 *lin, const void *x, const float *xback, int64_t m, float limit, TY *y, int64_t ldy, const PgRouted &rt, Share sh)
{
    using C = Cfg<BN>;
    CUtensorMap mx;
    const cuuint64_t xd[2] = {(cuuint64_t)lin->k, (cuuint64_t)m}, xs[1] = {(cuuint64_t)lin->k * 2};
    const cuuint32_t xb[2] = {64, (cuuint32_t)(BN / CG)};
    int32_t rc = pg_encode_map(&mx, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, x, 2, xd, xs, xb);
    if (rc) return rc;
    auto kern = linear4_tc_kernel<BN, ACT, TY>;
    static std::atomic<uint64_t> set{0};
    PG_CUDA(pg_max_smem_once(kern, (int)C::SMEM, ctx->device, set));
    const int64_t tiles = ((m + BN - 1) / BN) * ((lin->n + CG * BM - 1) / (CG * BM)), pairs = ctx->sm_count / CG;
    PG_REQUIRE(tiles < (1ll << 31) - 65536, "linear4: too many tiles");
    const int64_t grid = sh.blocks ? (tiles * ((lin->k + BK - 1) / BK) + sh.blocks - 1) / sh.blocks : std::min<int64_t>(tiles, pairs);
    sh.tickets = reinterpret_cast<unsigned int *>(ctx->splitk);
    sh.slabs = reinterpret_cast<float *>(reinterpret_cast<unsigned char *>(ctx->splitk) + PG_LM_TICKET_BYTES);
    return launch_pdl_cluster(ctx, kern, dim3((unsigned)(grid * CG)), dim3(C::THREADS), C::SMEM, CG, mx, lin->w, lin->row, xback, (int)m, (int)lin->n, (int)lin->k,
                              (int)lin->record, (int)lin->tiles, (int)(lin->experts * lin->tiles), limit, y, ldy, rt, sh, ctx->d_status, ctx->wait_limit_ns);
}

template <int ACT, typename TY>
int32_t dispatch(pg_ctx *ctx, const pg_linear4 *lin, const void *x, const float *xback, int64_t m, float limit, TY *y, int64_t ldy, const PgRouted &rt, int64_t pairs)
{
    const int kblocks = (int)((lin->k + BK - 1) / BK);
    Share sh = {0, nullptr, nullptr};
    int bn = 128;
    if (rt.blocks) {
        // rows an expert has on average
        const int64_t rows = (pairs + lin->experts - 1) / lin->experts;
        bn = rows <= 24 ? 32 : rows <= 48 ? 64 : 128;
    } else {
        // cycles, from measurements: of a block of 128 k (its unpacking, products and sums), and of a pair's stretch what it costs to put shared tiles
        // together.  (17 to 300 rows of five matrices from 4096 x 4096 to 28672 x 4096, BN 32, 64 and 128: at most 2 % from the best of the six.  Shared
        // stretches against whole tiles: 100 rows 4096 x 14336 30.6 and 51.9 us, 200 rows 4096 x 4096 25.6 and 20.4.)
        double best = 1e30;
        const int64_t sm_pairs = ctx->sm_count / CG;
        for (int cand : {32, 64, 128}) {
            const int64_t tiles = ((m + cand - 1) / cand) * ((lin->n + CG * BM - 1) / (CG * BM)), rounds = (tiles + sm_pairs - 1) / sm_pairs;
            const double block = cand == 32 ? 550.0 : cand == 64 ? 600.0 : 800.0, whole = (double)rounds * kblocks * block;
            if (whole < best) best = whole, bn = cand, sh.blocks = 0;
            if (tiles > 1024) continue;
            const int64_t blocks = std::max<int64_t>(2, (tiles * kblocks + sm_pairs - 1) / sm_pairs);
            const double time = blocks * block + 6000.0 + 60.0 * cand;
            if (time < best) best = time, bn = cand, sh.blocks = (int)blocks;
        }
    }
    if (sh.blocks) {
        const int32_t rc = pg_splitk_reserve(ctx, pgk_linear4_tc_workspace(ctx));
        if (rc != PG_OK) return rc;
    }
    if (bn == 128) return launch<128, ACT, TY>(ctx, lin, x, xback, m, limit, y, ldy, rt, sh);
    if (bn == 64) return launch<64, ACT, TY>(ctx, lin, x, xback, m, limit, y, ldy, rt, sh);
    return launch<32, ACT, TY>(ctx, lin, x, xback, m, limit, y, ldy, rt, sh);
}

}  // namespace

size_t pgk_linear4_tc_workspace(const pg_ctx *ctx) { return PG_LM_TICKET_BYTES + (size_t)ctx->sm_count * 2 * 128 * BM * sizeof(float); }

int32_t pgk_linear4_tc(pg_ctx *ctx, const pg_linear4 *lin, const bf16 *a, int64_t lda, int64_t m, int act, float limit, void *y, int y_dtype, int64_t ldy,
                       const PgRouted *routed, const pg_route *route)
{
    static const PgRouted no_route = {};
    const PgRouted &rt = routed ? *routed : no_route;
    const int64_t pairs = route ? route->m * route->top : 0;
    const size_t xbytes = (size_t)m * lin->k * 2;
    int32_t rc = pg_scratch_reserve_recording(ctx, xbytes + (size_t)m * sizeof(float));
    if (rc != PG_OK) return rc;
    float *back = reinterpret_cast<float *>((unsigned char *)ctx->scratch + xbytes);
    // (a row's loads all on their way at once: up to 4096 columns with 128 threads, up to 16384 with 512)
    const bool wide = lin->k > 128 * RW_KEEP * 8;
    rc = launch_pdl(ctx, wide ? linear4_rows_kernel<512> : linear4_rows_kernel<128>, dim3((unsigned)(route ? rt.by_token ? route->m : pairs : m)), dim3(wide ? 512 : 128), 0, a, lda, (int)lin->k, rt,
                    route ? (const int32_t *)route->pair_row : (const int32_t *)nullptr, (uint4 *)ctx->scratch, back);
    if (rc != PG_OK) return rc;
    if (act == PG_ACT_GELU_TANH_GLU) return dispatch<PG_ACT_GELU_TANH_GLU, bf16>(ctx, lin, ctx->scratch, back, m, limit, (bf16 *)y, ldy, rt, pairs);
    if (act == PG_ACT_CLAMPED_SWISH_GLU) return dispatch<PG_ACT_CLAMPED_SWISH_GLU, bf16>(ctx, lin, ctx->scratch, back, m, limit, (bf16 *)y, ldy, rt, pairs);
    if (y_dtype == PG_BF16) return dispatch<PG_ACT_NONE, bf16>(ctx, lin, ctx->scratch, back, m, limit, (bf16 *)y, ldy, rt, pairs);
    return dispatch<PG_ACT_NONE, float>(ctx, lin, ctx->scratch, back, m, limit, (float *)y, ldy, rt, pairs);
}
