// Decode-size product y = act(a W^T) with weights of 4 bits (csrc/pg_linear4.cu), at most 16 rows, one pass over the weights.
//
//   * The weights are the M side of mma.sync m16n8k16 (16 rows x 16 k), activation rows its 8 columns; up to 16 rows of a take two column
//     tiles on the same unpacked quants.  Quants become f16 integers (exact), sums of a group are scaled in f32.
//   * The activations are bf16 and enter as f16: a warp divides each row of its part of K by a power of two of its own (four_range) and
//     multiplies the sums back: exact down to 2^-27 of the part's largest, and smaller ones are off by 2^-36 of that at most.
//   * One persistent CTA of 16 warps per SM.  `kw` warps share a tile of 16 weight rows, each with one part of K of at most 512 elements (256 with more than
//     eight rows), whose activations it holds as operands, 64 words of a lane's 128 registers (parts of 512 do not quite fit: 156 to 236 bytes of a lane
//     are kept in local memory; parts of 256: up to 48); a fill of its ring is one bulk copy, quants and scales.  The parts meet in shared memory in a
//     fixed order; the warps of a tile take turns in adding.
//   * K beyond 16 such parts: sp CTAs take the same tiles, their sums go to slabs, the last one in (a ticket) adds in a fixed order.
//   * ROUTED: rows come in blocks of 16 that share an expert.
//
// What bounds it: instructions and their latency.  A record of 16 x 64 weights is some 60 instructions of a warp (quants to f16 32 of them at half rate)
// and 8 products, four warps to a scheduler: 28672 x 4096 takes 18.9 us with one row (3.3 TB/s), 20.3 with eight, 33.5 with 16, whose two column tiles
// leave room for parts of 256 only.  4096 x 4096 with one row: 6.5 us, launch, first copies and the hand-over of the parts.
//
// Every mbarrier wait is bounded; a warp that gave up goes on through the remaining barriers without computing.
#include <algorithm>
#include <type_traits>

#include "pg_async.cuh"
#include "pg_four.cuh"

namespace {

constexpr int V4_WARPS = 16, V4_THREADS = V4_WARPS * 32;
constexpr int V4_SLOTS_MAX = 8;
constexpr int V4_CELLS = 4;                               // tiles whose parts may be on their way at once
__host__ __device__ constexpr int v4_ring(int nt) { return nt == 1 ? 2 * 4608 : 4 * 2304; }    // bytes of a warp's ring
__host__ __device__ constexpr int v4_kw_max(int nt) { return nt == 1 ? 512 : 256; }   // (64 words of the activations to a lane)

// shared memory: ring | parts of a tile [V4_CELLS][16 warps][32 lanes][4 NT] | barriers
// slabs (K over several CTAs): [sp][items][32 lanes][4 NT]
template <int ACT, int NT, bool ROUTED, int G32, typename TY>
__global__ void __launch_bounds__(V4_THREADS, 1)
    linear4_gemv_kernel(const bf16 *__restrict__ a, int64_t lda, int M, const unsigned char *__restrict__ w, const float *__restrict__ wrow, int N, int K, int record,
                        int tiles, int kw, int KW, int KH, int slots, float limit, TY *__restrict__ y, int64_t ldy, const PgRouted rt, int sp, float *slabs,
                        unsigned int *tickets, int32_t *status, unsigned long long limit_ns)
{
    constexpr int CELL = 4 * NT;                          // floats per lane
    constexpr int KWM = v4_kw_max(NT);
    extern __shared__ __align__(128) unsigned char smem[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), r = lane >> 2, t = lane & 3;
    const int my_part = sp > 1 ? (int)blockIdx.x % sp : 0;
    const int groups = V4_WARPS / kw, slot_idx = warp / kw, kpart = warp - slot_idx * kw;
    float *part = reinterpret_cast<float *>(smem + V4_WARPS * v4_ring(NT));
    unsigned char *tail = reinterpret_cast<unsigned char *>(part + V4_CELLS * V4_WARPS * 32 * CELL);
    const uint32_t my_bar = pg_smem(tail) + (uint32_t)warp * (V4_SLOTS_MAX * 8);
    const uint32_t cell_full = pg_smem(tail) + V4_WARPS * V4_SLOTS_MAX * 8 + (uint32_t)slot_idx * (V4_CELLS * 16), cell_free = cell_full + V4_CELLS * 8;
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tail + V4_WARPS * V4_SLOTS_MAX * 8 + V4_WARPS * V4_CELLS * 16);
    const uint32_t ring = pg_smem(smem) + (uint32_t)(warp * v4_ring(NT));
    if (threadIdx.x == 0) *abort_flag = 0;
    if (threadIdx.x < V4_WARPS * V4_SLOTS_MAX) {
        pg_mbar_init(pg_smem(tail) + 8 * threadIdx.x, 1);
        pg_mbar_fence();
    } else if (threadIdx.x < V4_WARPS * V4_SLOTS_MAX + groups * V4_CELLS * 2) {
        const int i = threadIdx.x - V4_WARPS * V4_SLOTS_MAX;   // the parts are there; they have been added
        pg_mbar_init(pg_smem(tail) + 8 * threadIdx.x, i / V4_CELLS % 2 ? 1 : max(1, kw - 1));
        pg_mbar_fence();
    }
    static_assert(V4_WARPS * (V4_SLOTS_MAX + V4_CELLS * 2) <= V4_THREADS, "a thread per barrier");
    __syncthreads();

    const int ka0 = my_part * KH, k0 = ka0 + kpart * KW;
    const int klen = max(0, min(KW, min(K, ka0 + KH) - k0));   // a multiple of 64 and of the group; 0 only in a short last range
    const int64_t unit = blockIdx.x / sp, units = gridDim.x / sp;
    if (ROUTED) asm volatile("griddepcontrol.wait;" ::: "memory");
    const int nblk = ROUTED ? __ldcg(rt.blocks) : 1;
    const int64_t items = (int64_t)nblk * tiles, per = (items + units * groups - 1) / (units * groups);
    // a route's items in stretches, so that a block's activations are brought in once; else turn by turn
    const int64_t first = ROUTED ? (unit * groups + slot_idx) * per : unit * groups + slot_idx, step = ROUTED ? 1 : units * groups;
    const int mine = first >= items ? 0 : ROUTED ? (int)min(per, items - first) : (int)((items - first + step - 1) / step);
    const int total = klen > 0 ? mine : 0;
    const uint32_t fill_bytes = (uint32_t)(klen / 64 * record);
    const int64_t row_bytes = (int64_t)(K / 64) * record;

    // a tile of the weights' layout; with a route the tiles of a block's expert follow one another, and the expert is looked up where a block begins
    const int blk0 = ROUTED ? (int)(first / tiles) : 0, tile0 = ROUTED ? (int)(first - (int64_t)blk0 * tiles) : 0;
    auto expert_of = [&](int blk) -> int64_t { return blk < nblk ? __ldcg(rt.block_expert + blk) : 0; };
    const int64_t base0 = !ROUTED ? first : mine > 0 ? expert_of(blk0) * tiles + tile0 : 0;
    // fills follow one another through the slots; without a route they lie a constant distance apart
    int fill_slot = 0, fill_blk = blk0, fill_tile = tile0;
    const unsigned char *next = w + base0 * row_bytes + k0 / 64 * record;
    auto issue = [&]() {
        if (lane == 0) {
            const uint32_t bar = my_bar + (uint32_t)fill_slot * 8;
            pg_mbar_expect(bar, fill_bytes);
            pg_bulk_load(ring + (uint32_t)fill_slot * fill_bytes, next, fill_bytes, bar);
        }
        next += step * row_bytes;
        if (ROUTED && ++fill_tile == tiles) {
            fill_tile = 0;
            next = w + expert_of(++fill_blk) * tiles * row_bytes + k0 / 64 * record;
        }
        if (++fill_slot == slots) fill_slot = 0;
    };
    for (int f = 0; f < slots; f++)
        if (f < total) issue();
    if (!ROUTED) asm volatile("griddepcontrol.wait;" ::: "memory");

    // activations of the warp's part of K: word 4 c + i of column r (and r + 8): the pairs of columns 32 c + 8 t + 2 i, every second one over 16 (the
    // quants beside it come 16 times too large: as q - 8 they take a constant more, which the registers do not have, 36.9 -> 38.6 us with 16 rows of
    // 28672 x 4096; so every bf16 number down to 2^-27 of the part's largest is exact)
    uint32_t x[NT][KWM / 8];
    float back[NT][2];                                    // what the sums of columns 2 t and 2 t + 1 are multiplied by
    auto bring = [&](int blk) {
#pragma unroll
        for (int j = 0; j < NT; j++) {
            int64_t at = r + 8 * j;
            bool in = at < M;
            if (ROUTED) {
                const int p = __ldcg(rt.row_pair + blk * PG_ROUTE_SMALL + r + 8 * j);
                in = p >= 0;
                at = rt.by_token ? p / rt.top : blk * PG_ROUTE_SMALL + r + 8 * j;
            }
            const bf16 *src = a + at * lda + k0 + t * 8;
            uint4 v[KWM / 32];
            float top = 0.0f;
#pragma unroll
            for (int c = 0; c < KWM / 32; c++) v[c] = in && c * 32 < klen ? __ldcg(reinterpret_cast<const uint4 *>(src + c * 32)) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
            for (int c = 0; c < KWM / 32; c++) {
                const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
                for (int i = 0; i < 4; i++) top = fmaxf(top, fmaxf(fabsf(pg_bf16_lo(w[i])), fabsf(pg_bf16_hi(w[i]))));
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            float down, up;
            four_range(top, down, up);
#pragma unroll
            for (int c = 0; c < KWM / 32; c++) {
                const uint32_t w[4] = {v[c].x, v[c].y, v[c].z, v[c].w};
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float by = i & 1 ? down * 0.0625f : down;
                    x[j][4 * c + i] = four_pack_f16(pg_bf16_lo(w[i]) * by, pg_bf16_hi(w[i]) * by);
                }
            }
            back[j][0] = __shfl_sync(0xffffffffu, up, 8 * t);          // (lane 4 c has column c)
            back[j][1] = __shfl_sync(0xffffffffu, up, 8 * t + 4);
        }
    };

    // bit 2 j + i: there is a row 8 j + 2 t + i
    auto rows_of = [&](int blk) {
        uint32_t in = 0;
#pragma unroll
        for (int j = 0; j < 2 * NT; j++) {
            const int m = 8 * (j >> 1) + 2 * t + (j & 1);
            in |= (uint32_t)(ROUTED ? __ldcg(rt.row_pair + blk * PG_ROUTE_SMALL + m) >= 0 : m < M) << j;
        }
        return in;
    };
    // outputs of a tile; lane: weight rows r and r + 8, rows 2 t and 2 t + 1 of the activations
    auto finish = [&](const float (&acc)[NT][4], int blk, int tile, uint32_t in) {
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int64_t m = (ROUTED ? blk * PG_ROUTE_SMALL : 0) + 8 * j + 2 * t + i;
                if (!(in >> (2 * j + i) & 1u)) continue;
                const float v0 = acc[j][i], v1 = acc[j][2 + i];
                if (ACT != PG_ACT_NONE) {
                    pg_put(y + m * ldy + tile * 8 + r, pg_glu<ACT>(v0, v1, limit));
                } else {
                    const int n = tile * 16 + r;
                    if (n < N) pg_put(y + m * ldy + n, v0);
                    if (n + 8 < N) pg_put(y + m * ldy + n + 8, v1);
                }
            }
    };

    bool ok = true, second = NT == 2;
    int slot = 0, cell = 0;
    uint32_t phase = 0, cell_phase = 0;
    if (!ROUTED && mine > 0 && klen > 0) bring(0);
    int blk = blk0 - 1, tile = ROUTED ? tiles - 1 : (int)(first - step);
    uint32_t in = ROUTED ? 0 : rows_of(0);
    const float *fac = wrow + (base0 - step) * 16 + r;    // the factors of rows r and r + 8 of the tile
    for (int j = 0; j < mine; j++) {
        float acc[NT][4] = {};
        const int64_t it = first + j * step;
        tile += (int)step, fac += step * 16;
        if (ROUTED && (tile == tiles || j == 0)) {        // another block, another expert
            blk++, tile = j == 0 ? tile0 : 0;
            if (j > 0) fac = wrow + expert_of(blk) * tiles * 16 + r;
            in = rows_of(blk);
            if (klen > 0) bring(blk);
            second = NT == 2 && __shfl_sync(0xffffffffu, (int)(in >> 2 & 1u), 0);   // (a block's rows are filled from the first on)
        }
        const int turn = (j + slot_idx) & (kw - 1);       // the warp that adds the parts up
        if (klen > 0) {
            const float f0 = __ldg(fac), f1 = __ldg(fac + 8);
            ok = ok && pg_mbar_wait_warp(my_bar + (uint32_t)slot * 8, phase, abort_flag, status, limit_ns);
            if (ok) {
                const uint32_t slot_at = ring + (uint32_t)slot * fill_bytes;
                uint32_t at = slot_at + 16u * (uint32_t)(4 * r + (t ^ (r >> 1 & 3))), s_at = slot_at + 512u + (uint32_t)r * 4;
                // (without a way out between the records their loads and products overlap)
                auto records = [&](auto full) {
                    constexpr bool whole = decltype(full)::value;
                    float sum[NT][4];
#pragma unroll
                    for (int b = 0; b < KWM / 64; b++) {
                        if (!whole && b * 64 >= klen) break;
                        const uint4 q4 = pg_lds128(at);
                        const uint32_t q[4] = {q4.x, q4.y, q4.z, q4.w};
#pragma unroll
                        for (int h = 0; h < 2; h++) {
#pragma unroll
                            for (int u = 0; u < 2; u++) {
                                const uint32_t w0 = u ? q[h] >> 8 : q[h], w1 = u ? q[2 + h] >> 8 : q[2 + h];
                                const uint32_t a0 = four_f16_lo(w0), a1 = four_f16_lo(w1), a2 = four_f16_hi16(w0), a3 = four_f16_hi16(w1);
                                const int i = 8 * b + 4 * h + 2 * u;
                                if ((2 * b + h) % G32 == 0 && u == 0) {
                                    four_mma_f16_first(sum[0], a0, a1, a2, a3, x[0][i], x[0][i + 1]);
                                    if (NT == 2 && (!ROUTED || second)) four_mma_f16_first(sum[NT - 1], a0, a1, a2, a3, x[NT - 1][i], x[NT - 1][i + 1]);
                                } else {
                                    four_mma_f16(sum[0], a0, a1, a2, a3, x[0][i], x[0][i + 1]);
                                    if (NT == 2 && (!ROUTED || second)) four_mma_f16(sum[NT - 1], a0, a1, a2, a3, x[NT - 1][i], x[NT - 1][i + 1]);
                                }
                            }
                            if ((2 * b + h + 1) % G32 == 0) { // the group ends behind this half of the record
                                uint32_t both;                // the scales of rows r and r + 8
                                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(both) : "r"(s_at + (G32 == 1 ? h * 32 : 0)));
                                const float2 sc = __half22float2(*reinterpret_cast<const __half2 *>(&both));
#pragma unroll
                                for (int n = 0; n < NT; n++) {
                                    if (n == 1 && ROUTED && !second) break;
                                    acc[n][0] = fmaf(sc.x, sum[n][0], acc[n][0]), acc[n][1] = fmaf(sc.x, sum[n][1], acc[n][1]);
                                    acc[n][2] = fmaf(sc.y, sum[n][2], acc[n][2]), acc[n][3] = fmaf(sc.y, sum[n][3], acc[n][3]);
                                }
                            }
                        }
                        at += record, s_at += record;
                    }
                };
                if (klen == KWM)
                    records(std::true_type{});
                else
                    records(std::false_type{});
                __syncwarp();                             // every lane has read the slot
                if (j + slots < total) issue();
                if (++slot == slots) slot = 0, phase ^= 1;
#pragma unroll
                for (int n = 0; n < NT; n++) {            // (the row's factor first: what is multiplied is never far beyond the result)
                    acc[n][0] = acc[n][0] * f0 * back[n][0], acc[n][1] = acc[n][1] * f0 * back[n][1];
                    acc[n][2] = acc[n][2] * f1 * back[n][0], acc[n][3] = acc[n][3] * f1 * back[n][1];
                }
            }
        }
        if (kw > 1) {
            // the others leave their parts and go on; the warp whose turn it is waits for them.  It too waits until the cell's last use is over: before
            // that the phase of cell_full that it would wait on has not begun
            float *cells = part + ((size_t)(cell * V4_WARPS + slot_idx * kw) * 32 + lane) * CELL;
            ok = ok && pg_mbar_wait_warp(cell_free + 8 * cell, cell_phase ^ 1, abort_flag, status, limit_ns);
            if (kpart != turn) {
                if (ok) {
#pragma unroll
                    for (int n = 0; n < NT; n++) reinterpret_cast<float4 *>(cells + (size_t)kpart * 32 * CELL)[n] = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
                    pg_mbar_arrive_warp(cell_full + 8 * cell, lane);
                }
            } else {
                ok = ok && pg_mbar_wait_warp(cell_full + 8 * cell, cell_phase, abort_flag, status, limit_ns);
                if (ok) {
                    float all[NT][4] = {};
#pragma unroll 4
                    for (int p = 0; p < kw; p++) {        // in the order of K, its own where its turn is
#pragma unroll
                        for (int n = 0; n < NT; n++) {
                            float4 v = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
                            if (p != turn) v = reinterpret_cast<const float4 *>(cells + (size_t)p * 32 * CELL)[n];
                            all[n][0] += v.x, all[n][1] += v.y, all[n][2] += v.z, all[n][3] += v.w;
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[n][i] = all[n][i];
                    pg_mbar_arrive_warp(cell_free + 8 * cell, lane);
                }
            }
            if (++cell == V4_CELLS) cell = 0, cell_phase ^= 1;
        }
        if (kpart == turn && ok) {
            if (sp > 1) {
                float4 *dst = reinterpret_cast<float4 *>(slabs + (((int64_t)my_part * items + it) * 32 + lane) * CELL);
#pragma unroll
                for (int n = 0; n < NT; n++) dst[n] = make_float4(acc[n][0], acc[n][1], acc[n][2], acc[n][3]);
            } else {
                finish(acc, blk, tile, in);
            }
        }
    }
    if (sp > 1) {
        __shared__ int last_in;
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
            __threadfence();
            last_in = atomicAdd(tickets + unit, 1u) == (unsigned)(sp - 1);
            if (last_in) tickets[unit] = 0;
        }
        __syncthreads();
        if (last_in) {
            __threadfence();
            // the unit's items, a warp each
            const int64_t count = ROUTED ? max((int64_t)0, min(groups * per, items - unit * groups * per)) : 0;
            for (int64_t i = warp;; i += V4_WARPS) {
                int64_t it;
                if (ROUTED) {
                    if (i >= count) break;
                    it = unit * groups * per + i;
                } else {
                    it = unit * groups + i % groups + i / groups * (units * groups);
                    if (unit * groups + i / groups * (units * groups) >= items) break;
                    if (it >= items) continue;
                }
                const int blk = ROUTED ? (int)(it / tiles) : 0;
                float acc[NT][4] = {};
#pragma unroll 4
                for (int p = 0; p < sp; p++) {
                    const float4 *src = reinterpret_cast<const float4 *>(slabs + (((int64_t)p * items + it) * 32 + lane) * CELL);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const float4 v = __ldcg(src + n);
                        acc[n][0] += v.x, acc[n][1] += v.y, acc[n][2] += v.z, acc[n][3] += v.w;
                    }
                }
                finish(acc, blk, (int)(it - (int64_t)blk * tiles), rows_of(blk));
            }
        }
    }
    if (!ok) {
        // copies that are still in flight get a bounded time to land before the shared memory goes
        const unsigned long long t0 = pg_globaltimer_ns();
        while (pg_globaltimer_ns() - t0 < 2000000ull) {
        }
    }
}

// parts of K that CTAs share, and how long a CTA's and a warp's part is
struct Parts {
    int sp, KH, kw, KW;
};
int split_of(int64_t k, int nt) { return (int)((k + V4_WARPS * v4_kw_max(nt) - 1) / (V4_WARPS * v4_kw_max(nt))); }
Parts parts_of(const pg_linear4 *lin, int64_t items, int sms, int nt)
{
    const int K = (int)lin->k, unit = (int)std::max<int64_t>(64, lin->group), most = v4_kw_max(nt);
    Parts p;
    p.sp = split_of(K, nt);
    p.KH = p.sp > 1 ? (int)pg_up((K + p.sp - 1) / p.sp, unit) : K;
    const int64_t units = std::max(1, sms / p.sp);
    // as few parts as registers allow, more while every (tile, part) still finds a warp of its own
    p.kw = 1;
    while (p.kw < V4_WARPS && pg_up((p.KH + p.kw - 1) / p.kw, unit) > most) p.kw *= 2;
    while (p.kw < V4_WARPS && p.KH / (p.kw * 2) >= unit && items * (p.kw * 2) <= units * V4_WARPS) p.kw *= 2;
    p.KW = (int)pg_up((p.KH + p.kw - 1) / p.kw, unit);
    return p;
}

template <int ACT, int NT, bool ROUTED, int G32, typename TY>
int32_t launch(pg_ctx *ctx, const pg_linear4 *lin, const bf16 *a, int64_t lda, int M, const Parts &p, int grid, float limit, TY *y, int64_t ldy, const PgRouted &rt)
{
    auto kern = linear4_gemv_kernel<ACT, NT, ROUTED, G32, TY>;
    constexpr int smem = V4_WARPS * v4_ring(NT) + V4_CELLS * V4_WARPS * 32 * 4 * NT * 4 + V4_WARPS * (V4_SLOTS_MAX * 8 + V4_CELLS * 16) + 16;
    static_assert(smem <= 226 * 1024, "shared memory of the streaming form");
    static std::atomic<uint64_t> set{0};
    PG_CUDA(pg_max_smem_once(kern, smem, ctx->device, set));
    const int slots = std::min(V4_SLOTS_MAX, v4_ring(NT) / (int)(p.KW / 64 * lin->record));
    unsigned int *tickets = reinterpret_cast<unsigned int *>(ctx->splitk);
    float *slabs = p.sp > 1 ? reinterpret_cast<float *>(reinterpret_cast<unsigned char *>(ctx->splitk) + PG_LM_TICKET_BYTES) : nullptr;
    return launch_pdl(ctx, kern, dim3((unsigned)grid), dim3(V4_THREADS), (size_t)smem, a, lda, M, lin->w, lin->row, (int)lin->n, (int)lin->k,
                      (int)lin->record, (int)lin->tiles, p.kw, p.KW, p.KH, slots, limit, y, ldy, rt, p.sp, slabs, tickets, ctx->d_status, ctx->wait_limit_ns);
}

// slabs of a call
size_t slab_bytes(int sp, int64_t items, int nt) { return sp > 1 ? PG_LM_TICKET_BYTES + (size_t)sp * (size_t)items * 32 * 4 * nt * sizeof(float) : 0; }

}  // namespace

size_t pgk_linear4_gemv_workspace(const pg_linear4 *lin)
{
    // (a route of up to 16 tokens has a block per expert at most)
    return std::max(slab_bytes(split_of(lin->k, 2), lin->tiles * lin->experts, 2), slab_bytes(split_of(lin->k, 1), lin->tiles, 1));
}

int32_t pgk_linear4_gemv(pg_ctx *ctx, const pg_linear4 *lin, const bf16 *a, int64_t lda, int64_t m, int act, float limit, void *y, int y_dtype, int64_t ldy,
                         const PgRouted *routed, int64_t max_blocks)
{
    const int64_t items = lin->tiles * (routed ? max_blocks : 1);
    const int nt = m > 8 ? 2 : 1;   // (the rows of an expert belong to different tokens, see pg_route.cu)
    const Parts p = parts_of(lin, items, ctx->sm_count, nt);
    PG_REQUIRE(p.KW <= v4_kw_max(nt) && p.sp <= 16, "linear4: K too long");
    if (p.sp > 1) {
        const int32_t rc = pg_splitk_reserve(ctx, slab_bytes(p.sp, items, nt));
        if (rc != PG_OK) return rc;
    }
    const int groups = V4_WARPS / p.kw;
    const int grid = (int)std::min<int64_t>(ctx->sm_count / p.sp, (items + groups - 1) / groups) * p.sp;
    static const PgRouted no_route = {};
    const PgRouted &rt = routed ? *routed : no_route;
#define PG_V4(ACT, NT, RT, TY)                                                                                                                   \
    do {                                                                                                                                         \
        if (lin->group == 32) return launch<ACT, NT, RT, 1, TY>(ctx, lin, a, lda, (int)m, p, grid, limit, (TY *)y, ldy, rt);                     \
        if (lin->group == 64) return launch<ACT, NT, RT, 2, TY>(ctx, lin, a, lda, (int)m, p, grid, limit, (TY *)y, ldy, rt);                     \
        return launch<ACT, NT, RT, 4, TY>(ctx, lin, a, lda, (int)m, p, grid, limit, (TY *)y, ldy, rt);                                           \
    } while (0)
#define PG_V4_ACT(ACT, TY)                  \
    do {                                    \
        if (routed && nt == 2) PG_V4(ACT, 2, true, TY); \
        if (routed) PG_V4(ACT, 1, true, TY); \
        if (nt == 2) PG_V4(ACT, 2, false, TY); \
        PG_V4(ACT, 1, false, TY);           \
    } while (0)
    if (act == PG_ACT_GELU_TANH_GLU) PG_V4_ACT(PG_ACT_GELU_TANH_GLU, bf16);
    if (act == PG_ACT_CLAMPED_SWISH_GLU) PG_V4_ACT(PG_ACT_CLAMPED_SWISH_GLU, bf16);
    if (y_dtype == PG_BF16) PG_V4_ACT(PG_ACT_NONE, bf16);
    PG_V4_ACT(PG_ACT_NONE, float);
#undef PG_V4
#undef PG_V4_ACT
}
