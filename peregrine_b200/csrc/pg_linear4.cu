// Products with weights of 4 bits and a scale per group of K (include/peregrine_b200_lm.h): the handle, the layout of the weights, and
// the choice of kernel.
//
// W[n][k] = s[n][k / group] (q[n][k] - 8).  A record is 16 rows x 64 k: 512 bytes of quants, then one or (groups of 32) two times 16 scales.
//
// Quants: lane (r = lane / 4, t = lane % 4) of a warp has 16 bytes, at 16 (4 r + (t ^ (r / 2 & 3))): in this order neither a warp that reads all of
// them nor threads that each read their row's eight bytes of the four lanes meet a bank twice.  Words c = 0, 1 hold row r, words 2 + c row r + 8, columns
// 32 c + 8 t + {0 .. 7}: bits 0-3 columns 0 (low half) and 1 (high half), bits 4-7 columns 2 and 3, bits 8-11 4 and 5, bits 12-15 6 and 7.  Once the
// quants are f16 numbers that is an A operand of mma.sync m16n8k16, and a row's words are its columns in their order.  Scales: rows r and r + 8 side
// by side; where a group is 128 long its two records both have them, so that a record is all that a block of 64 k needs.
//
// Scales are kept as f16 divided by a power of two per row, which brings the row's largest to [2^11, 2^12): a scale's 8 bits are then an f16 number,
// exactly, as long as the row's scales are within 2^28 of each other (below, the smaller ones lose bits that are under 2^-36 of the largest), and so is
// scale * (q - 8), a multiple of it with 11 bits at most.  All forms of the product take these weights, which are what pg_linear4_read says.
#include <algorithm>
#include <new>

#include "pg_four.cuh"

namespace {

// One CTA of 128 threads per 16 rows.  QUANTS: from quants [n][k / 2] (two a byte, the first in the low half) and bf16 scales [n][k / group];
// else from bf16 weights [n][k].
template <bool QUANTS>
__global__ void __launch_bounds__(128)
    linear4_pack_kernel(const void *__restrict__ src, const bf16 *__restrict__ scales, int n, int k, int group, int record, unsigned char *__restrict__ out,
                        float *__restrict__ row)
{
    extern __shared__ float sm[];                      // scales [k / group][16] | largest of each row [16]
    const int tile = blockIdx.x, tiles = gridDim.x, groups = k / group;
    const int64_t e = blockIdx.y;
    float *top = sm + groups * 16;
    int *mag = reinterpret_cast<int *>(top);
    if (threadIdx.x < 16) mag[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * groups; i += 128) {
        const int r = i & 15, g = i >> 4, at = tile * 16 + r;
        float v = 0.0f;
        if (at < n) {
            if constexpr (QUANTS) {
                v = __bfloat162float(scales[(e * n + at) * groups + g]);
            } else {
                const bf16 *w = reinterpret_cast<const bf16 *>(src) + (e * n + at) * (int64_t)k + (int64_t)g * group;
                float best = 0.0f, most = -1.0f;
                bool fine = true;
                for (int j = 0; j < group; j++) {
                    const float x = __bfloat162float(w[j]), a = fabsf(x);
                    fine = fine && isfinite(x);
                    if (a > most) most = a, best = x;
                }
                v = fine ? four_scale(best) : __uint_as_float(0x7fc00000u);
            }
        }
        sm[g * 16 + r] = v;
        if (isfinite(v)) atomicMax(mag + r, __float_as_int(fabsf(v)));   // (magnitudes order as integers)
    }
    __syncthreads();
    // 2^row: the largest scale in [2^11, 2^12)
    float down = 1.0f;
    if (threadIdx.x < 16) {
        const int ex = max(mag[threadIdx.x] >> 23, 16);
        down = __uint_as_float((uint32_t)min(265 - ex, 254) << 23);
        row[(e * tiles + tile) * 16 + threadIdx.x] = __uint_as_float((uint32_t)(254 - min(265 - ex, 254)) << 23);
    }
    __syncthreads();
    if (threadIdx.x < 16) top[threadIdx.x] = down;
    __syncthreads();
    unsigned char *dst = out + (e * tiles + tile) * (int64_t)(k / 64) * record;
    const int per = (record - 512) / 32;               // scales of a row in a record
    for (int i = threadIdx.x; i < k / 64 * per * 16; i += 128) {
        const int b = i / (per * 16), c = i / 16 % per, x = i % 16, r = (x >> 1) + 8 * (x & 1);
        reinterpret_cast<__half *>(dst + (int64_t)b * record + 512)[c * 16 + x] = __float2half_rn(sm[(b * 64 + c * 32) / group * 16 + r] * top[r]);
    }
    for (int i = threadIdx.x; i < k / 64 * 32; i += 128) {
        const int b = i >> 5, lane = i & 31, r = lane >> 2, t = lane & 3;
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            w[j] = 0;
#pragma unroll
            for (int c = 0; c < 8; c++) {
                const int rr = r + 8 * (j >> 1), at = tile * 16 + rr, col = b * 64 + 32 * (j & 1) + 8 * t + c;
                uint32_t v = 8;
                if (at < n) {
                    if constexpr (QUANTS) {
                        const uint8_t byte = reinterpret_cast<const uint8_t *>(src)[((e * n + at) * (int64_t)k + col) >> 1];
                        v = (col & 1) ? byte >> 4 : byte & 15;
                    } else {
                        v = four_quant(__bfloat162float(reinterpret_cast<const bf16 *>(src)[(e * n + at) * (int64_t)k + col]), sm[(col / group) * 16 + rr]);
                    }
                }
                w[j] |= v << ((c & 1) * 16 + (c >> 1) * 4);
            }
        }
        *reinterpret_cast<uint4 *>(dst + (int64_t)b * record + 16 * (4 * r + (t ^ (r >> 1 & 3)))) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// values as f32 [experts][n][k]
__global__ void __launch_bounds__(256) linear4_read_kernel(const unsigned char *__restrict__ w, const float *__restrict__ row, int n, int k, int record, int tiles,
                                                           int64_t total, float *__restrict__ out)
{
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int col = (int)(i % k);
    const int64_t at = i / k, e = at / n;
    const int rr = (int)(at - e * n), tile = rr / 16, x = rr % 16, r = x % 8, hi = x / 8;
    const int64_t base = e * tiles + tile;
    const int b = col / 64, c = col % 64, t = c % 32 / 8, j = 2 * hi + c / 32, y = c % 8;
    const unsigned char *rec = w + (base * (k / 64) + b) * record;
    const uint32_t v = *reinterpret_cast<const uint32_t *>(rec + 16 * (4 * r + (t ^ (r >> 1 & 3))) + 4 * j) >> ((y & 1) * 16 + (y >> 1) * 4) & 15u;
    const __half s = reinterpret_cast<const __half *>(rec + 512)[(record > 544 ? c / 32 * 16 : 0) + 2 * r + hi];
    out[i] = __half2float(s) * row[base * 16 + x] * (float)((int)v - 8);
}

int32_t create(pg_ctx *ctx, const void *src, const void *scales, int64_t n, int64_t k, int64_t group, int64_t experts, pg_linear4 **out)
{
    PG_REQUIRE(out != nullptr, "linear4: out is null");
    *out = nullptr;
    PG_REQUIRE(src && n > 0 && k > 0 && experts > 0, "linear4: bad arguments");
    PG_REQUIRE(((uintptr_t)(scales ? scales : src) & 1) == 0, "linear4: bf16 numbers not aligned");
    PG_REQUIRE(group == 32 || group == 64 || group == 128, "linear4: groups of %lld (32, 64 or 128 are there)", (long long)group);
    PG_REQUIRE(k % 64 == 0 && k % group == 0, "linear4: K must be a multiple of 64 and of the group (K = %lld, groups of %lld)", (long long)k, (long long)group);
    PG_REQUIRE(n <= (1 << 24) && k <= (1 << 16) && experts <= 65535 && experts * n < (1ll << 31) - 4096, "linear4: shape too large");
    PG_REQUIRE(!ctx->capturing, "linear4: weights cannot be laid out while a graph is being recorded");
    pg_linear4 *l = new (std::nothrow) pg_linear4();
    if (!l) PG_FAIL(PG_ERR_NOMEM, "out of host memory");
    l->n = n, l->k = k, l->group = group, l->experts = experts, l->tiles = (n + 15) / 16, l->device = ctx->device;
    l->record = group == 32 ? 576 : 544;
    const size_t wb = (size_t)experts * l->tiles * (k / 64) * l->record, rb = (size_t)experts * l->tiles * 64;
    l->bytes = (int64_t)(wb + rb);
    int32_t rc = pg_splitk_reserve(ctx, std::max(pgk_linear4_gemv_workspace(l), pgk_linear4_tc_workspace(ctx)));
    if (rc == PG_OK) {
        const cudaError_t e = cudaMalloc(&l->mem, (size_t)pg_up(wb, 128) + rb);
        if (e != cudaSuccess) {
            cudaGetLastError();
            pg_set_error("linear4: %s", cudaGetErrorString(e));
            rc = e == cudaErrorMemoryAllocation ? PG_ERR_NOMEM : PG_ERR_CUDA;
        }
    }
    if (rc != PG_OK) {
        delete l;
        return rc;
    }
    unsigned char *p = (unsigned char *)l->mem;
    l->w = p;
    l->row = (const float *)(p + pg_up(wb, 128));
    const size_t smem = (size_t)(k / group * 16 + 16) * sizeof(float);
    const dim3 grid((unsigned)l->tiles, (unsigned)experts);
    auto go = [&](auto kern, std::atomic<uint64_t> &set) -> int32_t {
        PG_CUDA(pg_max_smem_once(kern, 160 * 1024, ctx->device, set));
        return launch_whole(ctx, kern, grid, dim3(128), smem, src, (const bf16 *)scales, (int)n, (int)k, (int)group, (int)l->record,
                            (unsigned char *)l->w, (float *)l->row);
    };
    static std::atomic<uint64_t> set_q{0}, set_w{0};
    rc = scales ? go(linear4_pack_kernel<true>, set_q) : go(linear4_pack_kernel<false>, set_w);
    // the source may be freed, and the weights read on other streams, when the call returns
    if (rc == PG_OK && cudaStreamSynchronize(ctx->stream) != cudaSuccess) {
        pg_set_error("linear4: %s", cudaGetErrorString(cudaGetLastError()));
        rc = PG_ERR_CUDA;
    }
    if (rc != PG_OK) {
        cudaFree(l->mem);
        delete l;
        return rc;
    }
    *out = l;
    return PG_OK;
}

int32_t check(const pg_ctx *ctx, const pg_linear4 *lin, const void *a, int32_t dtype, int32_t act, const void *y, int32_t y_dtype, int64_t ldy)
{
    PG_REQUIRE(lin && a && y, "linear4: null pointer");
    PG_REQUIRE(lin->device == ctx->device, "linear4: the weights are on device %d, the context on %d", lin->device, ctx->device);
    PG_REQUIRE(dtype == PG_BF16, "linear4: activations are bf16");
    PG_REQUIRE(y_dtype == PG_F32 || y_dtype == PG_BF16, "linear4: bad output type");
    PG_REQUIRE(act >= PG_ACT_NONE && act <= PG_ACT_CLAMPED_SWISH_GLU && (act == PG_ACT_NONE || (lin->n % 16 == 0 && y_dtype == PG_BF16)), "linear4: bad activation");
    PG_REQUIRE(ldy >= (act == PG_ACT_NONE ? lin->n : lin->n / 2) && ((uintptr_t)a & 15) == 0, "linear4: output rows too short or operand not aligned");
    PG_REQUIRE(((uintptr_t)y & (y_dtype == PG_BF16 ? 1 : 3)) == 0, "linear4: output not aligned");
    return PG_OK;
}

}  // namespace

extern "C" {

PG_API int32_t pg_linear4_pack(pg_ctx *ctx, const void *d_q, const void *d_scales_bf16, int64_t n, int64_t k, int64_t group, int64_t experts, pg_linear4 **out)
{
    PG_ENTER(ctx);
    PG_REQUIRE(d_scales_bf16 != nullptr, "linear4: bad arguments");
    return create(ctx, d_q, d_scales_bf16, n, k, group, experts, out);
}

PG_API int32_t pg_linear4_quantize(pg_ctx *ctx, const void *d_w_bf16, int64_t n, int64_t k, int64_t group, int64_t experts, pg_linear4 **out)
{
    PG_ENTER(ctx);
    return create(ctx, d_w_bf16, nullptr, n, k, group, experts, out);
}

PG_API int32_t pg_linear4_free(pg_ctx *ctx, pg_linear4 *lin)
{
    if (!lin) return PG_OK;
    PG_ENTER(ctx);
    PG_CUDA(cudaStreamSynchronize(ctx->stream));
    cudaFree(lin->mem);
    delete lin;
    return PG_OK;
}

PG_API int64_t pg_linear4_bytes(const pg_linear4 *lin) { return lin ? lin->bytes : 0; }

PG_API int32_t pg_linear4_read(pg_ctx *ctx, const pg_linear4 *lin, float *d_w)
{
    PG_ENTER(ctx);
    PG_REQUIRE(lin && d_w && ((uintptr_t)d_w & 3) == 0 && lin->device == ctx->device, "linear4_read: bad arguments");
    const int64_t total = lin->experts * lin->n * lin->k;
    PG_REQUIRE(total < (1ll << 31) * 256, "linear4_read: too many weights for one call");
    return launch_whole(ctx, linear4_read_kernel, dim3((unsigned)((total + 255) / 256)), dim3(256), 0, lin->w, lin->row, (int)lin->n, (int)lin->k, (int)lin->record,
                        (int)lin->tiles, total, d_w);
}

PG_API int32_t pg_linear4_run(pg_ctx *ctx, const pg_linear4 *lin, const void *d_a, int64_t lda, int32_t dtype, int64_t m, int32_t act, float limit, void *d_y,
                              int32_t y_dtype, int64_t ldy)
{
    PG_ENTER(ctx);
    const int32_t rc = check(ctx, lin, d_a, dtype, act, d_y, y_dtype, ldy);
    if (rc != PG_OK) return rc;
    PG_REQUIRE(lin->experts == 1, "linear4: a stack of experts takes a route");
    PG_REQUIRE(m >= 0 && m < (1ll << 31) - 256 && lda >= lin->k && lda % 8 == 0, "linear4: rows of a are %lld apart, K is %lld (and a multiple of 8 is wanted)", (long long)lda,
               (long long)lin->k);
    if (m == 0) return PG_OK;
    if (m <= 16) return pgk_linear4_gemv(ctx, lin, (const bf16 *)d_a, lda, m, act, limit, d_y, y_dtype, ldy, nullptr, 1);
    return pgk_linear4_tc(ctx, lin, (const bf16 *)d_a, lda, m, act, limit, d_y, y_dtype, ldy, nullptr, nullptr);
}

PG_API int32_t pg_linear4_run_routed(pg_ctx *ctx, const pg_linear4 *lin, const pg_route *route, const void *d_a, int32_t dtype, int32_t by_token, int32_t act, float limit,
                                     void *d_y, int32_t y_dtype, int64_t ldy)
{
    PG_ENTER(ctx);
    const int32_t rc = check(ctx, lin, d_a, dtype, act, d_y, y_dtype, ldy);
    if (rc != PG_OK) return rc;
    PG_REQUIRE(route && lin->experts == route->experts, "linear4: the route has another number of experts");
    if (route->m == 0) return PG_OK;
    const PgRouted rt = {route->blocks, route->block_expert, route->row_pair, (int)route->top, by_token};
    const int64_t pairs = route->m * route->top;
    if (route->block == PG_ROUTE_SMALL)
        return pgk_linear4_gemv(ctx, lin, (const bf16 *)d_a, lin->k, route->m, act, limit, d_y, y_dtype, ldy, &rt, pairs < route->experts ? pairs : route->experts);
    const int64_t rows = pg_route_rows(pairs, route->experts);
    PG_REQUIRE(rows <= route->max_rows, "linear4: the route is larger than it was created for");
    return pgk_linear4_tc(ctx, lin, (const bf16 *)d_a, lin->k, rows, act, limit, d_y, y_dtype, ldy, &rt, route);
}

}  // extern "C"
