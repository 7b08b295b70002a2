// product_i8.cu -- products in 8-bit integers (cc_product_i8 of include/crabml_seqops.h): activations coded row by row, exact integer sums, one factor per token
// and one per output channel.
#include <cooperative_groups.h>
#include <cuda.h>
#include <math.h>

#include <algorithm>

#include "../../include/crabml_seqops.h"
#include "capi_checks.cuh"
#include "split_gemm.cuh"

// ---- activations -> codes ------------------------------------------------------------------------------------------------------------------
// round(127 x / a), ties to even, as the exact quotient rounds.  127 / a and the product err by less than 2e-5 of a step; where that leaves it open, and for rows whose
// 127 / a is no ordinary number, the quotient is taken in 64 bits: two 24-bit numbers' quotient that is not a tie is 2^-25 of itself away from one at least.
__device__ __forceinline__ int i8_code(float x, float a, float r) {
    const float y = x * r, n = rintf(y);
    if (fabsf(y - n) < 0.49998f && a > 1e-30f) return (int)n;
    return (int)rint((double)x * 127.0 / (double)a);
}
__device__ __forceinline__ unsigned i8_code4(const float4& v, float a, float r) {
    return ((unsigned)i8_code(v.x, a, r) & 255u) | ((unsigned)i8_code(v.y, a, r) & 255u) << 8 | ((unsigned)i8_code(v.z, a, r) & 255u) << 16 | (unsigned)i8_code(v.w, a, r) << 24;
}
__device__ __forceinline__ unsigned i8_top4(const float4& v) {
    const unsigned x = __float_as_uint(v.x) & 0x7fffffffu, y = __float_as_uint(v.y) & 0x7fffffffu, z = __float_as_uint(v.z) & 0x7fffffffu, w = __float_as_uint(v.w) & 0x7fffffffu;
    return max(max(x, y), max(z, w));
}
// four numbers of a row of k from c on, zeros behind it
__device__ __forceinline__ float4 i8_load4(const float* row, int c, int k, bool vec) {
    if (vec && c + 4 <= k) return *(const float4*)(row + c);
    return make_float4(c < k ? row[c] : 0.0f, c + 1 < k ? row[c + 1] : 0.0f, c + 2 < k ? row[c + 2] : 0.0f, c + 3 < k ? row[c + 3] : 0.0f);
}
#define I8_THREADS 256
#define I8_KEEP 4                            // float4 of a row that a thread keeps: rows of up to 16 THREADS are read once.  16 of them, 256 threads for all rows, left two CTAs
                                             // an SM: 2048 rows of 4096 took 24 us instead of I8_ROWS_US
// codes [T][kp], zeros behind a row's k; factors [T].  A CTA a row
template <int THREADS>
__global__ void __launch_bounds__(THREADS) i8_rows_kernel(const float* __restrict__ x, int64_t rs, int k, int kp, int vec, int8_t* __restrict__ codes, float* __restrict__ factors) {
    __shared__ unsigned tops[THREADS / 32];
    pdl_enter();
    const int64_t t = blockIdx.x;
    const float* row = x + t * rs;
    unsigned top = 0;
    float4 keep[I8_KEEP];
#pragma unroll
    for (int i = 0; i < I8_KEEP; i++) {
        const int c = (i * THREADS + threadIdx.x) * 4;
        if (i * THREADS * 4 >= k) break;
        keep[i] = i8_load4(row, c, k, vec);
    }
#pragma unroll
    for (int i = 0; i < I8_KEEP; i++) {
        if (i * THREADS * 4 >= k) break;
        top = max(top, i8_top4(keep[i]));
    }
    for (int c = (I8_KEEP * THREADS + threadIdx.x) * 4; c < k; c += THREADS * 4) top = max(top, i8_top4(i8_load4(row, c, k, vec)));
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 32; w++) top = max(top, tops[w]);
    const bool finite = top < 0x7f800000u, some = finite && top;
    const float a = __uint_as_float(top), r = 127.0f / a;
    unsigned* to = (unsigned*)(codes + t * kp);
#pragma unroll
    for (int i = 0; i < I8_KEEP; i++) {
        const int c = (i * THREADS + threadIdx.x) * 4;
        if (c < kp) to[c >> 2] = some && c < k ? i8_code4(keep[i], a, r) : 0u;
    }
    for (int c = (I8_KEEP * THREADS + threadIdx.x) * 4; c < kp; c += THREADS * 4) to[c >> 2] = some ? i8_code4(i8_load4(row, c, k, vec), a, r) : 0u;
    if (threadIdx.x == 0) factors[t] = finite ? a / 127.0f : NAN;
}

// ---- up to I8_FEW tokens: one kernel ------------------------------------------------------------------------------------------------------------
// Every CTA codes the tokens by itself, into shared memory, while its first weights are on their way; a warp takes an output channel, 4096 codes of it at a time,
// the next ones under way behind the sums of these.
#define I8_FEW 8
#define I8_RUN 8                             // pieces of 16 codes of a lane: 4096 codes of a warp
// 16 codes of a row that may start anywhere: the five words around them; near the end of the matrix byte by byte
__device__ __forceinline__ int4 i8_load16(const int8_t* p, const int8_t* end) {
    if (p + 20 <= end) {
        const unsigned* u = (const unsigned*)((uintptr_t)p & ~(uintptr_t)3);
        const unsigned s = ((unsigned)(uintptr_t)p & 3u) * 8u, u0 = u[0], u1 = u[1], u2 = u[2], u3 = u[3], u4 = s ? u[4] : 0u;
        return make_int4((int)__funnelshift_r(u0, u1, s), (int)__funnelshift_r(u1, u2, s), (int)__funnelshift_r(u2, u3, s), (int)__funnelshift_r(u3, u4, s));
    }
    int z[4] = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 16; j++)
        if (p + j < end) z[j / 4] |= (int)(uint8_t)p[j] << (j % 4 * 8);
    return make_int4(z[0], z[1], z[2], z[3]);
}
template <int TB>
__global__ void __launch_bounds__(I8_THREADS) i8_few_kernel(const int8_t* __restrict__ w, const float* __restrict__ ws, const float* __restrict__ x, int64_t rs, float* __restrict__ out, int T,
                                                            int m, int k, int kp, int vec) {
    extern __shared__ __align__(16) int8_t i8_codes[];              // [TB][kp]
    __shared__ unsigned tops[I8_THREADS / 32][TB];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = gridDim.x * (I8_THREADS / 32), segs = (k + 4095) >> 12;
    const bool wide = (k & 15) == 0;
    const int8_t* end = w + (int64_t)m * k;
    int row = blockIdx.x * (I8_THREADS / 32) + warp, seg = 0;
    int4 next[I8_RUN];
    auto fetch = [&](int r, int s) {
#pragma unroll
        for (int i = 0; i < I8_RUN; i++) {
            const int c = s * 4096 + i * 512 + lane * 16;
            if (r < m && c < k) next[i] = wide ? ld_stream_16(w + (int64_t)r * k + c) : i8_load16(w + (int64_t)r * k + c, end);
        }
    };
    pdl_enter();
    fetch(row, 0);
    float xs[TB];
#pragma unroll
    for (int t = 0; t < TB; t++) {
        unsigned top = 0;
        if (t < T)
            for (int c = threadIdx.x * 4; c < k; c += I8_THREADS * 4) top = max(top, i8_top4(i8_load4(x + t * rs, c, k, vec)));
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) tops[warp][t] = top;
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TB; t++) {
        unsigned top = 0;
#pragma unroll
        for (int i = 0; i < I8_THREADS / 32; i++) top = max(top, tops[i][t]);
        const bool finite = top < 0x7f800000u, some = finite && top && t < T;
        const float a = __uint_as_float(top), r = 127.0f / a;
        for (int c = threadIdx.x * 4; c < kp; c += I8_THREADS * 4) *(unsigned*)(i8_codes + t * kp + c) = some ? i8_code4(i8_load4(x + t * rs, c, k, vec), a, r) : 0u;
        xs[t] = finite ? a / 127.0f : NAN;
    }
    __syncthreads();
    int acc[TB];
#pragma unroll
    for (int t = 0; t < TB; t++) acc[t] = 0;
    while (row < m) {
        int4 u[I8_RUN];
#pragma unroll
        for (int i = 0; i < I8_RUN; i++) u[i] = next[i];
        const int s = seg, r = row;
        if (++seg == segs) { seg = 0; row += warps; }
        fetch(row, seg);
#pragma unroll
        for (int i = 0; i < I8_RUN; i++) {
            const int c = s * 4096 + i * 512 + lane * 16;
            if (c >= k) break;
#pragma unroll
            for (int t = 0; t < TB; t++) {
                const int4 v = *(const int4*)(i8_codes + t * kp + c);
                acc[t] = __dp4a(u[i].x, v.x, __dp4a(u[i].y, v.y, __dp4a(u[i].z, v.z, __dp4a(u[i].w, v.w, acc[t]))));
            }
        }
        if (seg) continue;
        const float factor = ws[r];
#pragma unroll
        for (int t = 0; t < TB; t++) {
            const int sum = __reduce_add_sync(0xffffffffu, acc[t]);
            if (lane == 0 && t < T) out[(int64_t)t * m + r] = (float)sum * factor * xs[t];
            acc[t] = 0;
        }
    }
}
template <int TB>
static cudaError_t i8_launch_few(cc_device* dev, const int8_t* w, const float* ws, const float* x, int64_t rs, float* out, int T, int m, int k, int kp, int vec) {
    const size_t smem = (size_t)TB * kp;
    const int per = (int)std::min<size_t>(4, 200 * 1024 / (smem + 1024)), rows = I8_THREADS / 32;
    const int64_t grid = std::min<int64_t>((m + rows - 1) / rows, (int64_t)per * dev->sm_count);
    cudaError_t e = cudaSuccess;
    if (smem > 48 * 1024) e = cudaFuncSetAttribute(i8_few_kernel<TB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) e = cc_launch_pdl(dev, i8_few_kernel<TB>, (unsigned)grid, I8_THREADS, smem, w, ws, x, rs, out, T, m, k, kp, vec);
    dev->launches++;
    return e;
}

// ---- many rows: tcgen05.mma on 8-bit tiles -----------------------------------------------------------------------------------------------------
// A tile is 128 output channels (the instruction's rows, TMEM's lanes) x BN tokens; a step of 128 codes of both comes by TMA into a ring, one thread issues
// four instructions of 32 codes for it (kind::i8, 32-bit integer accumulators in TMEM), four warps finish.  Lanes are neighbouring channels: an output row is stored
// 128 bytes at a time.  A CTA walks over tiles with two accumulators, so that a tile's end overlaps the next one's steps.  Few tiles: a cluster shares the
// depth of one, each CTA sends the others the integer sums of the lanes that they finish, and any order gives the same sum.
// Every wait is bounded (sg_wait): on expiry the CTA raises `fail`, all roles leave their loops, TMEM is freed and the host reports it.
#define GI_THREADS 256
#define GI_K 128
struct GiShared {
    unsigned long long full[8], empty[8], acc_full[2], acc_empty[2], drained;
    unsigned tmem_base;
    int fail;
};
__host__ __device__ constexpr int gi_stages(int bn) { return 192 * 1024 / ((128 + bn) * GI_K) < 8 ? 192 * 1024 / ((128 + bn) * GI_K) : 8; }
__host__ __device__ constexpr size_t gi_smem(int bn) { return (size_t)gi_stages(bn) * (128 + bn) * GI_K + 1024; }
__device__ __forceinline__ void gi_umma(unsigned tmem_d, uint64_t a, uint64_t b, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// 32-bit integer accumulator, signed 8-bit A and B, both K-major
__host__ __device__ constexpr unsigned gi_desc(int n) { return (2u << 4) | (1u << 7) | (1u << 10) | ((unsigned)(n >> 3) << 17) | (8u << 24); }

template <int N>
__device__ __forceinline__ void gi_load(unsigned addr, unsigned (&v)[N]) {
    static_assert(N == 16 || N == 32, "");
    sg_tmem16(addr, *(unsigned(*)[16])v);
    if (N == 32) sg_tmem16(addr + 16, *(unsigned(*)[16])(v + N - 16));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; i++) asm volatile("" : "+r"(v[i]));       // nothing is done with them before
}

template <int BN>
__global__ void __launch_bounds__(GI_THREADS, 1) i8_tile_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const float* __restrict__ ws,
                                                                const float* __restrict__ xs, float* __restrict__ out, int T, int m, int steps_all, int n_tiles, int parts, unsigned* err_dev,
                                                                unsigned* err_host) {
    namespace cg = cooperative_groups;
    constexpr int ST = gi_stages(BN), RUN = BN < 32 ? BN : 32;
    constexpr unsigned A_BYTES = 128 * GI_K, B_BYTES = BN * GI_K, COLS = 2 * BN < 32 ? 32 : 2 * BN;
    extern __shared__ __align__(1024) uint8_t gi_raw[];
    __shared__ GiShared sh;
    uint8_t* ring = (uint8_t*)(((uintptr_t)gi_raw + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = parts > 1 ? (int)cg::this_cluster().block_rank() : 0;
    const int s0 = (int)((int64_t)steps_all * part / parts), steps = (int)((int64_t)steps_all * (part + 1) / parts) - s0;
    const int tiles_n = (T + BN - 1) / BN, first = blockIdx.x / parts, stride = gridDim.x / parts;
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; i++) { pg_mbar_init(pg_smem(&sh.full[i]), 1); pg_mbar_init(pg_smem(&sh.empty[i]), 1); }
        for (int i = 0; i < 2; i++) { pg_mbar_init(pg_smem(&sh.acc_full[i]), 1); pg_mbar_init(pg_smem(&sh.acc_empty[i]), 4); }
        pg_mbar_init(pg_smem(&sh.drained), 1);
        sh.fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(pg_smem(&sh.tmem_base)), "n"(COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pg_fence_before();
    __syncthreads();
    pg_fence_after();
    const unsigned tmem = sh.tmem_base;
    pdl_enter();
    if (warp == 0) {
        if (lane == 0) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
            unsigned g = 0;
            bool ok = true;
            for (int tile = first; tile < n_tiles && ok; tile += stride) {
                const int mt = tile / tiles_n, nt = tile - mt * tiles_n;
                for (int s = 0; s < steps; s++, g++) {
                    const unsigned slot = g % ST, full = pg_smem(&sh.full[slot]), at = pg_smem(ring + (size_t)slot * (A_BYTES + B_BYTES));
                    if (!(ok = sg_wait(pg_smem(&sh.empty[slot]), ((g / ST) & 1u) ^ 1u, &sh.fail))) break;
                    pg_mbar_expect_tx(full, A_BYTES + B_BYTES);
                    pg_tma_load_2d(at, &map_w, full, (s0 + s) * GI_K, mt * 128);
                    pg_tma_load_2d(at + A_BYTES, &map_x, full, (s0 + s) * GI_K, nt * BN);
                }
            }
            int never = 0;                                            // no copy is under way when the CTA ends
            for (unsigned i = g > ST ? g - ST : 0; i < g; i++) sg_wait(pg_smem(&sh.full[i % ST]), (i / ST) & 1u, &never);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            unsigned g = 0, nth = 0;
            bool ok = true;
            for (int tile = first; tile < n_tiles && ok; tile += stride, nth++) {
                const unsigned acc = tmem + (nth & 1u) * BN;
                if (!(ok = sg_wait(pg_smem(&sh.acc_empty[nth & 1u]), ((nth >> 1) & 1u) ^ 1u, &sh.fail))) break;
                pg_fence_after();
                for (int s = 0; s < steps; s++, g++) {
                    const unsigned slot = g % ST, at = pg_smem(ring + (size_t)slot * (A_BYTES + B_BYTES));
                    if (!(ok = sg_wait(pg_smem(&sh.full[slot]), (g / ST) & 1u, &sh.fail))) break;
                    pg_fence_after();
                    const uint64_t a = pg_smem_desc(at), b = pg_smem_desc(at + A_BYTES);
#pragma unroll
                    for (int kk = 0; kk < GI_K / 32; kk++) gi_umma(acc, a + 2 * kk, b + 2 * kk, gi_desc(BN), s > 0 || kk > 0);
                    pg_umma_commit(pg_smem(&sh.empty[slot]));
                }
                if (ok) pg_umma_commit(pg_smem(&sh.acc_full[nth & 1u]));
            }
            int never = 0;                                            // nothing of this CTA is in flight when its TMEM is given back
            pg_umma_commit(pg_smem(&sh.drained));
            sg_wait(pg_smem(&sh.drained), 0, &never);
        }
        __syncwarp();
    } else if (warp >= 4 && parts == 1) {
        const int q = warp & 3;
        unsigned nth = 0;
        for (int tile = first; tile < n_tiles; tile += stride, nth++) {
            const int mt = tile / tiles_n, n0 = (tile - mt * tiles_n) * BN, row = mt * 128 + q * 32 + lane;
            if (!sg_wait_warp(pg_smem(&sh.acc_full[nth & 1u]), (nth >> 1) & 1u, &sh.fail)) break;
            pg_fence_after();
            const unsigned from = tmem + (nth & 1u) * BN + ((unsigned)(q * 32) << 16);
            const float factor = row < m ? ws[row] : 0.0f;
#pragma unroll 1
            for (int c0 = 0; c0 < BN && n0 + c0 < T; c0 += RUN) {
                unsigned v[RUN];
                gi_load<RUN>(from + c0, v);
                const float mine = lane < RUN && n0 + c0 + lane < T ? xs[n0 + c0 + lane] : 0.0f;
                if (c0 + RUN >= BN || n0 + c0 + RUN >= T) {           // the last of the accumulator: it may be filled again
                    pg_fence_before();
                    sg_arrive(pg_smem(&sh.acc_empty[nth & 1u]));
                }
                float* o = out + (int64_t)(n0 + c0) * m + row;
#pragma unroll
                for (int j = 0; j < RUN; j++) {
                    const float f = __shfl_sync(0xffffffffu, mine, j);
                    if (row < m && n0 + c0 + j < T) *o = (float)(int)v[j] * factor * f;
                    o += m;
                }
            }
        }
    }
    if (parts > 1) {                                                  // one tile: CTA p finishes the lanes of its 4 / parts warps
        cg::cluster_group cluster = cg::this_cluster();
        const int q = warp & 3, owners = 4 / parts, owner = q / owners, mt = first / tiles_n, n0 = (first - mt * tiles_n) * BN, row = mt * 128 + q * 32 + lane;
        if (warp >= 4) sg_wait_warp(pg_smem(&sh.acc_full[0]), 0, &sh.fail);
        pg_fence_after();
        __syncthreads();
        const int bad = *(volatile int*)&sh.fail;
        cluster.sync();                                               // every CTA's products are done: the rings are free
        const unsigned from = tmem + ((unsigned)(q * 32) << 16);
        // [sender][warp of the owner][column][lane]
        auto box = [&](int from_part, int at_part) { return ((size_t)(from_part < at_part ? from_part : from_part - 1) * owners + q % owners) * BN * 32; };
        if (warp >= 4 && owner != part) {
            int* to = cluster.map_shared_rank((int*)ring, owner) + box(part, owner);
#pragma unroll 1
            for (int c0 = 0; c0 < BN && n0 + c0 < T; c0 += RUN) {
                unsigned v[RUN];
                gi_load<RUN>(from + c0, v);
#pragma unroll
                for (int j = 0; j < RUN; j++) to[(c0 + j) * 32 + lane] = (int)v[j];
            }
        }
        cluster.sync();
        if (warp >= 4 && owner == part && !bad) {
            const float factor = row < m ? ws[row] : 0.0f;
#pragma unroll 1
            for (int c0 = 0; c0 < BN && n0 + c0 < T; c0 += RUN) {
                unsigned v[RUN];
                gi_load<RUN>(from + c0, v);
                const float mine = lane < RUN && n0 + c0 + lane < T ? xs[n0 + c0 + lane] : 0.0f;
                for (int p = 0; p < parts; p++) {
                    if (p == part) continue;
                    const int* o = (const int*)ring + box(p, part) + c0 * 32 + lane;
#pragma unroll
                    for (int j = 0; j < RUN; j++) v[j] += (unsigned)o[j * 32];
                }
                float* o = out + (int64_t)(n0 + c0) * m + row;
#pragma unroll
                for (int j = 0; j < RUN; j++) {
                    const float f = __shfl_sync(0xffffffffu, mine, j);
                    if (row < m && n0 + c0 + j < T) *o = (float)(int)v[j] * factor * f;
                    o += m;
                }
            }
        }
    }
    pg_fence_before();
    __syncthreads();
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(COLS) : "memory");
    if (threadIdx.x == 0 && sh.fail) {
        if (err_dev) atomicExch(err_dev, 5u);
        if (err_host) { *(volatile unsigned*)err_host = 5u; __threadfence_system(); }
    }
}
template <int BN>
static int gi_launch(cc_device* dev, const int8_t* w, const float* ws, const int8_t* x, const float* xs, float* out, int T, int m, int kp) {
    CUtensorMap mw, mx;
    int rc = cc_make_tmap_i8(dev, &mw, w, m, kp, 128);
    if (!rc) rc = cc_make_tmap_i8(dev, &mx, x, T, kp, BN);
    if (rc) return rc;
    const int64_t tiles = (int64_t)((m + 127) / 128) * ((T + BN - 1) / BN);
    const int steps = (kp + GI_K - 1) / GI_K;
    int parts = 1;
    while (parts < 4 && tiles * parts * 2 <= dev->sm_count && steps / (parts * 2) >= 2) parts *= 2;
    CC_REQUIRE(dev, tiles < ((int64_t)1 << 30), "product_i8: %lld tiles", (long long)tiles);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(parts > 1 ? tiles * parts : tiles < dev->sm_count ? tiles : dev->sm_count));
    cfg.blockDim = dim3(GI_THREADS); cfg.dynamicSmemBytes = gi_smem(BN); cfg.stream = dev->stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = dev->pdl ? 1 : 0;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)parts; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 2;
    CC_CUDA(dev, cudaFuncSetAttribute(i8_tile_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)gi_smem(BN)));
    CC_CUDA(dev, cudaLaunchKernelEx(&cfg, i8_tile_kernel<BN>, mw, mx, ws, xs, out, T, m, steps, (int)tiles, parts, dev->err_dev, dev->err_host));
    CC_LAUNCH_CHECK(dev);
    return CC_OK;
}
// rows of k codes -> rows of kp, zeros behind: what TMA can read where k is no multiple of 16
__global__ void i8_pad_kernel(const int8_t* __restrict__ w, int8_t* __restrict__ to, int64_t n4, int k, int kp4) {
    pdl_enter();
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= n4) return;
    const int64_t row = i / kp4;
    const int c = (int)(i - row * kp4) * 4;
    unsigned u = 0;
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (c + j < k) u |= (unsigned)(uint8_t)w[row * k + c + j] << (8 * j);
    ((unsigned*)to)[i] = u;
}

static int i8_product(cc_device* dev, const int8_t* w, const float* ws, const float* x, int64_t rs, float* out, int T, int m, int k) {
    const int kp = (k + 15) / 16 * 16, vec = rs % 4 == 0 && ((uintptr_t)x & 15) == 0;
    cudaError_t e;
    if (T <= I8_FEW && (size_t)(T <= 1 ? 1 : T <= 2 ? 2 : T <= 4 ? 4 : 8) * kp <= 160 * 1024) {
        e = T <= 1 ? i8_launch_few<1>(dev, w, ws, x, rs, out, T, m, k, kp, vec) : T <= 2 ? i8_launch_few<2>(dev, w, ws, x, rs, out, T, m, k, kp, vec)
            : T <= 4 ? i8_launch_few<4>(dev, w, ws, x, rs, out, T, m, k, kp, vec) : i8_launch_few<8>(dev, w, ws, x, rs, out, T, m, k, kp, vec);
        return e == cudaSuccess ? CC_OK : cc_fail(dev, CC_ERR_CUDA, "product_i8: %s", cudaGetErrorString(e));
    }
    const bool pad = k != kp;
    const size_t codes = ((size_t)T * kp + 255) / 256 * 256, factors = ((size_t)T * 4 + 255) / 256 * 256;
    void* mem = nullptr; size_t cls = 0;
    int rc = cc_pool_alloc(dev, codes + factors + (pad ? (size_t)m * kp : 0), &mem, &cls);
    if (rc) return rc;
    int8_t* xq = (int8_t*)mem;
    float* xs = (float*)((uint8_t*)mem + codes);
    e = k <= 4096 ? cc_launch_pdl(dev, i8_rows_kernel<256>, (unsigned)T, 256, 0, x, rs, k, kp, vec, xq, xs)
        : k <= 8192 ? cc_launch_pdl(dev, i8_rows_kernel<512>, (unsigned)T, 512, 0, x, rs, k, kp, vec, xq, xs) : cc_launch_pdl(dev, i8_rows_kernel<1024>, (unsigned)T, 1024, 0, x, rs, k, kp, vec, xq, xs);
    dev->launches++;
    if (pad && e == cudaSuccess) {
        int8_t* wp = (int8_t*)mem + codes + factors;
        const int64_t n4 = (int64_t)m * (kp / 4);
        e = cc_launch_pdl(dev, i8_pad_kernel, (unsigned)((n4 + 255) / 256), 256, 0, w, wp, n4, k, kp / 4);
        dev->launches++;
        w = wp;
    }
    if (e != cudaSuccess) rc = cc_fail(dev, CC_ERR_CUDA, "product_i8: %s", cudaGetErrorString(e));
    else rc = T <= 16 ? gi_launch<16>(dev, w, ws, xq, xs, out, T, m, kp) : T <= 32 ? gi_launch<32>(dev, w, ws, xq, xs, out, T, m, kp)
              : T <= 64 ? gi_launch<64>(dev, w, ws, xq, xs, out, T, m, kp) : T <= 128 ? gi_launch<128>(dev, w, ws, xq, xs, out, T, m, kp) : gi_launch<256>(dev, w, ws, xq, xs, out, T, m, kp);
    cc_pool_free(dev, mem, cls);
    return rc;
}

extern "C" CC_API int cc_product_i8(cc_device* dev, const cc_view* w, const cc_view* w_scale, const cc_view* x, cc_buf** out) {
    if (!dev) return CC_ERR_ARG;
    CC_ENTER(dev);
    if (LAZY(dev)) return cc_fail(dev, CC_ERR_UNSUPPORTED, "product_i8: not available on a lazy (graph / megakernel) device");
    if (!out) return cc_fail(dev, CC_ERR_ARG, "product_i8: out is NULL");
    *out = nullptr;
    if (!view_ok(w) || !view_ok(w_scale) || !view_ok(x)) return cc_fail(dev, CC_ERR_ARG, "product_i8: bad tensor view");
    CC_REQUIRE(dev, view_in_bounds(w) && view_in_bounds(w_scale) && view_in_bounds(x), "product_i8: a view addresses elements behind its buffer");
    CC_REQUIRE(dev, w->buf->dev == dev && w_scale->buf->dev == dev && x->buf->dev == dev, "product_i8: a tensor of another device");
    CC_REQUIRE(dev, w->buf->dtype == CC_I8 && w->ndim == 2 && view_contiguous(w), "product_i8: w is not a contiguous I8 matrix");
    REQUIRE_F32(dev, w_scale, "product_i8 w_scale"); REQUIRE_F32(dev, x, "product_i8 x");
    const int64_t m = w->shape[0], k = w->shape[1], T = x->shape[0];
    CC_REQUIRE(dev, view_contiguous(w_scale) && view_len(w_scale) == m, "product_i8: w_scale is not [%lld]", (long long)m);
    CC_REQUIRE(dev, x->ndim == 2 && x->shape[1] == k && x->strides[1] == 1 && x->strides[0] >= k, "product_i8: x is not rows of %lld", (long long)k);
    CC_REQUIRE(dev, k >= 1 && k <= 131072 && m < ((int64_t)1 << 30) && T < ((int64_t)1 << 24), "product_i8: %lld rows, %lld x %lld", (long long)T, (long long)m, (long long)k);
    cc_buf* o = nullptr;
    int rc = cc_new_activation(dev, T * m, CC_F32, false, &o);
    if (rc) return rc;
    if (T > 0 && m > 0) rc = i8_product(dev, (const int8_t*)w->buf->plane[0], (const float*)w_scale->buf->plane[0], (const float*)x->buf->plane[0], x->strides[0], (float*)o->base, (int)T,
                                        (int)m, (int)k);
    if (rc) { cc_tensor_release(o); return rc; }
    *out = o;
    return CC_OK;
}
