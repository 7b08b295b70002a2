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
// Four of them, one question for all (2048 rows of 4096: 12 us with a question each and conversions, 11 so): y + 1.5 * 2^23 has the nearest whole number in its lowest bits
__device__ __forceinline__ int i8_code(float x, float a) { return (int)rint((double)x * 127.0 / (double)a); }
__device__ __forceinline__ unsigned i8_code4(const float4& v, float a, float r) {
    constexpr float M = 12582912.0f;
    const float y[4] = {v.x * r, v.y * r, v.z * r, v.w * r};
    float n[4], far = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        n[i] = y[i] + M;
        far = fmaxf(far, fabsf(y[i] - (n[i] - M)));
    }
    if (far < 0.49998f && a > 1e-30f)
        return __byte_perm(__byte_perm(__float_as_uint(n[0]), __float_as_uint(n[1]), 0x0040), __byte_perm(__float_as_uint(n[2]), __float_as_uint(n[3]), 0x0040), 0x5410);
    return ((unsigned)i8_code(v.x, a) & 255u) | ((unsigned)i8_code(v.y, a) & 255u) << 8 | ((unsigned)i8_code(v.z, a) & 255u) << 16 | (unsigned)i8_code(v.w, a) << 24;
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
                                             // an SM: 2048 rows of 4096 took 24 us instead of 11
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

// ---- one token: one kernel ------------------------------------------------------------------------------------------------------------------
// Every CTA codes the token by itself, into shared memory, while its first weights are on their way; a warp takes an output channel, 4096 codes of it at a time,
// the next ones under way behind the sums of these.  (From two tokens on the two kernels below are as fast or faster: this one with 2, 4 and 8 tokens against
// 11008 x 4096 took 18, 28 and 56 us, they take 17.  So they are where every CTA would code much: one token against 11008 x 4096 14 and 17 us, 4096 x 14336 23 and 18.)
#define I8_TOKEN_K 8192
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
__global__ void __launch_bounds__(I8_THREADS) i8_token_kernel(const int8_t* __restrict__ w, const float* __restrict__ ws, const float* __restrict__ x, float* __restrict__ out, int m, int k, int kp,
                                                              int vec) {
    extern __shared__ __align__(16) int8_t i8_codes[];              // [kp]
    __shared__ unsigned tops[I8_THREADS / 32];
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
    unsigned top = 0;
    for (int c = threadIdx.x * 4; c < k; c += I8_THREADS * 4) top = max(top, i8_top4(i8_load4(x, c, k, vec)));
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) tops[warp] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < I8_THREADS / 32; i++) top = max(top, tops[i]);
    const bool finite = top < 0x7f800000u, some = finite && top;
    const float a = __uint_as_float(top), xs = finite ? a / 127.0f : NAN;
    for (int c = threadIdx.x * 4; c < kp; c += I8_THREADS * 4) *(unsigned*)(i8_codes + c) = some ? i8_code4(i8_load4(x, c, k, vec), a, 127.0f / a) : 0u;
    __syncthreads();
    int acc = 0;
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
            const int4 v = *(const int4*)(i8_codes + c);
            acc = __dp4a(u[i].x, v.x, __dp4a(u[i].y, v.y, __dp4a(u[i].z, v.z, __dp4a(u[i].w, v.w, acc))));
        }
        if (seg) continue;
        const int sum = __reduce_add_sync(0xffffffffu, acc);
        if (lane == 0) out[r] = (float)sum * ws[r] * xs;
        acc = 0;
    }
}
static cudaError_t i8_launch_token(cc_device* dev, const int8_t* w, const float* ws, const float* x, float* out, int m, int k, int kp, int vec) {
    const int rows = I8_THREADS / 32;
    dev->launches++;
    return cc_launch_pdl(dev, i8_token_kernel, (unsigned)std::min<int64_t>((m + rows - 1) / rows, (int64_t)4 * dev->sm_count), I8_THREADS, (size_t)kp, w, ws, x, out, m, k, kp, vec);
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
__host__ __device__ constexpr int gi_ctas(int bn) { return bn <= 32 ? 2 : 1; }      // of an SM: narrow tiles are read from memory, and twice as many may share a depth
__host__ __device__ constexpr int gi_ring(int bn) { return (gi_ctas(bn) == 2 ? 112 : 192) * 1024 / ((128 + bn) * GI_K); }
__host__ __device__ constexpr int gi_stages(int bn) { return gi_ring(bn) < 8 ? gi_ring(bn) : 8; }
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
__global__ void __launch_bounds__(GI_THREADS, gi_ctas(BN)) i8_tile_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const float* __restrict__ ws,
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
    const int steps = (kp + GI_K - 1) / GI_K, slots = gi_ctas(BN) * dev->sm_count;
    int parts = 1;
    while (parts < 4 && tiles * parts * 2 <= slots && steps / (parts * 2) >= 2) parts *= 2;
    CC_REQUIRE(dev, tiles < ((int64_t)1 << 30), "product_i8: %lld tiles", (long long)tiles);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(parts > 1 ? tiles * parts : tiles < slots ? tiles : slots));
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

// ---- the same with two SMs on a tile ----------------------------------------------------------------------------------------------------------
// A step of 128 x 256 x 128 takes the tensor core 512 cycles and brings 48 KB, which are written to shared memory and read from it once: 750 cycles of its 128 bytes.  A pair of SMs (a
// cluster of two, cta_group::2) has 256 channels x BN tokens: each holds 128 channels and half of the tokens, 32 KB a step, and the pair's instruction reads both halves.  The
// even CTA issues the products; the copies of both are counted on its barriers, and what it commits arrives in both.
struct GpShared {
    unsigned long long full[8], empty[8], acc_full[2], acc_empty[2], drained;
    unsigned tmem_base;
    int fail;
};
__host__ __device__ constexpr int gp_bytes(int bn) { return (128 + bn / 2) * GI_K; }
__host__ __device__ constexpr int gp_stages(int bn) { return 192 * 1024 / gp_bytes(bn) < 8 ? 192 * 1024 / gp_bytes(bn) : 8; }
__host__ __device__ constexpr size_t gp_smem(int bn) { return (size_t)gp_stages(bn) * gp_bytes(bn) + 1024; }
__device__ __forceinline__ void gp_umma(unsigned tmem_d, uint64_t a, uint64_t b, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}\n" ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// what this thread has issued so far arrives on the barrier, when it is complete, in both CTAs
__device__ __forceinline__ void gp_commit(unsigned bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ unsigned gp_even(unsigned addr) {         // the even CTA's own of it
    unsigned a;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(a) : "r"(addr));
    return a;
}
__device__ __forceinline__ void gp_tma_load(unsigned dst, const void* tmap, unsigned bar, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(tmap), "r"(bar), "r"(x), "r"(y) : "memory");
}
template <int BN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GI_THREADS, 1) i8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_cut,
                                                                                         const float* __restrict__ ws, const float* __restrict__ xs, float* __restrict__ out, int T, int m, int steps, int n_whole, int cut,
                                                                                         int n_tiles, unsigned* err_dev, unsigned* err_host) {
    namespace cg = cooperative_groups;
    constexpr int ST = gp_stages(BN);
    constexpr unsigned A_BYTES = 128 * GI_K, BYTES = gp_bytes(BN), COLS = 2 * BN;
    extern __shared__ __align__(1024) uint8_t gi_raw[];
    __shared__ GpShared sh;
    uint8_t* ring = (uint8_t*)(((uintptr_t)gi_raw + 1023) & ~(uintptr_t)1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)cg::this_cluster().block_rank();
    const int tiles_n = (T + BN - 1) / BN, first = blockIdx.x / 2, stride = gridDim.x / 2;
    // the first n_whole tiles are 256 x BN, the ones behind them BN / cut wide
    auto place = [&](int tile, int& mt, int& n0) {
        const int of = tile < n_whole ? tile : n_whole + (tile - n_whole) / cut;
        mt = of / tiles_n;
        n0 = (of - mt * tiles_n) * BN + (tile < n_whole ? 0 : (tile - n_whole) % cut * (BN / cut));
        return tile < n_whole ? BN : BN / cut;
    };
    if (threadIdx.x == 0) {
        for (int i = 0; i < ST; i++) { pg_mbar_init(pg_smem(&sh.full[i]), 1); pg_mbar_init(pg_smem(&sh.empty[i]), 1); }
        for (int i = 0; i < 2; i++) { pg_mbar_init(pg_smem(&sh.acc_full[i]), 1); pg_mbar_init(pg_smem(&sh.acc_empty[i]), 8); }
        pg_mbar_init(pg_smem(&sh.drained), 1);
        sh.fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(pg_smem(&sh.tmem_base)), "n"(COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    pg_fence_before();
    __syncthreads();
    cg::this_cluster().sync();
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
                int mt, n0;
                const int wide = place(tile, mt, n0);
                for (int s = 0; s < steps; s++, g++) {
                    const unsigned slot = g % ST, own = pg_smem(&sh.full[slot]), full = gp_even(own), at = pg_smem(ring + (size_t)slot * BYTES);
                    if (!(ok = sg_wait(pg_smem(&sh.empty[slot]), ((g / ST) & 1u) ^ 1u, &sh.fail))) break;
                    if (rank == 0) pg_mbar_expect_tx(own, 2 * A_BYTES + wide * GI_K);
                    gp_tma_load(at, &map_w, full, s * GI_K, mt * 256 + rank * 128);
                    gp_tma_load(at + A_BYTES, wide == BN ? &map_x : &map_cut, full, s * GI_K, n0 + rank * (wide / 2));
                }
            }
            int never = 0;                                            // no copy is under way when the CTAs end (the even one sees those of both), and no arrival
            for (unsigned i = g > ST ? g - ST : 0; i < g; i++) {
                if (rank == 0) sg_wait(pg_smem(&sh.full[i % ST]), (i / ST) & 1u, &never);
                sg_wait(pg_smem(&sh.empty[i % ST]), (i / ST) & 1u, &never);
            }
            if (!ok || never)                                         // something did not come in time: a while for whatever is still to
                for (int i = 0; i < 1000; i++) __nanosleep(1000);
        }
        __syncwarp();
    } else if (warp == 1) {
        int never = 0;                                                // nothing is in flight when the TMEM is given back
        if (lane == 0 && rank == 1) sg_wait(pg_smem(&sh.drained), 0, &never);
        if (lane == 0 && rank == 0) {
            unsigned g = 0, nth = 0;
            bool ok = true;
            for (int tile = first; tile < n_tiles && ok; tile += stride, nth++) {
                int mt, n0;
                const unsigned acc = tmem + (nth & 1u) * BN, desc = gi_desc(place(tile, mt, n0)) + (8u << 24);
                if (!(ok = sg_wait(pg_smem(&sh.acc_empty[nth & 1u]), ((nth >> 1) & 1u) ^ 1u, &sh.fail))) break;
                pg_fence_after();
                for (int s = 0; s < steps; s++, g++) {
                    const unsigned slot = g % ST, at = pg_smem(ring + (size_t)slot * BYTES);
                    if (!(ok = sg_wait(pg_smem(&sh.full[slot]), (g / ST) & 1u, &sh.fail))) break;
                    pg_fence_after();
                    const uint64_t a = pg_smem_desc(at), b = pg_smem_desc(at + A_BYTES);
#pragma unroll
                    for (int kk = 0; kk < GI_K / 32; kk++) gp_umma(acc, a + 2 * kk, b + 2 * kk, desc, s > 0 || kk > 0);
                    gp_commit(pg_smem(&sh.empty[slot]));
                }
                if (ok) gp_commit(pg_smem(&sh.acc_full[nth & 1u]));
            }
            gp_commit(pg_smem(&sh.drained));
            sg_wait(pg_smem(&sh.drained), 0, &never);
        }
        __syncwarp();
    } else if (warp >= 4) {
        const int q = warp & 3;
        unsigned nth = 0;
        for (int tile = first; tile < n_tiles; tile += stride, nth++) {
            int mt, n0;
            const int wide = place(tile, mt, n0), row = mt * 256 + rank * 128 + q * 32 + lane;
            if (!sg_wait_warp(pg_smem(&sh.acc_full[nth & 1u]), (nth >> 1) & 1u, &sh.fail)) break;
            pg_fence_after();
            const unsigned from = tmem + (nth & 1u) * BN + ((unsigned)(q * 32) << 16);
            const float factor = row < m ? ws[row] : 0.0f;
#pragma unroll 1
            for (int c0 = 0; c0 < wide && n0 + c0 < T; c0 += 32) {
                unsigned v[32];
                gi_load<32>(from + c0, v);
                const float mine = n0 + c0 + lane < T ? xs[n0 + c0 + lane] : 0.0f;
                float* o = out + (int64_t)(n0 + c0) * m + row;
#pragma unroll
                for (int j = 0; j < 32; j++) {
                    const float f = __shfl_sync(0xffffffffu, mine, j);
                    if (row < m && n0 + c0 + j < T) *o = (float)(int)v[j] * factor * f;
                    o += m;
                }
            }
            pg_fence_before();                                        // the accumulator may be filled again
            __syncwarp();
            if (lane == 0) asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(gp_even(pg_smem(&sh.acc_empty[nth & 1u]))) : "memory");
        }
    }
    pg_fence_before();
    __syncthreads();
    cg::this_cluster().sync();
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(COLS) : "memory");
    if (threadIdx.x == 0 && sh.fail) {
        if (err_dev) atomicExch(err_dev, 5u);
        if (err_host) { *(volatile unsigned*)err_host = 5u; __threadfence_system(); }
    }
}
// tiles of 256 x 256, whole waves of them; those of the last one that is not full are cut across the tokens, as far as there are pairs: 2048 tokens, 14336 x 4096 are 6 waves of 74 and 4 tiles more
static int gp_launch(cc_device* dev, const int8_t* w, const float* ws, const int8_t* x, const float* xs, float* out, int T, int m, int kp) {
    constexpr int BN = 256;
    const int64_t tiles = (int64_t)((m + 255) / 256) * ((T + BN - 1) / BN);
    CC_REQUIRE(dev, tiles < ((int64_t)1 << 30), "product_i8: %lld tiles", (long long)tiles);
    const int pairs = dev->sm_count / 2, rest = (int)(tiles % pairs), whole = (int)tiles - rest;
    int cut = 1;
    while (cut < 8 && rest * cut * 2 <= pairs) cut *= 2;
    CUtensorMap mw, mx, mc;
    int rc = cc_make_tmap_i8(dev, &mw, w, m, kp, 128);
    if (!rc) rc = cc_make_tmap_i8(dev, &mx, x, T, kp, BN / 2);
    if (!rc) rc = cc_make_tmap_i8(dev, &mc, x, T, kp, BN / 2 / cut);
    if (rc) return rc;
    CC_CUDA(dev, cudaFuncSetAttribute(i8_pair_kernel<BN>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)gp_smem(BN)));
    CC_CUDA(dev, cc_launch_pdl(dev, i8_pair_kernel<BN>, (unsigned)(2 * std::min(whole + rest * cut, pairs)), GI_THREADS, gp_smem(BN), mw, mx, mc, ws, xs, out, T, m, (kp + GI_K - 1) / GI_K, whole, cut,
                               whole + rest * cut, dev->err_dev, dev->err_host));
    dev->launches++;
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
    if (T == 1 && k <= I8_TOKEN_K) {
        e = i8_launch_token(dev, w, ws, x, out, m, k, kp, vec);
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
    // Whole waves of tiles of 256 x 256 for pairs of SMs: those (2048 tokens, 14336 x 4096: 102 us instead of 115 with one SM a tile; 512 tokens, 11008 x 4096: 40 and 43).  Else tiles of 128
    // channels, whose depth a cluster shares where they are few (512 tokens, 4096 x 14336: 47 us, by pairs 59), as wide as the tokens: 16 columns cost a step what its weights cost
    else if (T > 128 && dev->sm_count > 1 && (int64_t)((m + 255) / 256) * ((T + 255) / 256) >= dev->sm_count / 2) rc = gp_launch(dev, w, ws, xq, xs, out, T, m, kp);
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
