// product.cu -- out = act(W x + bias) + residual in one call (include/crabml_seqops.h, cc_product), operands of 16 bits, sums of 32.
//
// Few rows (product_few_kernel): every weight is read once, so memory bounds it.  mma.sync.m16n8k16 with 16 rows of W as its first operand and 8 rows of x as the second: a lane takes
// 16 neighbouring bytes of a row of W straight into registers, and of a row of x from shared memory.  Which eight k a lane puts into two steps is free as long as both operands agree, so
// nothing is rearranged.  16 warps share the depth of 16 rows of W; their sums meet in shared memory, where bias, activation and residual follow.
// One row of 4096 x 4096 takes 9.7 us (a copy's rate would be 5.2: start, x into shared memory, the last tile's sums), two rows of 11008 x 4096 20 (4.5 TB/s).
#include <algorithm>

#include "act.cuh"
#include "half_types.cuh"
#include "umma.cuh"

struct PrArgs {
    const void *w, *x, *res;
    const float* bias;
    void* out;
    int64_t x_stride, res_stride;
    int m, k, rows, x_type, out_type, act;
    bool x_vec, w_vec;                        // rows start at multiples of 16 bytes
};
__device__ __forceinline__ float pr_finish(const PrArgs& a, float v, int row, int col) {
    if (a.bias) v += a.bias[col];
    v = act_apply(v, a.act);
    if (a.res) v += ht_read(a.res, (int64_t)row * a.res_stride + col, a.out_type);
    return v;
}
template <bool BF16>
__device__ __forceinline__ void pr_mma(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    if (BF16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <bool BF16>
__device__ __forceinline__ uint4 pr_pack8(const float (&v)[8]) {
    return BF16 ? make_uint4(ht_pack_bf16(v[0], v[1]), ht_pack_bf16(v[2], v[3]), ht_pack_bf16(v[4], v[5]), ht_pack_bf16(v[6], v[7]))
                : make_uint4(ht_pack_f16(v[0], v[1]), ht_pack_f16(v[2], v[3]), ht_pack_f16(v[4], v[5]), ht_pack_f16(v[6], v[7]));
}

#define PF_WARPS 16
#define PF_THREADS (PF_WARPS * 32)
#define PF_AHEAD 4                            // runs of 32 k that a warp has under way: 64 KB an SM
#define PF_ROWS 16
#define PF_ALONE (96 * 1024)
#define PF_ROOM (32 * 1024)
#define PF_ROOM_ODD (64 * 1024)
// Whether rows of x are few.  More, or longer ones, take tiles on the tensor cores, where an instruction takes all of x instead of 8 rows, and so do many rows of W, since every 16 of them cost
// a barrier here.  us, few / tiles, weights of 16-bit numbers:
// 4096 x 4096 with 1, 4, 8, 16 rows: 9.7 / 11.9, 10.7 / 12.0, 12.0 / 12.1, 15.1 / 12.3; 11008 x 4096 with 2, 16: 20.0 / 22.6, 25.1 / 21.8; 4096 x 14336 with 4: 27.0 / 24.7; 1024 x 1024 with 16: 6 / 7.7;
// 4096 x 1024 with 32: 9.9 / 9.0; one row: 8192 x 1024 8.4 / 8.9, 11008 x 1024 9.9 / 8.7, 11008 x 2048 12.9 / 13.2, 14336 x 2048 16.5 / 14.3, 131072 x 2048 110 / 86.  Rows of weights that start anywhere (k not a multiple of 8)
// are laid out for the tiles: 4096 x 255 with 16: 6.8 / 12.3; 4096 x 2047 with 16: 12.9 / 16.8; 14336 x 1023 with 16: 16.0 / 20.2; 4096 x 4095 with 1, 8: 13.7 / 23.3, 16.9 / 23.7; 14336 x 4095 with 8: 40 / 66;
// 4096 x 14335 with 1, 4: 35 / 67, 42 / 67
static bool pr_few(int64_t rows, int64_t m, int64_t k, bool w_vec) {
    return rows <= PF_ROWS && (!w_vec || m <= (k < 4096 ? 8192 : 12288)) && rows * k <= (!w_vec ? PF_ROOM_ODD : rows == 1 ? PF_ALONE : PF_ROOM);
}
// the two words of 16 bytes that hold n of 8 numbers of 16 bits, which start at any of them; neither is read without one of the n in it
__device__ __forceinline__ void pr_two_words(const uint16_t* from, int n, uint4& x, uint4& y) {
    x = y = make_uint4(0, 0, 0, 0);
    const int off = (int)((uintptr_t)from >> 1 & 7);
    const uint4* at = (const uint4*)((uintptr_t)from & ~(uintptr_t)15);
    if (n > 0) x = __ldg(at);
    if (n > 0 && off + min(n, 8) > 8) y = __ldg(at + 1);
}
// .. the numbers, zeros behind
__device__ __forceinline__ uint4 pr_join(const uint4& x, const uint4& y, int off, int n) {
    const unsigned w[7] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z};
    unsigned h[6], v[5];
#pragma unroll
    for (int j = 0; j < 6; j++) h[j] = off & 2 ? w[j + 1] : w[j];
    const unsigned last = off & 2 ? y.w : y.z;
#pragma unroll
    for (int j = 0; j < 5; j++) v[j] = off & 4 ? (j < 4 ? h[j + 2] : last) : h[j];
    unsigned r[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        r[j] = __funnelshift_r(v[j], v[j + 1], (off & 1) * 16);
        r[j] = 2 * j + 1 < n ? r[j] : 2 * j < n ? r[j] & 0xffffu : 0u;
    }
    return make_uint4(r[0], r[1], r[2], r[3]);
}
// rows of x into shared memory as 16-bit numbers, zeros behind the end of the last run
template <bool BF16>
__device__ __forceinline__ void pf_stage(const PrArgs& a, uint8_t* to, int pitch, int runs) {
    for (int e = threadIdx.x; e < a.rows * runs * 4; e += PF_THREADS) {
        const int r = e / (runs * 4), col = e % (runs * 4) * 8;
        float x[8] = {};
        const int64_t at = (int64_t)r * a.x_stride + col;
        if (col + 8 <= a.k) ht_read8(a.x, at, a.x_type, a.x_vec, x);
        else
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (col + j < a.k) x[j] = ht_read(a.x, at + j, a.x_type);
        *(uint4*)(to + r * pitch + col * 2) = pr_pack8<BF16>(x);
    }
}
// A CTA walks over the tiles of 16 rows of W blockIdx.x, + gridDim.x, ..; its warps take a tile's runs of 32 k by turns.
// PF_AHEAD runs of a warp are computed while the next ones, also of the next tile, are under way: 64 KB an SM and more.  ODD (rows of W start anywhere): a lane's 8 numbers lie in two words
__host__ __device__ constexpr int pf_pitch(int k) { return (k + 63) / 64 * 128 + 64; }      // eight lanes' 16 bytes: two rows, 64 bytes each, in all banks
template <int NT, bool BF16, bool ODD>
__global__ void __launch_bounds__(PF_THREADS, 1) product_few_kernel(const __grid_constant__ PrArgs a) {
    extern __shared__ __align__(16) uint8_t pf_raw[];
    __shared__ float sums[2][PF_WARPS][16][NT * 8 + 1];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, pitch = pf_pitch(a.k);
    const int tiles = (a.m + 15) >> 4, all = (a.k + 31) >> 5, mine = (all - warp + PF_WARPS - 1) / PF_WARPS;      // runs of a tile, and this warp's
    const uint8_t* x_lane = pf_raw + min(lane >> 2, a.rows - 1) * pitch + (lane & 3) * 16;        // rows behind the last one: any, no one reads their sums
    int z = 0;
    auto finish = [&](int tile, const float (&total)[NT][4]) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < 4; j++) sums[z][warp][(lane >> 2) + (j >> 1) * 8][n * 8 + (lane & 3) * 2 + (j & 1)] = total[n][j];
        __syncthreads();
        for (int e = tid; e < 16 * a.rows; e += PF_THREADS) {
            const int i = e & 15, n = e >> 4, col = tile * 16 + i;
            float s = 0.0f;
#pragma unroll
            for (int w = 0; w < PF_WARPS; w++) s += sums[z][w][i][n];
            if (col < a.m) ht_write(a.out, (int64_t)n * a.m + col, a.out_type, pr_finish(a, s, n, col));
        }
        z ^= 1;
    };
    auto multiply = [&](float (&acc)[NT][4], const uint4& u, const uint4& v, int run) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const uint4 b = *(const uint4*)((n == 0 ? x_lane : pf_raw + min(n * 8 + (lane >> 2), a.rows - 1) * pitch + (lane & 3) * 16) + run * 64);
            pr_mma<BF16>(acc[n], u.x, v.x, u.y, v.y, b.x, b.y);
            pr_mma<BF16>(acc[n], u.z, v.z, u.w, v.w, b.z, b.w);
        }
    };
    // the tensor cores cut a sum off at 24 bits after every 16 terms, always towards zero: sums of 128 terms go to registers and are rounded there (14336 terms of one sign: off by 1.1e-5 in
    // one chain a warp)
    constexpr int AHEAD = ODD ? PF_AHEAD / 2 : PF_AHEAD;
    uint4 u[AHEAD], v[AHEAD], u2[AHEAD], v2[AHEAD];                  // (the second words: ODD)
    const int64_t half = (int64_t)8 * a.k;
    auto load = [&](uint4 (&x)[AHEAD], uint4 (&y)[AHEAD], uint4 (&x2)[AHEAD], uint4 (&y2)[AHEAD], int tile, int i0) {
        // rows behind the last one: the last one again, no one reads their sums
        const uint16_t* w = (const uint16_t*)a.w + (int64_t)min(tile * 16 + (lane >> 2), a.m - 1) * a.k;
        const int64_t lower = tile * 16 + (lane >> 2) + 8 < a.m ? half : 0;
#pragma unroll
        for (int i = 0; i < AHEAD; i++) {
            const int c = (warp + (i0 + i) * PF_WARPS) * 32 + (lane & 3) * 8, n = tile < tiles ? a.k - c : 0;
            if (ODD) {
                pr_two_words(w + c, n, x[i], x2[i]);
                pr_two_words(w + lower + c, n, y[i], y2[i]);
            } else {
                x[i] = y[i] = make_uint4(0, 0, 0, 0);
                if (n > 0) {
                    const int4 p = ld_stream_16(w + c), q = ld_stream_16(w + lower + c);
                    x[i] = make_uint4((unsigned)p.x, (unsigned)p.y, (unsigned)p.z, (unsigned)p.w); y[i] = make_uint4((unsigned)q.x, (unsigned)q.y, (unsigned)q.z, (unsigned)q.w);
                }
            }
        }
    };
    pdl_enter();
    load(u, v, u2, v2, blockIdx.x, 0);
    pf_stage<BF16>(a, pf_raw, pitch, all);
    __syncthreads();
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int off = ODD ? (int)((uintptr_t)a.w / 2 + (unsigned)min(tile * 16 + (lane >> 2), a.m - 1) * (unsigned)a.k) & 7 : 0;      // (of the row 8 below, too)
        float total[NT][4] = {};
        for (int i0 = 0; i0 < mine; i0 += AHEAD) {
            uint4 nu[AHEAD], nv[AHEAD], nu2[AHEAD], nv2[AHEAD];
            const bool over = i0 + AHEAD >= mine;
            load(nu, nv, nu2, nv2, over ? tile + (int)gridDim.x : tile, over ? 0 : i0 + AHEAD);
            float acc[NT][4] = {};
#pragma unroll
            for (int i = 0; i < AHEAD; i++) {
                const int run = warp + (i0 + i) * PF_WARPS, n = a.k - run * 32 - (lane & 3) * 8;
                if (run < all) multiply(acc, ODD ? pr_join(u[i], u2[i], off, n) : u[i], ODD ? pr_join(v[i], v2[i], off, n) : v[i], run);      // (one for the warp)
            }
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 4; j++) total[n][j] += acc[n][j];
#pragma unroll
            for (int i = 0; i < AHEAD; i++) { u[i] = nu[i]; v[i] = nv[i]; u2[i] = nu2[i]; v2[i] = nv2[i]; }
        }
        if (mine <= 0) load(u, v, u2, v2, tile + (int)gridDim.x, 0);
        finish(tile, total);
    }
}
template <int NT>
static cudaError_t pf_launch(cc_device* dev, const PrArgs& a, bool bf16) {
    constexpr int room = NT == 1 ? pf_pitch(PF_ALONE) : PF_ROWS * 192 + PF_ROOM_ODD * 2;
    auto kernel = a.w_vec ? (bf16 ? product_few_kernel<NT, true, false> : product_few_kernel<NT, false, false>) : (bf16 ? product_few_kernel<NT, true, true> : product_few_kernel<NT, false, true>);
    cudaError_t e = cc_smem_limit(dev, CC_LIMIT_PRODUCT_FEW + (NT - 1) * 4 + bf16 * 2 + a.w_vec, kernel, room);
    if (e == cudaSuccess) e = cc_launch_pdl(dev, kernel, (unsigned)std::min((a.m + 15) / 16, dev->sm_count), PF_THREADS, (size_t)a.rows * pf_pitch(a.k), a);
    dev->launches++;
    return e;
}

#include "product_tile.cuh"

// rows of any of the types and any stride -> rows of `to` 16-bit numbers, zeros behind their k: what TMA can read
template <bool BF16>
__global__ void __launch_bounds__(256) product_rows_kernel(const void* __restrict__ x, int64_t stride, int type, int vec, int k, int to, int64_t n8, uint4* __restrict__ out) {
    pdl_enter();
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n8) return;
    const int64_t row = i / (to / 8);
    const int c = (int)(i - row * (to / 8)) * 8;
    if (type == (BF16 ? CC_BF16 : CC_F16)) {                         // (number by number, 4096 rows of 4095 took 26 us, so 11)
        const uint16_t* from = (const uint16_t*)x + row * stride + c;
        uint4 u, v;
        pr_two_words(from, k - c, u, v);
        out[i] = pr_join(u, v, (int)((uintptr_t)from >> 1 & 7), k - c);
        return;
    }
    float v[8] = {};
    if (c + 8 <= k) ht_read8(x, row * stride + c, type, vec, v);
    else
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (c + j < k) v[j] = ht_read(x, row * stride + c + j, type);
    out[i] = pr_pack8<BF16>(v);
}
static cudaError_t pr_rows(cc_device* dev, bool bf16, const void* x, int64_t stride, int type, bool vec, int64_t rows, int k, int to, void* out) {
    const int64_t n8 = rows * (to / 8);
    dev->launches++;
    return cc_launch_pdl(dev, bf16 ? product_rows_kernel<true> : product_rows_kernel<false>, (unsigned)((n8 + 255) / 256), 256, 0, x, stride, type, (int)vec, k, to, n8, (uint4*)out);
}
// clusters of 4 and of 8 CTAs, an SM each, that run at a time
template <bool BF16, bool DRAIN>
static int pt_clusters(cc_device* dev, int (&n)[2]) {
    if (!dev->clusters[0]) {
        auto kernel = product_pair_kernel<BF16, DRAIN>;
        CC_CUDA(dev, cc_smem_limit(dev, CC_LIMIT_PRODUCT_PAIR + BF16 * 2 + DRAIN, kernel, (int)pt_smem(256, true)));
        int found[2] = {0, 0};
        for (int i = 0; i < 2; i++) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(1024); cfg.blockDim = dim3(pt_threads(256, DRAIN)); cfg.dynamicSmemBytes = pt_smem(256, true);
            cudaLaunchAttribute at[1];
            at[0].id = cudaLaunchAttributeClusterDimension;
            at[0].val.clusterDim.x = 4u << i; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
            cfg.attrs = at; cfg.numAttrs = 1;
            CC_CUDA(dev, cudaOccupancyMaxActiveClusters(&found[i], kernel, &cfg));
        }
        dev->clusters[0] = std::max(found[0], 1); dev->clusters[1] = found[1];
    }
    n[0] = std::min(dev->clusters[0], dev->sm_count / 4); n[1] = std::min(dev->clusters[1], dev->sm_count / 8);
    return CC_OK;
}
template <int BN, bool BF16, bool DRAIN>
static int pt_launch(cc_device* dev, const PrArgs& a, const void* w, const void* x, int64_t x_stride, int kp, int parts) {
    CUtensorMap mw, mx;
    int rc = cc_make_tmap_rows(dev, &mw, w, a.m, a.k, (int64_t)kp * 2, 128, BF16);
    if (!rc) rc = cc_make_tmap_rows(dev, &mx, x, a.rows, a.k, x_stride * 2, BN, BF16);
    if (rc) return rc;
    const int64_t tiles = (int64_t)((a.m + 127) / 128) * ((a.rows + BN - 1) / BN);
    const int steps = (a.k + 63) / 64;
    CC_REQUIRE(dev, tiles < ((int64_t)1 << 30), "product: %lld tiles", (long long)tiles);
    auto kernel = product_tile_kernel<BN, BF16, DRAIN>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(parts > 1 ? tiles * parts : std::min<int64_t>(tiles, dev->sm_count)));
    cfg.blockDim = dim3(pt_threads(BN, DRAIN)); cfg.dynamicSmemBytes = pt_smem(BN, false); cfg.stream = dev->stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = dev->pdl ? 1 : 0;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)parts; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 2;
    CC_CUDA(dev, cc_smem_limit(dev, CC_LIMIT_PRODUCT_TILE + (BN == 32 ? 0 : BN == 64 ? 4 : BN == 128 ? 8 : 12) + BF16 * 2 + DRAIN, kernel, (int)pt_smem(BN, false)));
    CC_CUDA(dev, cudaLaunchKernelEx(&cfg, kernel, mw, mx, a, steps, (int)tiles, parts, dev->err_dev, dev->err_host));
    CC_LAUNCH_CHECK(dev);
    return CC_OK;
}
template <bool BF16, bool DRAIN>
static int pt_launch_pair(cc_device* dev, const PrArgs& a, const void* w, const void* x, int64_t x_stride, int kp, int parts) {
    const int64_t tiles = (int64_t)((a.m + 255) / 256) * ((a.rows + 255) / 256);
    CC_REQUIRE(dev, tiles < ((int64_t)1 << 28), "product: %lld tiles", (long long)tiles);
    const int pairs = dev->sm_count / 2, rest = parts > 1 ? 0 : (int)(tiles % pairs), whole = (int)tiles - rest;
    int cut = 1;
    while (cut < 4 && rest * cut * 2 <= pairs) cut *= 2;             // pieces of 64 rows: 16 for each group of the warps that finish
    CUtensorMap mw, mx, mc;
    int rc = cc_make_tmap_rows(dev, &mw, w, a.m, a.k, (int64_t)kp * 2, 128, BF16);
    if (!rc) rc = cc_make_tmap_rows(dev, &mx, x, a.rows, a.k, x_stride * 2, 128, BF16);
    if (!rc) rc = cc_make_tmap_rows(dev, &mc, x, a.rows, a.k, x_stride * 2, 128 / cut, BF16);
    if (rc) return rc;
    auto kernel = product_pair_kernel<BF16, DRAIN>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * (parts > 1 ? tiles * parts : std::min(whole + rest * cut, pairs))));
    cfg.blockDim = dim3(pt_threads(256, DRAIN)); cfg.dynamicSmemBytes = pt_smem(256, true); cfg.stream = dev->stream;
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = dev->pdl ? 1 : 0;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = (unsigned)(2 * parts); at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 2;
    CC_CUDA(dev, cc_smem_limit(dev, CC_LIMIT_PRODUCT_PAIR + BF16 * 2 + DRAIN, kernel, (int)pt_smem(256, true)));
    CC_CUDA(dev, cudaLaunchKernelEx(&cfg, kernel, mw, mx, mc, a, (a.k + 63) / 64, whole, cut, whole + rest * cut, parts, dev->err_dev, dev->err_host));
    CC_LAUNCH_CHECK(dev);
    return CC_OK;
}
// Several SMs share a tile's depth where there are too few tiles for all of them and the depth is worth the joining of their sums.  us, one / two / four parts (F32 results in brackets):
// 64 rows: 4096 x 512 7.8 / 7.9 / 9.1, x 4096 23.2 / 16.5 / 14.3, x 14336 80 / 42 / 29; eight where that many clusters run at a time:
// 16 rows of 1024 x 14336, four / eight 23 / 17; of 512 x 4096 10.7 / 10
template <int BN, bool BF16, bool DRAIN>
static int pt_single(cc_device* dev, const PrArgs& a, const void* w, const void* x, int64_t x_stride, int kp) {
    const int64_t tiles = (int64_t)((a.m + 127) / 128) * ((a.rows + BN - 1) / BN);
    const int steps = (a.k + 63) / 64;
    int parts = 1, at_once[2];
    while (parts < 4 && tiles * parts * 2 <= dev->sm_count && steps / (parts * 2) >= 4) parts *= 2;
    if (parts == 4 && steps >= 64 && 7 * (pt_workers(BN, DRAIN) / 4) * 16 * 128 * 4 <= pt_stages(BN, false) * pt_bytes(BN, false)) {      // (seven others' sums of a run of each group lie in the ring)
        const int rc = pt_clusters<BF16, DRAIN>(dev, at_once);
        if (rc) return rc;
        if (tiles <= at_once[1]) parts = 8;
    }
    return pt_launch<BN, BF16, DRAIN>(dev, a, w, x, x_stride, kp, parts);
}
// More than 128 rows go to pairs of SMs: 512 rows of 1024 x 512 take 13.8 us (13.1) on one SM each, 7.9 (11.3) on pairs.  Four parts where that many clusters of 8 SMs run at a time (16 of them took
// two rounds: 256 rows of 4096 x 4096 36.6 us), and else four SMs a tile of 128 channels: 512 rows of 1024 x 4096: pairs 20.7 (28.7), in two parts 23.6 (20.6), in four 19.2 (18.1), four SMs 18.6 (18.6);
// 256 rows of 4096 x 14336: pairs 55.9 (75.1), in two parts 47.8 (44.9), four SMs 38.4 (38.5).  512 rows of 1024 x 512: pairs 7.9 (11.3), in four parts 14.4 (13.0), of 1024 x 1024 9.9 (13.6), 15.0 (13.8).
// Two parts where four do not fit: 512 rows of 4096 x 4096 23.7 (32.6) / 25.5 (22.7), of 4096 x 14336 68.9 (88.2) / 55.9 (52.1)
template <bool BF16, bool DRAIN>
static int pt_tiles(cc_device* dev, const PrArgs& a, const void* w, const void* x, int64_t x_stride, int kp) {
    if (a.rows <= 32) return pt_single<32, BF16, DRAIN>(dev, a, w, x, x_stride, kp);
    if (a.rows <= 64) return pt_single<64, BF16, DRAIN>(dev, a, w, x, x_stride, kp);
    if (a.rows <= 128) return pt_single<128, BF16, DRAIN>(dev, a, w, x, x_stride, kp);
    const int64_t tiles = (int64_t)((a.m + 255) / 256) * ((a.rows + 255) / 256), singles = (int64_t)((a.m + 127) / 128) * ((a.rows + 255) / 256);
    const int steps = (a.k + 63) / 64;
    if (dev->sm_count < 2) return pt_launch<256, BF16, DRAIN>(dev, a, w, x, x_stride, kp, 1);      // (a device held to one SM)
    if (steps >= (DRAIN ? 16 : 64)) {
        int at_once[2];
        const int rc = pt_clusters<BF16, DRAIN>(dev, at_once);
        if (rc) return rc;
        if (tiles <= at_once[1]) return pt_launch_pair<BF16, DRAIN>(dev, a, w, x, x_stride, kp, 4);
        if (singles * 4 <= dev->sm_count) return pt_launch<256, BF16, DRAIN>(dev, a, w, x, x_stride, kp, 4);
        if (tiles <= at_once[0] && steps >= (DRAIN ? 16 : 96)) return pt_launch_pair<BF16, DRAIN>(dev, a, w, x, x_stride, kp, 2);
    }
    return pt_launch_pair<BF16, DRAIN>(dev, a, w, x, x_stride, kp, 1);
}
static int pr_many(cc_device* dev, const PrArgs& a, bool bf16) {
    // operands that TMA cannot read, or x of another type, are laid out first
    const int kp = (a.k + 7) / 8 * 8, type = bf16 ? CC_BF16 : CC_F16;
    const bool copy_w = kp != a.k || ((uintptr_t)a.w & 15), copy_x = kp != a.k || a.x_type != type || !a.x_vec;
    const size_t wb = copy_w ? (size_t)a.m * kp * 2 : 0, xb = copy_x ? (size_t)a.rows * kp * 2 : 0;
    void* mem = nullptr; size_t cls = 0;
    if (wb + xb) {
        const int rc = cc_pool_alloc(dev, wb + xb, &mem, &cls);
        if (rc) return rc;
    }
    const void *w = a.w, *x = a.x;
    int64_t x_stride = a.x_stride;
    cudaError_t e = cudaSuccess;
    if (copy_w) { e = pr_rows(dev, bf16, a.w, a.k, type, a.w_vec, a.m, a.k, kp, mem); w = mem; }
    if (copy_x && e == cudaSuccess) { x = (uint8_t*)mem + wb; e = pr_rows(dev, bf16, a.x, a.x_stride, a.x_type, a.x_vec, a.rows, a.k, kp, (void*)x); x_stride = kp; }
    int rc = e == cudaSuccess ? CC_OK : cc_fail(dev, CC_ERR_CUDA, "product: %s", cudaGetErrorString(e));
    const bool drain = a.out_type == CC_F32;
    if (!rc) rc = bf16 ? (drain ? pt_tiles<true, true>(dev, a, w, x, x_stride, kp) : pt_tiles<true, false>(dev, a, w, x, x_stride, kp))
                       : (drain ? pt_tiles<false, true>(dev, a, w, x, x_stride, kp) : pt_tiles<false, false>(dev, a, w, x, x_stride, kp));
    if (mem) cc_pool_free(dev, mem, cls);
    return rc;
}

extern "C" CC_API int cc_product(cc_device* dev, const cc_view* w, const cc_view* x, const cc_view* bias, int32_t act, const cc_view* residual, int32_t out_type, cc_buf** out) {
    if (!dev) return CC_ERR_ARG;
    CC_ENTER(dev);
    if (!out) return cc_fail(dev, CC_ERR_ARG, "product: out is NULL");
    *out = nullptr;
    if (LAZY(dev)) return cc_fail(dev, CC_ERR_UNSUPPORTED, "product: not available on a lazy (graph / megakernel) device");
    HT_ROWS(dev, x, "product x");
    if (!view_ok(w)) return cc_fail(dev, CC_ERR_ARG, "product: bad view of w");
    const bool bf16 = w->buf->dtype == CC_BF16;
    CC_REQUIRE(dev, bf16 || w->buf->dtype == CC_F16, "product: weights of type %d (F16 or BF16)", w->buf->dtype);
    HT_WHOLE(dev, w, w->buf->dtype, "product w");
    CC_REQUIRE(dev, w->ndim == 2 && w->shape[1] == x->shape[1], "product: w is not [rows, %lld]", (long long)x->shape[1]);
    const int64_t m = w->shape[0], k = w->shape[1], T = x->shape[0];
    CC_REQUIRE(dev, m >= 1 && m < (1 << 27) && k >= 1 && k < (1 << 27) && T < (1 << 27), "product: %lld rows of %lld by %lld", (long long)T, (long long)k, (long long)m);
    CC_REQUIRE(dev, ht_plain(out_type), "product: results of type %d (F32, F16 or BF16)", out_type);
    CC_REQUIRE(dev, act >= CC_ACT_NONE && act <= CC_ACT_RELU_SQUARED, "product: activation %d", act);
    if (bias) {
        HT_WHOLE(dev, bias, CC_F32, "product bias");
        CC_REQUIRE(dev, view_len(bias) == m, "product: bias is not [%lld]", (long long)m);
    }
    if (residual) {
        HT_ROWS(dev, residual, "product residual");
        CC_REQUIRE(dev, residual->buf->dtype == out_type && residual->shape[0] == T && residual->shape[1] == m, "product: residual is not [%lld, %lld] of the result's type", (long long)T, (long long)m);
    }
    cc_buf* o = nullptr;
    int rc = cc_new_activation(dev, T * m, out_type, false, &o);
    if (rc) return rc;
    if (T > 0) {
        PrArgs a{};
        a.w = w->buf->plane[0]; a.x = x->buf->plane[0]; a.res = residual ? residual->buf->plane[0] : nullptr; a.bias = bias ? (const float*)bias->buf->plane[0] : nullptr;
        a.out = o->base; a.x_stride = x->strides[0]; a.res_stride = residual ? residual->strides[0] : 0; a.m = (int)m; a.k = (int)k; a.rows = (int)T;
        a.x_type = x->buf->dtype; a.out_type = out_type; a.act = act;
        a.w_vec = k % 8 == 0 && ((uintptr_t)a.w & 15) == 0; a.x_vec = a.x_stride * ht_size(a.x_type) % 16 == 0 && ((uintptr_t)a.x & 15) == 0;
        if (!pr_few(T, m, k, a.w_vec)) rc = pr_many(dev, a, bf16);
        else {
            const cudaError_t e = T <= 8 ? pf_launch<1>(dev, a, bf16) : pf_launch<2>(dev, a, bf16);
            if (e != cudaSuccess) rc = cc_fail(dev, CC_ERR_CUDA, "product: %s", cudaGetErrorString(e));
        }
    }
    if (rc) { cc_tensor_release(o); return rc; }
    *out = o;
    return CC_OK;
}
