// latent_attn.cu -- attention over pages of latent rows (include/crabml_paged.h), absorbed: the queries are carried over to the latents (latent_fold_kernel), the cached rows themselves
// are keys and values of all heads (latent_rows_kernel), and what comes out is carried back (latent_unfold_kernel).
//
// A row of the scores is a query of one head: 16 heads of one token are 16 rows over the same keys, one tile of mma.sync.m16n8k16.  One token of 16 heads over rows of 512 + 64
// makes 30 operations a byte of the cache, so bytes bound it, as long as every row comes from memory once: a CTA (one per SM) brings 32 rows at a time into a ring of shared memory
// by bulk copies, a warp of its own issuing them, and 8 warps take them twice, as keys and as values:
//   scores   warp w adds up the columns 16 (w % 4 + 4 i) of 16 keys (w / 4); the queries stay in registers, sums of the four column groups meet in shared memory
//   weights  a thread 2 (or 4) keys of a row: exp2(score - largest), rounded to f16, back to shared memory
//   values   warp w adds up the columns 16 (w + 8 i) of all rows in registers; scaled when a row's largest score grows
// One barrier a step: scores of step k and values of step k - 1 lie on the same side of it.
// All steps of a call are dealt out in equal runs over the SMs; sums of cut segments are joined by latent_join_kernel.
//
// Sums, largest scores and sums of weights have 32 bits; queries on their way to the latents are brought near 2^4 by a power of two and rounded to f16, weights are rounded to f16 near
// 2^10 (2^-11 of each: the operands of the tensor cores; the result is rounded to 16 bits anyway), sums of latents enter the last product as two f16 numbers.
#include <algorithm>

#include "latent.cuh"
#include "split_gemm.cuh"

#define LR_WARPS 8
#define LR_CONS (LR_WARPS * 32)
#define LR_THREADS (LR_CONS + 32)
#define LR_KEYS 32                            // of a step
#define LR_BEGIN 4                            // what a segment's begin and end cost, in steps
#define LR_SLOTS 8                            // most slots of the ring
#define LR_SMEM (226 * 1024)
#define LR_SHIFT 10.0f                        // weights are exp2(score - largest + LR_SHIFT)
#define LR_KB 9                               // column blocks of 16 of a warp's scores: (LT_RANK + LT_REST) / 16 / 4
#define LR_VB 4                               // .. of its values: LT_RANK / 16 / 8
#define LR_CTAS 160
#define LR_LOG2E 1.4426950408889634f

// runs of consecutive tokens whose sequences take this form
#define LT_RUNS 64
struct LtRuns { int n, tiles; int lo[LT_RUNS], hi[LT_RUNS], tile0[LT_RUNS]; };
struct LrArgs {
    const PgSeq* seqs;
    const int* table;
    const __half *rows, *q, *uk, *uv;
    const float* sink;
    float *qf, *lat, *part;                   // queries over the latents [T H][cols]; results over the latents [T H][rank]; sums of cut segments [2 x CTA][16 MT][rank]
    float2* ml;                               // [2 x CTA][16 MT]: largest score (base 2), sum of weights
    void* out;
    float scale;
    int n_seqs, table_cols, page, shift, H, dim, vdim, rank, rest, cols, window, most, out_bf16, slots;      // most: sequences with more new tokens take the other form
};
struct LrDeal { int ctas, run_lo, run_more; struct { int seq, tile, off; } at[LR_CTAS]; };
struct LrCuts { struct { int seq, tile, slot, cta, n; } at[LR_CTAS]; };

__host__ __device__ __forceinline__ void lr_range(const PgSeq& s, const LrArgs& a, int* from, int* to) {
    *to = s.pos0 + s.count;
    *from = a.window > 0 && s.pos0 - a.window + 1 > 0 ? s.pos0 - a.window + 1 : 0;
}
__host__ __device__ __forceinline__ int lr_tiles(const PgSeq& s, const LrArgs& a, int rows) { return s.count > a.most ? 0 : (int)(((int64_t)s.count * a.H + rows - 1) / rows); }
__host__ __device__ __forceinline__ int lr_steps(const PgSeq& s, const LrArgs& a) {
    int from, to;
    lr_range(s, a, &from, &to);
    return LR_BEGIN + (to - from + LR_KEYS - 1) / LR_KEYS;
}

__device__ __forceinline__ void lt_ldsm(unsigned (&r)[4], unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void lt_ldsm_t(unsigned (&r)[4], unsigned addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void lt_mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float lt_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ unsigned lt_pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *(const unsigned*)&h;
}
// x, y as f16 (h) and what is left of them as f16 (l); an infinity's or NaN's rest is NaN
__device__ __forceinline__ void lt_cut(float x, float y, unsigned& h, unsigned& l) {
    const __half2 a = __floats2half2_rn(x, y);
    const float2 b = __half22float2(a);
    h = *(const unsigned*)&a;
    l = lt_pack(x - b.x, y - b.y);
}
__device__ __forceinline__ void lt_copy16(unsigned dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void lt_copies_done() { asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ bool lt_tile(const LtRuns& runs, int tile, int* lo, int* hi) {
    for (int i = 0; i < runs.n; i++) {
        const int t = tile - runs.tile0[i];
        if (t >= 0 && runs.lo[i] + t * 16 < runs.hi[i]) { *lo = runs.lo[i] + t * 16; *hi = min(*lo + 16, runs.hi[i]); return true; }
    }
    return false;
}

// ---- queries to the latents, results back ---------------------------------------------------------------------------------------------------
// qf[t, h, :rank] = U_h^T n[t, h], qf[t, h, rank:] = p[t, h], in 32 bits.  grid (heads, blocks of 64 columns and one for p, tiles of 16 tokens by turns); a warp 16 columns
#define LF_COLS 64
__global__ void __launch_bounds__(128) latent_fold_kernel(const LrArgs a, const __grid_constant__ LtRuns runs) {
    extern __shared__ __align__(16) uint8_t lf_raw[];
    __half *bs = (__half*)lf_raw, *as = bs + a.dim * (LF_COLS + 8);      // U_h's rows, 64 columns of them; queries [16][dim + 8]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, h = blockIdx.x, c0 = blockIdx.y * LF_COLS, width = a.dim + a.rest;
    pdl_enter();
    if (c0 >= a.rank) {                                                  // p
        for (int tile = blockIdx.z; tile < runs.tiles; tile += gridDim.z) {
            int lo, hi;
            if (!lt_tile(runs, tile, &lo, &hi)) return;
            for (int e = tid; e < (hi - lo) * a.rest; e += 128) {
                const int64_t row = (int64_t)(lo + e / a.rest) * a.H + h;
                a.qf[row * a.cols + a.rank + e % a.rest] = __half2float(a.q[row * width + a.dim + e % a.rest]);
            }
        }
        return;
    }
    for (int e = tid; e < a.dim * (LF_COLS / 8); e += 128) {
        const int r = e / (LF_COLS / 8), c = e % (LF_COLS / 8) * 8;
        if (c0 + c < a.rank) lt_copy16(pg_smem(bs + r * (LF_COLS + 8) + c), a.uk + ((int64_t)h * a.dim + r) * a.rank + c0 + c);
    }
    for (int tile = blockIdx.z; tile < runs.tiles; tile += gridDim.z) {
        int lo, hi;
        if (!lt_tile(runs, tile, &lo, &hi)) return;
        __syncthreads();
        for (int e = tid; e < 16 * a.dim / 8; e += 128) {
            const int r = e / (a.dim / 8), c = e % (a.dim / 8) * 8;
            *(uint4*)(as + r * (a.dim + 8) + c) = lo + r < hi ? __ldg((const uint4*)(a.q + ((int64_t)(lo + r) * a.H + h) * width + c)) : make_uint4(0, 0, 0, 0);
        }
        lt_copies_done();
        __syncthreads();
        if (c0 + warp * 16 >= a.rank) continue;
        float acc[2][4] = {};
#pragma unroll 4
        for (int k = 0; k < a.dim; k += 16) {
            unsigned x[4], b[4];
            lt_ldsm(x, pg_smem(as + ((lane & 7) + (lane >> 3 & 1) * 8) * (a.dim + 8) + k + (lane >> 4) * 8));
            lt_ldsm_t(b, pg_smem(bs + (k + (lane & 7) + (lane >> 3 & 1) * 8) * (LF_COLS + 8) + warp * 16 + (lane >> 4) * 8));
            lt_mma(acc[0], x, b[0], b[1]);
            lt_mma(acc[1], x, b[2], b[3]);
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const int t = lo + (lane >> 2) + y * 8;
                if (t < hi) *(float2*)(a.qf + ((int64_t)t * a.H + h) * a.cols + c0 + warp * 16 + i * 8 + (lane & 3) * 2) = make_float2(acc[i][2 * y], acc[i][2 * y + 1]);
            }
    }
}
// out[t, h] = V_h lat[t, h].  grid (heads, blocks of 32 columns, tiles of 16 tokens by turns); a warp 8 columns
#define LU_COLS 32
__global__ void __launch_bounds__(128) latent_unfold_kernel(const LrArgs a, const __grid_constant__ LtRuns runs) {
    extern __shared__ __align__(16) uint8_t lf_raw[];
    const int pitch = a.rank + 8;
    __half *bs = (__half*)lf_raw, *as = bs + LU_COLS * pitch;          // V_h's rows; sums of latents [h, l][16][pitch]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, h = blockIdx.x, c0 = blockIdx.y * LU_COLS;
    pdl_enter();
    for (int e = tid; e < LU_COLS * (a.rank / 8); e += 128) {
        const int r = e / (a.rank / 8), c = e % (a.rank / 8) * 8;
        if (c0 + r < a.vdim) lt_copy16(pg_smem(bs + r * pitch + c), a.uv + ((int64_t)h * a.vdim + c0 + r) * a.rank + c);
        else *(uint4*)(bs + r * pitch + c) = make_uint4(0, 0, 0, 0);
    }
    for (int tile = blockIdx.z; tile < runs.tiles; tile += gridDim.z) {
        int lo, hi;
        if (!lt_tile(runs, tile, &lo, &hi)) break;
        __syncthreads();
        for (int e = tid; e < 16 * a.rank / 4; e += 128) {
            const int r = e / (a.rank / 4), c = e % (a.rank / 4) * 4;
            const float4 v = lo + r < hi ? *(const float4*)(a.lat + ((int64_t)(lo + r) * a.H + h) * a.rank + c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            uint2 x, y;
            lt_cut(v.x, v.y, x.x, y.x); lt_cut(v.z, v.w, x.y, y.y);
            *(uint2*)(as + r * pitch + c) = x;
            *(uint2*)(as + (16 + r) * pitch + c) = y;
        }
        lt_copies_done();
        __syncthreads();
        float acc[4] = {};
        const int r = (lane & 7) + (lane >> 3 & 1) * 8, kc = (lane >> 4) * 8;
#pragma unroll 4
        for (int k = 0; k < a.rank; k += 16) {
            unsigned x[4], y[4], b0, b1;
            lt_ldsm(x, pg_smem(as + r * pitch + k + kc));
            lt_ldsm(y, pg_smem(as + (16 + r) * pitch + k + kc));
            asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];" : "=r"(b0), "=r"(b1) : "r"(pg_smem(bs + (warp * 8 + (lane & 7)) * pitch + k + (lane >> 3 & 1) * 8)));
            lt_mma(acc, x, b0, b1);
            lt_mma(acc, y, b0, b1);
        }
        const int c = c0 + warp * 8 + (lane & 3) * 2;
#pragma unroll
        for (int y = 0; y < 2; y++) {
            const int t = lo + (lane >> 2) + y * 8;
            if (t < hi && c < a.vdim) *(unsigned*)((uint16_t*)a.out + ((int64_t)t * a.H + h) * a.vdim + c) = a.out_bf16 ? ht_pack_bf16(acc[2 * y], acc[2 * y + 1]) : ht_pack_f16(acc[2 * y], acc[2 * y + 1]);
        }
    }
}

// ---- the cached rows as keys and values ----------------------------------------------------------------------------------------------------------
template <int MT>
struct LrShared {
    unsigned long long full[LR_SLOTS], empty[LR_SLOTS];
    int fail;
    unsigned wild;                            // rows whose sums are not finite
    float top[16 * MT], sum[16 * MT], inv[16 * MT];      // of a segment: factor of a row's scores, then its largest score and sum of weights; what a row is divided by
    float alpha[2][16 * MT];
    __align__(16) float sums[2][4][16 * MT][40];      // of a step: scores by column groups
    __align__(16) __half p[2][16 * MT][40];
};
__device__ __forceinline__ void lr_sync() { asm volatile("bar.sync 1, %0;" ::"n"(LR_CONS) : "memory"); }
__device__ __forceinline__ bool lr_sync_or(bool x) {
    unsigned r;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbar.red.or.pred q, 1, %2, p;\nselp.u32 %0, 1, 0, q;\n}\n" : "=r"(r) : "r"((unsigned)x), "n"(LR_CONS) : "memory");
    return r;
}
// Values that are not finite, times the weight 0 of a row that does not see them, make a NaN.  Rows whose sums hold one though their scores do not are added up again, one by one, over
// the keys that they see: a dot product over the block, which then adds 2 columns a thread.
template <int MT>
__device__ __noinline__ void lr_again(const LrArgs& a, LrShared<MT>& sh, const PgSeq s, int seq, int row0, int lo, int hi, float* lat, int64_t lat_stride) {
    for (unsigned left = sh.wild; left; left &= left - 1) {
        const int r = __ffs(left) - 1, tok = (row0 + r) / a.H, pos = s.pos0 + tok;
        const float* q = a.qf + ((int64_t)s.first * a.H + row0 + r) * a.cols;
        const float m = sh.top[r];
        float o0 = 0.0f, o1 = 0.0f;
        const int c = threadIdx.x * 2;
        for (int key = max(lo, a.window > 0 ? pos - a.window + 1 : 0); key <= min(hi - 1, pos); key++) {
            const __half* row = a.rows + ((int64_t)a.table[(int64_t)seq * a.table_cols + (key >> a.shift)] * a.page + (key & (a.page - 1))) * a.cols;
            float d = 0.0f;
            for (int e = threadIdx.x; e < a.cols; e += LR_CONS) d = fmaf(q[e], __half2float(row[e]), d);
            d = warp_sum(d);
            if ((threadIdx.x & 31) == 0) sh.sums[0][0][0][threadIdx.x >> 5] = d;
            lr_sync();
            d = 0.0f;
#pragma unroll
            for (int w = 0; w < LR_WARPS; w++) d += sh.sums[0][0][0][w];
            lr_sync();
            const float p = lt_exp2(d * (a.scale * LR_LOG2E) - m + LR_SHIFT);
            if (c < a.rank) { o0 = fmaf(p, __half2float(row[c]), o0); o1 = fmaf(p, __half2float(row[c + 1]), o1); }
        }
        if (c < a.rank) { lat[r * lat_stride + c] = o0 * sh.inv[r]; lat[r * lat_stride + c + 1] = o1 * sh.inv[r]; }
    }
}

template <int MT>
__global__ void __launch_bounds__(LR_THREADS, 1) latent_rows_kernel(const __grid_constant__ LrArgs a, const __grid_constant__ LrDeal deal, unsigned* err_dev, unsigned* err_host) {
    extern __shared__ __align__(16) uint8_t lr_raw[];
    __shared__ LrShared<MT> sh;
    constexpr int ROWS = 16 * MT, LANES = LR_CONS / ROWS, PER = LR_KEYS / LANES;      // threads of a row in a step's weights, and the keys of each
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const unsigned pitch = (unsigned)a.cols * 2 + 16, ring = pg_smem(lr_raw), slot_bytes = LR_KEYS * pitch;      // a row's pitch is an odd number of 16 bytes: ldmatrix without conflicts
    if (tid == 0) {
        for (int i = 0; i < a.slots; i++) { pg_mbar_init(pg_smem(&sh.full[i]), 1); pg_mbar_init(pg_smem(&sh.empty[i]), LR_WARPS); }
        sh.fail = 0; sh.wild = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // keys behind a segment's last one have the weight 0, and zeros, or a row from before, in their place
    for (unsigned i = tid * 16; i < a.slots * slot_bytes; i += LR_THREADS * 16) *(uint4*)(lr_raw + i) = make_uint4(0, 0, 0, 0);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    pdl_enter();
    __syncthreads();
    const int c = blockIdx.x;
    int seq = deal.at[c].seq, tile = deal.at[c].tile, off = deal.at[c].off, left = deal.run_lo + (c < deal.run_more ? 1 : 0);
    unsigned slot = 0, phase = 0;
    bool ok = true;
    auto advance = [&]() { if (++slot == (unsigned)a.slots) { slot = 0; phase ^= 1u; } };
    // the segments of this CTA's run: body(sequence, first and last step of its keys, whether it is cut)
    auto walk = [&](auto body) {
        bool first = true;
        while (left > 0 && seq < a.n_seqs) {
            const PgSeq s = a.seqs[seq];
            const int tiles = lr_tiles(s, a, ROWS);
            if (tile >= tiles) { seq++; tile = 0; off = 0; continue; }
            const int all = lr_steps(s, a), take = min(left, all - off);
            body(s, max(off - LR_BEGIN, 0), max(off + take - LR_BEGIN, 0), off > LR_BEGIN || off + take < all, first);
            first = false;
            left -= take;
            if (off + take == all) { tile++; off = 0; } else off += take;
        }
    };
    if (warp == LR_WARPS) {
        // ===== copies: a lane a row =====
        int issued = 0;
        walk([&](const PgSeq& s, int k0, int k1, bool, bool) {
            int from, to;
            lr_range(s, a, &from, &to);
            const int* table = a.table + (int64_t)seq * a.table_cols;
            auto row_of = [&](int k) {
                const int key = from + k * LR_KEYS + lane;
                return key < to ? a.rows + ((int64_t)table[key >> a.shift] * a.page + (key & (a.page - 1))) * a.cols : nullptr;
            };
            const __half* next = k0 < k1 ? row_of(k0) : nullptr;
            for (int k = k0; k < k1; k++) {
                const __half* row = next;
                if (k + 1 < k1) next = row_of(k + 1);
                if (ok) ok = sg_wait_warp(pg_smem(&sh.empty[slot]), phase ^ 1u, &sh.fail);
                if (ok) {
                    const unsigned bar = pg_smem(&sh.full[slot]);
                    if (lane == 0) pg_mbar_expect_tx(bar, (unsigned)(min(LR_KEYS, to - (from + k * LR_KEYS)) * a.cols * 2));
                    __syncwarp();
                    if (row) asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                                          ::"r"(ring + slot * slot_bytes + lane * pitch), "l"(row), "r"((unsigned)a.cols * 2), "r"(bar) : "memory");
                    issued++;
                }
                advance();
            }
        });
        int never = 0;                                                    // no copy is under way when the CTA ends
        for (int i = max(0, issued - a.slots); i < issued; i++) sg_wait(pg_smem(&sh.full[i % a.slots]), (unsigned)(i / a.slots) & 1u, &never);
    } else {
        const int kg = warp & 3, kh = warp >> 2, blocks = a.cols >> 4, v_blocks = a.rank >> 4;
        const int row = tid / LANES, part = tid % LANES;                  // of the weights
        const unsigned k_lane = (unsigned)(kh * 16 + (lane >> 4) * 8 + (lane & 7)) * pitch + (lane >> 3 & 1) * 16;      // scores: this lane's row of four 8 x 8 blocks
        const unsigned v_lane = (unsigned)((lane >> 3 & 1) * 8 + (lane & 7)) * pitch + (lane >> 4) * 16;
        const unsigned p_lane = (unsigned)((lane >> 3 & 1) * 8 + (lane & 7)) * 80 + (lane >> 4) * 16;
        walk([&](const PgSeq& s, int k0, int k1, bool cut, bool first) {
            int from, to;
            lr_range(s, a, &from, &to);
            const int row0 = tile * ROWS, n_rows = min(ROWS, s.count * a.H - row0);
            const float* qs = a.qf + ((int64_t)s.first * a.H + row0) * a.cols;
            // factors of the rows: near 2^4 by a power of two
            lr_sync();                                                    // the segment before is through
            if (tid == 0) sh.wild = 0;
            for (int r = warp; r < ROWS; r += LR_WARPS) {
                unsigned top = 0;                                        // as bits, so that NaN is the largest of all
                if (r < n_rows)
                    for (int e = lane * 4; e < a.cols; e += 128) {
                        const uint4 v = *(const uint4*)(qs + (int64_t)r * a.cols + e);
                        top = max(max(top, max(v.x & 0x7fffffffu, v.y & 0x7fffffffu)), max(v.z & 0x7fffffffu, v.w & 0x7fffffffu));
                    }
                top = __reduce_max_sync(0xffffffffu, top);
                const int ex = top < 0x00800000u || top >= 0x7f800000u ? 4 : max((int)(top >> 23) - 126, -100);
                if (lane == 0) {
                    sh.inv[r] = __uint_as_float((unsigned)(4 - ex + 127) << 23);
                    sh.top[r] = top >= 0x7f800000u ? NAN : __uint_as_float((unsigned)(ex - 4 + 127) << 23);
                }
            }
            lr_sync();
            unsigned q[MT][LR_KB][4];
#pragma unroll
            for (int t = 0; t < MT; t++)
#pragma unroll
                for (int i = 0; i < LR_KB; i++) {
                    const int b = kg + 4 * i;
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        const int r = t * 16 + (lane >> 2) + (x & 1) * 8;
                        float2 v = make_float2(0.0f, 0.0f);
                        if (b < blocks && r < n_rows) v = *(const float2*)(qs + (int64_t)r * a.cols + b * 16 + (x >> 1) * 8 + (lane & 3) * 2);
                        q[t][i][x] = lt_pack(v.x * sh.inv[r], v.y * sh.inv[r]);
                    }
                }
            const float f = sh.top[row] * (a.scale * LR_LOG2E);
            const int pos = row < n_rows ? s.pos0 + (row0 + row) / a.H : -1, key_lo = a.window > 0 ? pos - a.window + 1 : 0;
            float m = -INFINITY, l = 0.0f;
            float o[MT][LR_VB][2][4];
#pragma unroll
            for (int t = 0; t < MT; t++)
#pragma unroll
                for (int i = 0; i < LR_VB; i++)
#pragma unroll
                    for (int x = 0; x < 8; x++) o[t][i][x >> 2][x & 3] = 0.0f;
            bool grew = false;
            unsigned v_slot = slot;
#pragma unroll 1
            for (int k = k0; k <= k1; k++) {
                const int z = k & 1;
                const unsigned here = slot;
                if (k < k1) {
                    ok = ok && sg_wait_warp(pg_smem(&sh.full[slot]), phase, &sh.fail);
                    float x[MT][2][4];
#pragma unroll
                    for (int t = 0; t < MT; t++)
#pragma unroll
                        for (int i = 0; i < 8; i++) x[t][i >> 2][i & 3] = 0.0f;
                    const unsigned at = ring + slot * slot_bytes + k_lane;
#pragma unroll
                    for (int i = 0; i < LR_KB; i++) {
                        const int b = kg + 4 * i;
                        if (b < blocks) {
                            unsigned kb[4];
                            lt_ldsm(kb, at + b * 32);
#pragma unroll
                            for (int t = 0; t < MT; t++) { lt_mma(x[t][0], q[t][i], kb[0], kb[1]); lt_mma(x[t][1], q[t][i], kb[2], kb[3]); }
                        }
                    }
#pragma unroll
                    for (int t = 0; t < MT; t++)
#pragma unroll
                        for (int n = 0; n < 2; n++)
#pragma unroll
                            for (int y = 0; y < 2; y++)
                                *(float2*)&sh.sums[z][kg][t * 16 + (lane >> 2) + y * 8][kh * 16 + n * 8 + (lane & 3) * 2] = make_float2(x[t][n][2 * y], x[t][n][2 * y + 1]);
                    advance();
                }
                const bool scale = lr_sync_or(grew);
                if (k < k1) {
                    float x[PER], mx = -INFINITY, sum = 0.0f;
                    const int key0 = from + k * LR_KEYS + part * PER;
#pragma unroll
                    for (int i = 0; i < PER; i++) {
                        const float d = (sh.sums[z][0][row][part * PER + i] + sh.sums[z][1][row][part * PER + i]) + (sh.sums[z][2][row][part * PER + i] + sh.sums[z][3][row][part * PER + i]);
                        x[i] = key0 + i <= pos && key0 + i >= key_lo ? d * f : -INFINITY;      // (a row sees no key behind `to`)
                        mx = fmaxf(mx, x[i]);
                    }
#pragma unroll
                    for (int d = 1; d < LANES; d *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
                    const float m_new = fmaxf(m, mx), base = m_new == -INFINITY ? 0.0f : m_new, alpha = m == m_new ? 1.0f : lt_exp2(m - m_new);
                    grew = alpha != 1.0f;
                    m = m_new;
#pragma unroll
                    for (int i = 0; i < PER; i++) { x[i] = lt_exp2(x[i] - base + LR_SHIFT); sum += x[i]; }
                    l = fmaf(l, alpha, sum);
#pragma unroll
                    for (int i = 0; i < PER; i += 2) *(unsigned*)&sh.p[z][row][part * PER + i] = lt_pack(x[i], x[i + 1]);
                    if (part == 0) sh.alpha[z][row] = alpha;
                }
                if (k > k0) {                                             // the values of the step before
                    const unsigned at = ring + v_slot * slot_bytes + v_lane, ps = pg_smem(&sh.p[z ^ 1][0][0]) + p_lane;
                    if (scale) {
#pragma unroll
                        for (int t = 0; t < MT; t++) {
                            const float a0 = sh.alpha[z ^ 1][t * 16 + (lane >> 2)], a1 = sh.alpha[z ^ 1][t * 16 + (lane >> 2) + 8];
#pragma unroll
                            for (int i = 0; i < LR_VB; i++)
#pragma unroll
                                for (int n = 0; n < 2; n++) { o[t][i][n][0] *= a0; o[t][i][n][1] *= a0; o[t][i][n][2] *= a1; o[t][i][n][3] *= a1; }
                        }
                    }
#pragma unroll
                    for (int kk = 0; kk < LR_KEYS / 16; kk++) {
                        unsigned p[MT][4];
#pragma unroll
                        for (int t = 0; t < MT; t++) lt_ldsm(p[t], ps + t * 16 * 80 + kk * 32);
#pragma unroll
                        for (int i = 0; i < LR_VB; i++) {
                            const int b = warp + LR_WARPS * i;
                            if (b < v_blocks) {
                                unsigned v[4];
                                lt_ldsm_t(v, at + kk * 16 * pitch + b * 32);
#pragma unroll
                                for (int t = 0; t < MT; t++) { lt_mma(o[t][i][0], p[t], v[0], v[1]); lt_mma(o[t][i][1], p[t], v[2], v[3]); }
                            }
                        }
                    }
                    sg_arrive(pg_smem(&sh.empty[v_slot]));
                }
                v_slot = here;
            }
            // a cut segment leaves its sums, the others their result
#pragma unroll
            for (int d = 1; d < LANES; d *= 2) l += __shfl_xor_sync(0xffffffffu, l, d);
            const int place = 2 * c + (first ? 0 : 1);
            const bool any = k1 > k0 || !cut;
            if (part == 0) {
                float by = 1.0f;
                if (!cut) {
                    float total = l, g = 1.0f;
                    if (a.sink && row < n_rows) {
                        const float sk = a.sink[(row0 + row) % a.H] * LR_LOG2E, m2 = fmaxf(m, sk);
                        g = m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : exp2f(m - m2);
                        total = g * l + (sk == -INFINITY ? 0.0f : exp2f(sk - m2 + LR_SHIFT));
                    }
                    by = g / total;
                }
                if (cut && any) a.ml[(size_t)place * ROWS + row] = make_float2(m, l);
                sh.inv[row] = by;
                sh.top[row] = m;
                sh.sum[row] = l;
            }
            lr_sync();
            float* lat = cut ? a.part + (size_t)place * ROWS * a.rank : a.lat + ((int64_t)s.first * a.H + row0) * a.rank;
            unsigned wild = 0;
#pragma unroll
            for (int t = 0; t < MT; t++)
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const int r = t * 16 + (lane >> 2) + y * 8;
                    const float by = sh.inv[r];
#pragma unroll
                    for (int i = 0; i < LR_VB; i++) {
                        const int b = warp + LR_WARPS * i;
                        if (b < v_blocks && r < n_rows && any)
#pragma unroll
                            for (int n = 0; n < 2; n++) {
                                const float u = o[t][i][n][2 * y], v = o[t][i][n][2 * y + 1];
                                if (!(fabsf(u) < INFINITY && fabsf(v) < INFINITY) && fabsf(sh.sum[r]) < INFINITY) wild |= 1u << r;
                                *(float2*)(lat + (int64_t)r * a.rank + b * 16 + n * 8 + (lane & 3) * 2) = make_float2(u * by, v * by);
                            }
                    }
                }
            if (wild) atomicOr(&sh.wild, wild);
            if (lr_sync_or(wild != 0)) lr_again<MT>(a, sh, s, seq, row0, from + k0 * LR_KEYS, min(to, from + k1 * LR_KEYS), lat, a.rank);
        });
    }
    __syncthreads();
    if (tid == 0 && sh.fail) {
        if (err_dev) atomicExch(err_dev, 5u);
        if (err_host) { *(volatile unsigned*)err_host = 5u; __threadfence_system(); }
    }
}
// segments in several runs: grid (segments, rows, 128 columns); a warp takes every eighth slice.  (One thread a column, one slice after another: 43 us for the 148 slices of a long cache)
#define LJ_WARPS 8
template <int MT>
__global__ void __launch_bounds__(LJ_WARPS * 32) latent_join_kernel(const LrArgs a, const __grid_constant__ LrCuts cuts) {
    __shared__ float factor[LR_CTAS], red[2][LJ_WARPS];
    __shared__ float4 sums[LJ_WARPS][32];
    pdl_enter();
    constexpr int ROWS = 16 * MT;
    const auto cut = cuts.at[blockIdx.x];
    const PgSeq s = a.seqs[cut.seq];
    const int y = blockIdx.y, row = cut.tile * ROWS + y, lane = threadIdx.x & 31, w = threadIdx.x >> 5, c = blockIdx.z * 128 + lane * 4;
    if (row >= s.count * a.H) return;
    auto place = [&](int x) { return (size_t)(x == 0 ? cut.slot : 2 * (cut.cta + x - 1)) * ROWS + y; };
    static_assert(LR_CTAS <= LJ_WARPS * 32, "a thread a slice");
    const int x = threadIdx.x;
    const float2 z = x < cut.n ? a.ml[place(x)] : make_float2(-INFINITY, 0.0f);
    float m = warp_max(z.x);
    if (lane == 0) red[0][w] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LJ_WARPS; i++) m = fmaxf(m, red[0][i]);
    const float f = z.x == -INFINITY ? (z.y == 0.0f ? 0.0f : 1.0f) : exp2f(z.x - m);
    if (x < cut.n) factor[x] = f;
    float l = warp_sum(f * z.y);
    if (lane == 0) red[1][w] = l;
    __syncthreads();
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (c < a.rank) {
#pragma unroll 4
        for (int i = w; i < cut.n; i += LJ_WARPS) {
            const float by = factor[i];
            const float4 v = *(const float4*)(a.part + place(i) * a.rank + c);
            if (by != 0.0f) { o.x = fmaf(by, v.x, o.x); o.y = fmaf(by, v.y, o.y); o.z = fmaf(by, v.z, o.z); o.w = fmaf(by, v.w, o.w); }
        }
    }
    sums[w][lane] = o;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < LJ_WARPS; i++) l += red[1][i];
    __syncthreads();
    float g = 1.0f;
    if (a.sink) {
        const float sk = a.sink[row % a.H] * LR_LOG2E, m2 = fmaxf(m, sk);
        g = m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : exp2f(m - m2);
        l = g * l + (sk == -INFINITY ? 0.0f : exp2f(sk - m2 + LR_SHIFT));
    }
    const int col = blockIdx.z * 128 + threadIdx.x;
    if (threadIdx.x < 128 && col < a.rank) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < LJ_WARPS; i++) t += ((const float*)sums[i])[threadIdx.x];
        a.lat[((int64_t)s.first * a.H + row) * a.rank + col] = t * (g / l);
    }
}

// the runs of deal.ctas CTAs over all steps, and the segments that are in several of them (returned: how many)
static int lr_deal(const cc_page_plan* plan, const LrArgs& a, int rows, int64_t steps, LrDeal& deal, LrCuts& cuts) {
    deal.run_lo = (int)(steps / deal.ctas); deal.run_more = (int)(steps % deal.ctas);
    int64_t before = 0, next = 0;                                  // steps in front of the sequence, and of run c
    int c = 0, n_cuts = 0;
    for (int seq = 0; seq < (int)plan->seqs.size() && c < deal.ctas; seq++) {
        const int n = lr_tiles(plan->seqs[seq], a, rows), all = n ? lr_steps(plan->seqs[seq], a) : 0;
        for (; c < deal.ctas && next < before + (int64_t)n * all; next += deal.run_lo + (c < deal.run_more ? 1 : 0), c++) {
            const int tile = (int)((next - before) / all), off = (int)((next - before) - (int64_t)tile * all);
            deal.at[c] = {seq, tile, off};
            if (off <= LR_BEGIN) continue;                         // the segment's keys are all this run's, or there are none of them in front
            auto& cut = cuts.at[n_cuts ? n_cuts - 1 : 0];
            if (n_cuts && cut.seq == seq && cut.tile == tile) { cut.n++; continue; }
            const auto& last = deal.at[c - 1];                     // the run in front begins with the segment, or within its first steps, or ends with it
            cuts.at[n_cuts++] = {seq, tile, 2 * (c - 1) + (last.seq == seq && last.tile == tile ? 0 : 1), c, 2};
        }
        before += (int64_t)n * all;
    }
    return n_cuts;
}
template <int MT>
static int lr_run(cc_device* dev, const cc_page_plan* plan, LrArgs a, const LtRuns& runs) {
    constexpr int ROWS = 16 * MT;
    int64_t steps = 0, tiles = 0;
    for (const PgSeq& s : plan->seqs) {
        const int n = lr_tiles(s, a, ROWS);
        tiles += n;
        steps += (int64_t)n * (n ? lr_steps(s, a) : 0);
    }
    if (!tiles) return CC_OK;
    LrDeal deal;
    LrCuts cuts;
    CC_REQUIRE(dev, steps < ((int64_t)1 << 31) * 64, "paged_latent_attention: too many rows");
    deal.ctas = (int)std::min<int64_t>(std::min(LR_CTAS, dev->sm_count), (steps + LR_BEGIN + 1) / (LR_BEGIN + 2));
    const int n_cuts = lr_deal(plan, a, ROWS, steps, deal, cuts);
    const size_t qf = (size_t)plan->tokens * a.H * a.cols * 4, lat = (size_t)plan->tokens * a.H * a.rank * 4, part = n_cuts ? (size_t)2 * deal.ctas * ROWS * a.rank * 4 : 0;
    void* ws = nullptr; size_t cls = 0;
    const int rc = cc_pool_alloc(dev, qf + lat + part + (size_t)2 * deal.ctas * ROWS * sizeof(float2), &ws, &cls);
    if (rc) return rc;
    a.qf = (float*)ws; a.lat = (float*)((uint8_t*)ws + qf); a.part = (float*)((uint8_t*)ws + qf + lat); a.ml = (float2*)((uint8_t*)ws + qf + lat + part);
    const int slot = LR_KEYS * (a.cols * 2 + 16);
    a.slots = std::min(LR_SLOTS, (LR_SMEM - (int)sizeof(LrShared<MT>)) / slot);
    const unsigned z = (unsigned)std::min(runs.tiles, 64);
    const size_t fold = (size_t)a.dim * (LF_COLS + 8) * 2 + 16 * (a.dim + 8) * 2, unfold = (size_t)(LU_COLS + 32) * (a.rank + 8) * 2;
    cudaError_t e = cudaFuncSetAttribute(latent_fold_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, LT_DIM * (LF_COLS + 8) * 2 + 16 * (LT_DIM + 8) * 2);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(latent_rows_kernel<MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, LR_SMEM - (int)sizeof(LrShared<MT>));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(latent_unfold_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (LU_COLS + 32) * (LT_RANK + 8) * 2);
    if (e == cudaSuccess) e = cc_launch_pdl(dev, latent_fold_kernel, dim3((unsigned)a.H, (unsigned)((a.rank + LF_COLS - 1) / LF_COLS + (a.rest ? 1 : 0)), z), 128, fold, a, runs);
    if (e == cudaSuccess) e = cc_launch_pdl(dev, latent_rows_kernel<MT>, (unsigned)deal.ctas, LR_THREADS, (size_t)a.slots * slot, a, deal, dev->err_dev, dev->err_host);
    if (e == cudaSuccess && n_cuts) { e = cc_launch_pdl(dev, latent_join_kernel<MT>, dim3((unsigned)n_cuts, ROWS, (unsigned)(a.rank + 127) / 128), LJ_WARPS * 32, 0, a, cuts); dev->launches++; }
    if (e == cudaSuccess) e = cc_launch_pdl(dev, latent_unfold_kernel, dim3((unsigned)a.H, (unsigned)((a.vdim + LU_COLS - 1) / LU_COLS), z), 128, unfold, a, runs);
    dev->launches += 3;
    cc_pool_free(dev, ws, cls);
    if (e != cudaSuccess) return cc_fail(dev, CC_ERR_CUDA, "paged_latent_attention: %s", cudaGetErrorString(e));
    return CC_OK;
}

#include "latent_tile.cuh"

#define LT_FEW 64                             // new tokens of a sequence; with more its keys and values are laid out

extern "C" CC_API int cc_paged_latent_attention(cc_device* dev, const cc_page_plan* plan, const cc_view* pages, int32_t rank, const cc_view* q, int32_t H, const cc_view* uk,
                                                const cc_view* uv, float scale, int32_t window, const cc_view* sink, int32_t form, int32_t out_type, cc_buf** out) {
    PG_ENTER(dev, plan, "paged_latent_attention");
    if (!out) return cc_fail(dev, CC_ERR_ARG, "paged_latent_attention: out is NULL");
    *out = nullptr;
    LtPages c;
    int rc = lt_check_pages(dev, plan, pages, rank, "paged_latent_attention", &c);
    if (rc) return rc;
    HT_WHOLE(dev, q, CC_F16, "paged_latent_attention q"); HT_WHOLE(dev, uk, CC_F16, "paged_latent_attention uk"); HT_WHOLE(dev, uv, CC_F16, "paged_latent_attention uv");
    const int64_t T = plan->tokens;
    CC_REQUIRE(dev, H > 0 && H <= 8192, "paged_latent_attention: %d heads", H);
    CC_REQUIRE(dev, uk->ndim == 2 && uv->ndim == 2 && uk->shape[1] == rank && uv->shape[1] == rank && uk->shape[0] % H == 0 && uv->shape[0] % H == 0,
               "paged_latent_attention: uk and uv are not [%d heads of rows, %d]", H, rank);
    const int64_t dim = uk->shape[0] / H, vdim = uv->shape[0] / H;
    CC_REQUIRE(dev, dim >= 16 && dim <= LT_DIM && dim % 16 == 0 && vdim >= 16 && vdim <= LT_DIM && vdim % 16 == 0, "paged_latent_attention: heads of %lld and %lld (multiples of 16 up to %d)",
               (long long)dim, (long long)vdim, LT_DIM);
    CC_REQUIRE(dev, q->ndim == 2 && q->shape[0] == T && q->shape[1] == H * (dim + c.rest), "paged_latent_attention: q is not [%lld, %d * %lld]", (long long)T, H, (long long)(dim + c.rest));
    CC_REQUIRE(dev, T * H < ((int64_t)1 << 31), "paged_latent_attention: %lld tokens of %d heads", (long long)T, H);
    if (sink) {
        HT_WHOLE(dev, sink, CC_F32, "paged_latent_attention sink");
        CC_REQUIRE(dev, view_len(sink) == H, "paged_latent_attention: sink is not [%d]", H);
    }
    for (const cc_view* v : {q, uk, uv}) CC_REQUIRE(dev, ((uintptr_t)v->buf->plane[0] & 15) == 0, "paged_latent_attention: a tensor does not start at a multiple of 16 bytes");
    CC_REQUIRE(dev, form == CC_LATENT_AUTO || form == CC_LATENT_ABSORBED || form == CC_LATENT_EXPANDED, "paged_latent_attention: form %d", form);
    CC_REQUIRE(dev, out_type == CC_F16 || out_type == CC_BF16, "paged_latent_attention: results of type %d (F16 or BF16)", out_type);
    // tensor maps count rows in 32 bits
    const bool expands = dim <= TL_DIM && vdim <= TL_DIM && plan->n_pages * plan->page < ((int64_t)1 << 31) && (int64_t)H * LT_DIM < ((int64_t)1 << 31);
    CC_REQUIRE(dev, form != CC_LATENT_EXPANDED || expands, "paged_latent_attention: heads of %lld and %lld are not expanded (up to %d)", (long long)dim, (long long)vdim, TL_DIM);
    cc_buf* o = nullptr;
    rc = cc_new_activation(dev, T * H * vdim, out_type, false, &o);
    if (rc) return rc;
    if (T > 0) {
        LrArgs a{};
        a.seqs = plan->d_seqs; a.table = plan->d_table; a.rows = c.rows;
        a.q = (const __half*)q->buf->plane[0]; a.uk = (const __half*)uk->buf->plane[0]; a.uv = (const __half*)uv->buf->plane[0];
        a.sink = sink ? (const float*)sink->buf->plane[0] : nullptr; a.out = o->base; a.scale = scale;
        a.n_seqs = plan->n_seqs; a.table_cols = plan->table_cols; a.page = plan->page; a.shift = plan->shift; a.H = H; a.dim = (int)dim; a.vdim = (int)vdim;
        a.rank = c.rank; a.rest = c.rest; a.cols = c.cols; a.window = window > 0 ? window : 0; a.out_bf16 = out_type == CC_BF16;
        a.most = form == CC_LATENT_EXPANDED ? 0 : form == CC_LATENT_ABSORBED || !expands ? 0x7fffffff : LT_FEW;
        LtRuns runs{};
        bool wide = false;
        for (const PgSeq& s : plan->seqs) {
            if (s.count == 0 || s.count > a.most) continue;
            wide = wide || (int64_t)s.count * H > 16;
            if (runs.n && runs.hi[runs.n - 1] == s.first) { runs.hi[runs.n - 1] = s.first + s.count; continue; }
            if (runs.n == LT_RUNS) { runs.hi[runs.n - 1] = s.first + s.count; continue; }      // many runs: the last one takes all that lies behind (other tokens' results are overwritten)
            runs.lo[runs.n] = s.first; runs.hi[runs.n++] = s.first + s.count;
        }
        for (int i = 0; i < runs.n; i++) { runs.tile0[i] = runs.tiles; runs.tiles += (runs.hi[i] - runs.lo[i] + 15) / 16; }
        rc = wide ? lr_run<2>(dev, plan, a, runs) : lr_run<1>(dev, plan, a, runs);
        if (!rc && a.most < 0x7fffffff) rc = tl_run(dev, plan, a);      // behind the others: their last products may run over tokens of these
    }
    if (rc) { cc_tensor_release(o); return rc; }
    *out = o;
    return CC_OK;
}
