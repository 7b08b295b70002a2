// latent_attn.cu -- attention over pages of latent rows (include/crabml_paged.h), absorbed: the queries are carried over to the latents (latent_fold_kernel), the cached rows themselves
// are keys and values of all heads (latent_rows_kernel), and what comes out is carried back (latent_unfold_kernel).
//
// A row of the scores is a query of one head: 16 heads of one token are 16 rows over the same keys, one tile of mma.sync.m16n8k16.  One token of 16 heads over rows of 512 + 64
// makes 30 operations a byte of the cache, so bytes bound it, as long as every row comes from memory once: a CTA (one per SM) brings 32 rows at a time into a ring of shared memory
// by copies of 64 columns, and 8 warps take them twice, as keys and as values:
//   scores   warp w adds up the columns 16 (w % 4 + 4 i) of 16 keys (w / 4); the queries stay in registers, sums of the four column groups meet in shared memory
//   weights  a thread two keys of a row: exp2(score - largest), rounded to f16, back to shared memory
//   values   warp w adds up the columns 16 (w + 8 i) of all rows in registers; scaled when a row's largest score grows
// That is a chain of 2700 cycles a step, mostly latencies, while the step's bytes take 1600; so two such groups of 8 warps take the steps by turns and add up their sums at a segment's end.
// All steps of a call are dealt out in equal runs over the SMs; sums of cut segments are joined by latent_join_kernel.
// 64 sequences of 20 to 4000 rows, 16 heads of 128 + 64 over 512 + 64: 56 us, of which this kernel 41 (154 MB: 3.7 TB/s with starts, restarts at segments and sums); one token over 32000 rows 29, this
// kernel 17 (37 MB), of which 11 start and end, fold 4, join 4, unfold 5.
//
// Sums, largest scores and sums of weights have 32 bits; queries on their way to the latents are brought near 2^4 by a power of two and rounded to f16, weights are rounded to f16 near
// 2^10 (2^-11 of each: the operands of the tensor cores; the result is rounded to 16 bits anyway), sums of latents enter the last product as two f16 numbers, the number and 2^11 times its rest.
#include <cuda.h>

#include <algorithm>

#include "latent.cuh"
#include "latent_ring.cuh"
#include "split_gemm.cuh"

#define LR_THREADS (LR_GROUPS * 256)
#define LR_BLOCK 4096                         // 32 rows of 64 columns
#define LR_ROWS 16                            // queries of a tile
#define LR_KEYS 32                            // of a step
#define LR_BEGIN 6                            // what a segment's begin and end cost, in steps (64 sequences of 20 to 4000 tokens: counted as 4 59 us, 6 56.5, 9 57)
#define LR_SMEM (226 * 1024)                  // with what stands in LrShared
#define LR_SHIFT 10.0f                        // weights are exp2(score - largest + LR_SHIFT)
#define LR_KB 9                               // column blocks of 16 of a warp's scores: (LT_RANK + LT_REST) / 16 / 4
#define LR_VB 4                               // .. of its values: LT_RANK / 16 / 8
#define LR_RUNS 5                             // runs of 128 columns of a row
#define LR_CTAS 160
#define LJ_FEW 8                              // slices of a segment that are added up over all columns at a time
#define LR_LOG2E 1.4426950408889634f

// runs of consecutive tokens whose sequences take this form
#define LT_RUNS 64
#define LT_TOKENS 32                          // of a tile of the products in front and behind
struct LtRuns { int n, tiles; int lo[LT_RUNS], hi[LT_RUNS], tile0[LT_RUNS]; };
struct LrArgs {
    const PgSeq* seqs;
    const int* table;
    const __half *rows, *q, *uk, *uv;
    const float* sink;
    float *qf, *lat, *part;                   // queries over the latents [T H][cols]; results over the latents [T H][rank]; sums of cut segments [2 x CTA][LR_ROWS][rank]
    float2* ml;                               // [2 x CTA][LR_ROWS]: largest score (base 2), sum of weights
    int4* steps;                              // [CTA][run_lo + 1]: what each step asks for
    void* out;
    float scale;
    int n_seqs, table_cols, page, shift, H, dim, vdim, rank, rest, cols, window, out_bf16, slots;
    int most, token0, token1;                 // sequences with more new tokens take the other form; the tokens of this portion
};
struct LrDeal { int ctas, run_lo, run_more; struct { int seq, tile, off; } at[LR_CTAS]; };
struct LrCuts { struct { int seq, tile, slot, cta, n; } at[LR_CTAS]; };

// a sequence's part in this portion of the call's tokens: none of those that take the other form
__host__ __device__ __forceinline__ PgSeq lr_clip(PgSeq s, const LrArgs& a) {
    const int lo = s.first > a.token0 ? s.first : a.token0, hi = s.first + s.count < a.token1 ? s.first + s.count : a.token1;
    if (s.count > a.most || hi <= lo) { s.count = 0; return s; }
    s.pos0 += lo - s.first; s.first = lo; s.count = hi - lo;
    return s;
}
__host__ __device__ __forceinline__ void lr_range(const PgSeq& s, const LrArgs& a, int* from, int* to) {
    *to = s.pos0 + s.count;
    *from = a.window > 0 && s.pos0 - a.window + 1 > 0 ? (s.pos0 - a.window + 1) & ~(LR_KEYS - 1) : 0;      // steps are whole pages, or parts of one
}
__host__ __device__ __forceinline__ int lr_tiles(const PgSeq& s, const LrArgs& a) { return (int)(((int64_t)s.count * a.H + LR_ROWS - 1) / LR_ROWS); }
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
// x, y as f16 (h) and LT_UP times what is left of them as f16 (l), at most |x|, so that small numbers, which f16 holds in steps of 2^-24, keep their bits; an infinity's or NaN's rest is NaN
#define LT_UP 2048.0f
__device__ __forceinline__ void lt_cut(float x, float y, unsigned& h, unsigned& l) {
    const __half2 a = __floats2half2_rn(x, y);
    const float2 b = __half22float2(a);
    h = *(const unsigned*)&a;
    l = lt_pack((x - b.x) * LT_UP, (y - b.y) * LT_UP);
}
__device__ __forceinline__ void lt_copy16(unsigned dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void lt_copies_done() { asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ bool lt_tile(const LtRuns& runs, int tile, int* lo, int* hi) {
    for (int i = 0; i < runs.n; i++) {
        const int t = tile - runs.tile0[i];
        if (t >= 0 && runs.lo[i] + t * LT_TOKENS < runs.hi[i]) { *lo = runs.lo[i] + t * LT_TOKENS; *hi = min(*lo + LT_TOKENS, runs.hi[i]); return true; }
    }
    return false;
}

// a CTA's run of steps, segment by segment; the begin of a segment counts LR_BEGIN of them
struct LrWalk {
    int seq, tile, off, left;
    // the next piece: false at the end.  first and last step of its keys; whether others have the rest of the segment
    template <class F>
    __device__ __forceinline__ bool piece(const LrArgs& a, F body) {
        while (left > 0 && seq < a.n_seqs) {
            const PgSeq s = lr_clip(a.seqs[seq], a);
            if (tile >= lr_tiles(s, a)) { seq++; tile = 0; off = 0; continue; }
            const int all = lr_steps(s, a), take = min(left, all - off), from = off;
            left -= take;
            body(s, seq, tile, max(from - LR_BEGIN, 0), max(from + take - LR_BEGIN, 0), from > LR_BEGIN || from + take < all);
            if (from + take == all) { tile++; off = 0; } else off += take;
            return true;
        }
        return false;
    }
};
// what a step asks for: two pages, the row in them where it begins, how many of them (0: nothing)
__device__ __forceinline__ int4 lr_pages(const LrArgs& a, int seq, int key0, int to) {
    const int rows = min(a.page, LR_KEYS), there = (min(LR_KEYS, to - key0) + rows - 1) / rows;
    const int* t = a.table + (int64_t)seq * a.table_cols + (key0 >> a.shift);
    return make_int4(t[0], there > 1 ? t[1] : 0, key0 & (a.page - 1), there);
}

// ---- queries to the latents, results back ---------------------------------------------------------------------------------------------------
// qf[t, h, :rank] = U_h^T n[t, h], qf[t, h, rank:] = p[t, h], in 32 bits.  grid (heads, blocks of 64 columns and one for p, tiles of LT_TOKENS tokens by turns); a warp 16 columns.
// The blocks behind write down what the steps of each CTA of latent_rows_kernel ask for, a warp a CTA
#define LF_COLS 64
__global__ void __launch_bounds__(128) latent_fold_kernel(const __grid_constant__ LrArgs a, const __grid_constant__ LtRuns runs, const __grid_constant__ LrDeal deal) {
    extern __shared__ __align__(16) uint8_t lf_raw[];
    __half *bs = (__half*)lf_raw, *as = bs + a.dim * (LF_COLS + 8);      // U_h's rows, 64 columns of them; queries [LT_TOKENS][dim + 8]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, h = blockIdx.x, c0 = blockIdx.y * LF_COLS, width = a.dim + a.rest;
    pdl_enter();
    const int fold_blocks = (a.rank + LF_COLS - 1) / LF_COLS;
    if ((int)blockIdx.y > fold_blocks) {
        const int c = (((int)blockIdx.y - fold_blocks - 1) * a.H + h) * 4 + warp, room = deal.run_lo + 1;
        if (c >= deal.ctas || blockIdx.z) return;
        LrWalk walk = {deal.at[c].seq, deal.at[c].tile, deal.at[c].off, deal.run_lo + (c < deal.run_more ? 1 : 0)};
        int4* to_list = a.steps + (int64_t)c * room;
        int n = 0;
        while (walk.piece(a, [&](const PgSeq& s, int seq, int, int k0, int k1, bool) {
            int from, to;
            lr_range(s, a, &from, &to);
            for (int k = k0 + lane; k < k1; k += 32) to_list[n + k - k0] = lr_pages(a, seq, from + k * LR_KEYS, to);
            n += k1 - k0;
        })) {}
        for (int i = n + lane; i < room; i += 32) to_list[i] = make_int4(0, 0, 0, 0);
        return;
    }
    if ((int)blockIdx.y == fold_blocks) {                                // p
        for (int tile = blockIdx.z; tile < runs.tiles; tile += gridDim.z) {
            int lo, hi;
            if (!lt_tile(runs, tile, &lo, &hi)) return;
#pragma unroll 2
            for (int e = tid; e < (hi - lo) * (a.rest / 8); e += 128) {
                const int64_t row = (int64_t)(lo + e / (a.rest / 8)) * a.H + h;
                const int c = e % (a.rest / 8) * 8;
                const uint4 v = __ldg((const uint4*)(a.q + row * width + a.dim + c));
                const float2 x = __half22float2(*(const __half2*)&v.x), y = __half22float2(*(const __half2*)&v.y), z = __half22float2(*(const __half2*)&v.z), w = __half22float2(*(const __half2*)&v.w);
                float4* at = (float4*)(a.qf + row * a.cols + a.rank + c);
                at[0] = make_float4(x.x, x.y, y.x, y.y); at[1] = make_float4(z.x, z.y, w.x, w.y);
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
        const int mt = (hi - lo + 15) >> 4, runs8 = a.dim / 8;
        __syncthreads();
        for (int e = tid; e < mt * 16 * runs8; e += 128) {
            const int r = e / runs8, c = e % runs8 * 8;
            if (lo + r < hi) lt_copy16(pg_smem(as + r * (a.dim + 8) + c), a.q + ((int64_t)(lo + r) * a.H + h) * width + c);
            else *(uint4*)(as + r * (a.dim + 8) + c) = make_uint4(0, 0, 0, 0);
        }
        lt_copies_done();
        __syncthreads();
        if (c0 + warp * 16 >= a.rank) continue;
        float acc[LT_TOKENS / 16][2][4];
#pragma unroll
        for (int i = 0; i < LT_TOKENS / 16 * 8; i++) acc[i >> 3][i >> 2 & 1][i & 3] = 0.0f;
#pragma unroll 2
        for (int k = 0; k < a.dim; k += 16) {
            unsigned x[4], b[4];
            lt_ldsm_t(b, pg_smem(bs + (k + (lane & 7) + (lane >> 3 & 1) * 8) * (LF_COLS + 8) + warp * 16 + (lane >> 4) * 8));
#pragma unroll
            for (int m = 0; m < LT_TOKENS / 16; m++)
                if (m < mt) {
                    lt_ldsm(x, pg_smem(as + (m * 16 + (lane & 7) + (lane >> 3 & 1) * 8) * (a.dim + 8) + k + (lane >> 4) * 8));
                    lt_mma(acc[m][0], x, b[0], b[1]);
                    lt_mma(acc[m][1], x, b[2], b[3]);
                }
        }
#pragma unroll
        for (int m = 0; m < LT_TOKENS / 16; m++)
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const int t = lo + m * 16 + (lane >> 2) + y * 8;
                    if (t < hi) *(float2*)(a.qf + ((int64_t)t * a.H + h) * a.cols + c0 + warp * 16 + i * 8 + (lane & 3) * 2) = make_float2(acc[m][i][2 * y], acc[m][i][2 * y + 1]);
                }
    }
}
// out[t, h] = V_h lat[t, h].  grid (heads, blocks of 32 columns, tiles of LT_TOKENS tokens by turns); a warp 8 columns and half of the depth
#define LU_COLS 32
#define LU_THREADS 256
__host__ __device__ constexpr int lu_smem(int rank) { return (LU_COLS + 2 * LT_TOKENS) * (rank + 8) * 2; }
__global__ void __launch_bounds__(LU_THREADS) latent_unfold_kernel(const __grid_constant__ LrArgs a, const __grid_constant__ LtRuns runs) {
    extern __shared__ __align__(16) uint8_t lf_raw[];
    __shared__ float sums[LT_TOKENS][LU_COLS + 1];
    const int pitch = a.rank + 8;
    __half *bs = (__half*)lf_raw, *as = bs + LU_COLS * pitch;          // V_h's rows; sums of latents [h, l][LT_TOKENS][pitch]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, h = blockIdx.x, c0 = blockIdx.y * LU_COLS, cg = warp & 3, part = warp >> 2;
    pdl_enter();
    for (int e = tid; e < LU_COLS * (a.rank / 8); e += LU_THREADS) {
        const int r = e / (a.rank / 8), c = e % (a.rank / 8) * 8;
        if (c0 + r < a.vdim) lt_copy16(pg_smem(bs + r * pitch + c), a.uv + ((int64_t)h * a.vdim + c0 + r) * a.rank + c);
        else *(uint4*)(bs + r * pitch + c) = make_uint4(0, 0, 0, 0);
    }
    for (int tile = blockIdx.z; tile < runs.tiles; tile += gridDim.z) {
        int lo, hi;
        if (!lt_tile(runs, tile, &lo, &hi)) break;
        const int mt = (hi - lo + 15) >> 4, runs4 = a.rank / 4;
        __syncthreads();
#pragma unroll 4
        for (int e = tid; e < mt * 16 * runs4; e += LU_THREADS) {
            const int r = e / runs4, c = e % runs4 * 4;
            const float4 v = lo + r < hi ? *(const float4*)(a.lat + ((int64_t)(lo + r) * a.H + h) * a.rank + c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            uint2 x, y;
            lt_cut(v.x, v.y, x.x, y.x); lt_cut(v.z, v.w, x.y, y.y);
            *(uint2*)(as + r * pitch + c) = x;
            *(uint2*)(as + (LT_TOKENS + r) * pitch + c) = y;
        }
        lt_copies_done();
        __syncthreads();
        float acc[LT_TOKENS / 16][2][4];
#pragma unroll
        for (int i = 0; i < LT_TOKENS / 16 * 8; i++) acc[i >> 3][i >> 2 & 1][i & 3] = 0.0f;
        const int r = (lane & 7) + (lane >> 3 & 1) * 8, kc = (lane >> 4) * 8, half = a.rank / 32 * 16;
#pragma unroll 4
        for (int k = part ? half : 0; k < (part ? a.rank : half); k += 16) {
            unsigned b0, b1;
            asm volatile("ldmatrix.sync.aligned.m8n8.x2.shared.b16 {%0, %1}, [%2];" : "=r"(b0), "=r"(b1) : "r"(pg_smem(bs + (cg * 8 + (lane & 7)) * pitch + k + (lane >> 3 & 1) * 8)));
#pragma unroll
            for (int m = 0; m < LT_TOKENS / 16; m++)
                if (m < mt) {
                    unsigned x[4], y[4];
                    lt_ldsm(x, pg_smem(as + (m * 16 + r) * pitch + k + kc));
                    lt_ldsm(y, pg_smem(as + (LT_TOKENS + m * 16 + r) * pitch + k + kc));
                    lt_mma(acc[m][0], x, b0, b1);
                    lt_mma(acc[m][1], y, b0, b1);
                }
        }
        const int c = cg * 8 + (lane & 3) * 2;
#pragma unroll
        for (int m = 0; m < LT_TOKENS / 16; m++)
#pragma unroll
            for (int y = 0; y < 2; y++) {
                const int t = m * 16 + (lane >> 2) + y * 8;
                if (part == 1) { sums[t][c] = fmaf(acc[m][1][2 * y], 1.0f / LT_UP, acc[m][0][2 * y]); sums[t][c + 1] = fmaf(acc[m][1][2 * y + 1], 1.0f / LT_UP, acc[m][0][2 * y + 1]); }
            }
        __syncthreads();
        if (part == 0) {
#pragma unroll
            for (int m = 0; m < LT_TOKENS / 16; m++)
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const int t = m * 16 + (lane >> 2) + y * 8;
                    const float u = fmaf(acc[m][1][2 * y], 1.0f / LT_UP, acc[m][0][2 * y]) + sums[t][c], v = fmaf(acc[m][1][2 * y + 1], 1.0f / LT_UP, acc[m][0][2 * y + 1]) + sums[t][c + 1];
                    if (lo + t < hi && c0 + c < a.vdim) *(unsigned*)((uint16_t*)a.out + ((int64_t)(lo + t) * a.H + h) * a.vdim + c0 + c) = a.out_bf16 ? ht_pack_bf16(u, v) : ht_pack_f16(u, v);
                }
        }
    }
}

// ---- the cached rows as keys and values ----------------------------------------------------------------------------------------------------------
struct LrShared {
    unsigned long long full[LR_GROUPS * LR_SLOTS];
    int fail;
    unsigned wild;                            // rows whose sums are not finite
    float top[LR_GROUPS][LR_ROWS], sum[LR_GROUPS][LR_ROWS];      // of a segment: largest score and sum of weights of each group
    float factor[LR_ROWS];                    // of a row's scores
    float alpha[LR_GROUPS][LR_ROWS];
    __align__(16) float sums[LR_GROUPS][4][LR_ROWS][40];      // of a step: scores by column groups.  At a segment's end, sums on their way from group to group
    __align__(16) __half p[LR_GROUPS][LR_ROWS][40];
};
static_assert(sizeof(float) * LR_GROUPS * 4 * LR_ROWS * 40 >= LR_THREADS / LR_GROUPS * 16 * sizeof(float) && sizeof(float) * LR_GROUPS * 4 * LR_ROWS * 40 >= LR_ROWS * (LT_RANK + LT_REST + 8) * 2, "half of a group's sums, and the queries, pass here");
static_assert((LR_SMEM - (int)sizeof(LrShared) - 1024) / ((LT_RANK + LT_REST) / 64 * LR_BLOCK) >= LR_SLOTS_LEAST, "the widest rows leave too few slots");
__device__ __forceinline__ void lr_sync(int group) { asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "n"(LR_THREADS / LR_GROUPS) : "memory"); }
__device__ __forceinline__ bool lr_sync_or(int group, bool x) {
    unsigned r;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbar.red.or.pred q, %2, %3, p;\nselp.u32 %0, 1, 0, q;\n}\n" : "=r"(r) : "r"((unsigned)x), "r"(1 + group), "n"(LR_THREADS / LR_GROUPS) : "memory");
    return r;
}
__device__ __forceinline__ void lr_zero(unsigned at) { asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory"); }
// Values that are not finite, times the weight 0 of a row that does not see them, make a NaN.  Rows whose sums hold one though their scores do not are added up again, one by one, over
// the keys that they see: a dot product over the block, which then adds a column a thread.  The query is rounded as it was, so that a cut segment's other pieces go with this one; the largest score
// and the sum of weights are made again with the sums, whose scores are added up in another order
__device__ __noinline__ float lr_again(const LrArgs& a, LrShared& sh, const PgSeq s, int seq, int row0, int lo, int hi, int r, float& m, float& l) {
    const int tok = (row0 + r) / a.H, pos = s.pos0 + tok, c = threadIdx.x;
    const float* q = a.qf + ((int64_t)s.first * a.H + row0 + r) * a.cols;
    const float factor = sh.factor[r], up = 1.0f / factor;          // a power of two
    float o = 0.0f;
    m = -INFINITY; l = 0.0f;
    for (int key = max(lo, a.window > 0 ? pos - a.window + 1 : 0); key <= min(hi - 1, pos); key++) {
        const __half* row = a.rows + ((int64_t)a.table[(int64_t)seq * a.table_cols + (key >> a.shift)] * a.page + (key & (a.page - 1))) * a.cols;
        float d = 0.0f;
        for (int e = threadIdx.x; e < a.cols; e += LR_THREADS) d = fmaf(__half2float(__float2half_rn(q[e] * up)), __half2float(row[e]), d);
        d = warp_sum(d);
        if ((threadIdx.x & 31) == 0) sh.sums[0][0][0][threadIdx.x >> 5] = d;
        __syncthreads();
        d = 0.0f;
#pragma unroll
        for (int w = 0; w < LR_THREADS / 32; w++) d += sh.sums[0][0][0][w];
        __syncthreads();
        const float z = d * (factor * (a.scale * LR_LOG2E)), m_new = fmaxf(m, z), alpha = m == m_new ? 1.0f : lt_exp2(m - m_new), p = lt_exp2(z - (m_new == -INFINITY ? 0.0f : m_new) + LR_SHIFT);
        m = m_new;
        l = fmaf(l, alpha, p);
        if (c < a.rank) o = fmaf(p, __half2float(row[c]), o * alpha);
    }
    return o;
}
static_assert(LR_THREADS >= LT_RANK, "a thread a column");

__global__ void __launch_bounds__(LR_THREADS, 1) latent_rows_kernel(const __grid_constant__ CUtensorMap map_whole, const __grid_constant__ CUtensorMap map_rows, const __grid_constant__ LrArgs a, const __grid_constant__ LrDeal deal, unsigned* err_dev,
                                                                    unsigned* err_host) {
    extern __shared__ __align__(1024) uint8_t lr_raw[];
    __shared__ LrShared sh;
    const int tid = threadIdx.x, lane = tid & 31, group = tid / (LR_THREADS / LR_GROUPS), in_group = tid % (LR_THREADS / LR_GROUPS), warp = in_group >> 5;
    const unsigned ring = (pg_smem(lr_raw) + 1023) & ~1023u, n_blocks = (unsigned)((a.cols + 63) >> 6), slot_bytes = n_blocks * LR_BLOCK;
    if (tid == 0) {
        for (int i = 0; i < LR_GROUPS * a.slots; i++) pg_mbar_init(pg_smem(&sh.full[i]), 1);
        sh.fail = 0; sh.wild = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_whole) : "memory");
    }
    pdl_enter();
    __syncthreads();
    LrWalk walk = {deal.at[blockIdx.x].seq, deal.at[blockIdx.x].tile, deal.at[blockIdx.x].off, deal.run_lo + ((int)blockIdx.x < deal.run_more ? 1 : 0)};
    // a step's rows: one copy for all whole blocks of 64 columns of a page, and one for the columns behind them.  (A copy for each block, by all 8 warps, took the group 1000 cycles of a step; row by row,
    // a lane a row, 2500)
    const int box_rows = min(a.page, LR_KEYS), whole = a.cols >> 6;
    auto ask = [&](int step, const int4& p) {
        const LrPlace place = lr_place(step, a.slots);
        const unsigned bar = pg_smem(&sh.full[place.bar]), at = ring + place.slot * slot_bytes;
        if (pg_elect()) {
            pg_mbar_expect_tx(bar, (unsigned)(p.w * box_rows) * (slot_bytes / LR_KEYS));
            for (int i = 0; i < p.w; i++) {
                const int page = i ? p.y : p.x;
                const unsigned to = at + i * box_rows * 128;
                // (a box's blocks lie one behind the other: those of a page of 16 rows go to half a block each, so they come one by one)
                if (box_rows == LR_KEYS && whole)
                    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                                 ::"r"(to), "l"(&map_whole), "r"(bar), "r"(0), "r"(p.z), "r"(0), "r"(page) : "memory");
                for (unsigned b = box_rows == LR_KEYS ? (unsigned)whole : 0u; b < n_blocks; b++)
                    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                                 ::"r"(to + b * LR_BLOCK), "l"(&map_rows), "r"(bar), "r"(b * 64), "r"(p.z), "r"(page) : "memory");
            }
        }
        __syncwarp();
    };
    const int room = deal.run_lo + 1;
    const int4* list = a.steps + (int64_t)blockIdx.x * room;
    auto what = [&](int i) { return i < room ? list[i] : make_int4(0, 0, 0, 0); };
    int coming = a.slots + group;                                     // group 0 asks for the steps slots, slots + 2, .., group 1 for those between
    int4 next = what(coming);
    if (tid < 32 * a.slots) {                                         // the first slots, a warp each
        const int4 p = what(tid >> 5);
        if (p.w) ask(tid >> 5, p);
    }
    const int kg = warp & 3, kh = warp >> 2, blocks = a.cols >> 4, v_blocks = a.rank >> 4;
    const int row = in_group >> 4, part = in_group & 15;              // of the weights: 16 threads a row, two keys each
    // a slot: blocks of 64 columns, 32 rows of 128 bytes under the 128-byte swizzle.  This lane's row of four 8 x 8 blocks: scores take columns 16 (kg + 4 i), block i; values 16 (warp + 8 i), block warp / 4 + 2 i
    const unsigned k_lane = (unsigned)(kh * 16 + (lane >> 4) * 8 + (lane & 7)) * 128 + (((kg * 2 + (lane >> 3 & 1)) ^ (lane & 7)) << 4);
    const unsigned v_lane = (unsigned)(warp >> 2) * LR_BLOCK + (unsigned)((lane >> 3 & 1) * 8 + (lane & 7)) * 128 + ((((warp & 3) * 2 + (lane >> 4)) ^ (lane & 7)) << 4);
    const unsigned p_at = pg_smem(&sh.p[group][0][0]) + (unsigned)((lane >> 3 & 1) * 8 + (lane & 7)) * 80 + (lane >> 4) * 16;
    int n = 0, last = -1;                                             // steps of the run so far; this group's last one whose slot is free and not asked for
    bool ok = true, first = true;
    auto again = [&]() {                                              // (all warps of the group are through with step `last`)
        if (last < 0) return;
        if (warp == 0) {
            if (next.w && ok) ask(last + a.slots, next);
            coming += LR_GROUPS;
            next = what(coming);
        }
        last = -1;
    };
    while (walk.piece(a, [&](const PgSeq& s, int seq, int tile, int k0, int k1, bool cut) {
        int from, to;
        lr_range(s, a, &from, &to);
        const int row0 = tile * LR_ROWS, n_rows = min(LR_ROWS, s.count * a.H - row0);
        const float* qs = a.qf + ((int64_t)s.first * a.H + row0) * a.cols;
        // the rows near 2^4 by a power of two, as f16, by way of shared memory.  A warp a row
        if (tid == 0) sh.wild = 0;
        __half* staged = (__half*)&sh.sums[0][0][0][0];
        const int staged_pitch = a.cols + 8;                          // an odd number of 16 bytes: ldmatrix without conflicts
        {
            const int r = tid >> 5;
            unsigned top = 0;                                        // as bits, so that NaN is the largest of all
            uint4 v[LR_RUNS];
#pragma unroll
            for (int i = 0; i < LR_RUNS; i++) {
                const int e = (i * 32 + lane) * 4;
                v[i] = r < n_rows && e < a.cols ? *(const uint4*)(qs + (int64_t)r * a.cols + e) : make_uint4(0, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < LR_RUNS; i++) top = max(max(top, max(v[i].x & 0x7fffffffu, v[i].y & 0x7fffffffu)), max(v[i].z & 0x7fffffffu, v[i].w & 0x7fffffffu));
            top = __reduce_max_sync(0xffffffffu, top);
            const int ex = top < 0x00800000u || top >= 0x7f800000u ? 4 : max((int)(top >> 23) - 126, -100);
            const float up = __uint_as_float((unsigned)(4 - ex + 127) << 23);
            if (lane == 0) sh.factor[r] = top >= 0x7f800000u ? NAN : __uint_as_float((unsigned)(ex - 4 + 127) << 23);
#pragma unroll
            for (int i = 0; i < LR_RUNS; i++) {
                const int e = (i * 32 + lane) * 4;
                if (e < a.cols)
                    *(uint2*)(staged + r * staged_pitch + e) = make_uint2(lt_pack(__uint_as_float(v[i].x) * up, __uint_as_float(v[i].y) * up), lt_pack(__uint_as_float(v[i].z) * up, __uint_as_float(v[i].w) * up));
            }
        }
        __syncthreads();
        again();
        unsigned q[LR_KB][4];
#pragma unroll
        for (int i = 0; i < LR_KB; i++) {
            if (kg + 4 * i < blocks) lt_ldsm(q[i], pg_smem(staged + ((lane & 7) + (lane >> 3 & 1) * 8) * staged_pitch + (kg + 4 * i) * 16 + (lane >> 4) * 8));
            else q[i][0] = q[i][1] = q[i][2] = q[i][3] = 0u;
        }
        __syncthreads();                                              // the staged rows are read: sums go there
        const float f = sh.factor[row] * (a.scale * LR_LOG2E);
        const int pos = row < n_rows ? s.pos0 + (row0 + row) / a.H : -1, key_lo = a.window > 0 ? pos - a.window + 1 : 0;
        float m = -INFINITY, l = 0.0f;
        float o[LR_VB][2][4];
#pragma unroll
        for (int i = 0; i < LR_VB; i++)
#pragma unroll
            for (int x = 0; x < 8; x++) o[i][x >> 2][x & 3] = 0.0f;
        const int skip = (n + group) % LR_GROUPS;                       // the run's even steps are group 0's
#pragma unroll 1
        for (int k = k0 + skip; k < k1; k += LR_GROUPS) {
            const int here = n + k - k0;
            const LrPlace place = lr_place(here, a.slots);
            ok = ok && sg_wait_warp(pg_smem(&sh.full[place.bar]), place.parity, &sh.fail);
            const unsigned at = ring + place.slot * slot_bytes;
            float x[2][4];
#pragma unroll
            for (int i = 0; i < 8; i++) x[i >> 2][i & 3] = 0.0f;
#pragma unroll
            for (int i = 0; i < LR_KB; i++)
                if (kg + 4 * i < blocks) {
                    unsigned kb[4];
                    lt_ldsm(kb, at + k_lane + i * LR_BLOCK);
                    lt_mma(x[0], q[i], kb[0], kb[1]);
                    lt_mma(x[1], q[i], kb[2], kb[3]);
                }
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int y = 0; y < 2; y++) *(float2*)&sh.sums[group][kg][(lane >> 2) + y * 8][kh * 16 + i * 8 + (lane & 3) * 2] = make_float2(x[i][2 * y], x[i][2 * y + 1]);
            if (const int there = to - (from + k * LR_KEYS); there < LR_KEYS) {      // what lies behind a sequence's end has the weight 0, which would make a NaN of a NaN
                const unsigned n16 = (unsigned)(LR_KEYS - there) * 8 * ((a.cols + 63) >> 6);
                for (unsigned e = in_group; e < n16; e += LR_THREADS / LR_GROUPS)
                    lr_zero(at + e / ((LR_KEYS - there) * 8) * LR_BLOCK + there * 128 + e % ((LR_KEYS - there) * 8) * 16);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // before the slot's next rows
            }
            lr_sync(group);
            again();
            float z[2];
            {
                const float2 u0 = *(const float2*)&sh.sums[group][0][row][part * 2], u1 = *(const float2*)&sh.sums[group][1][row][part * 2], u2 = *(const float2*)&sh.sums[group][2][row][part * 2],
                             u3 = *(const float2*)&sh.sums[group][3][row][part * 2];
                const int key = from + k * LR_KEYS + part * 2;        // (a row sees no key behind `to`)
                z[0] = key <= pos && key >= key_lo ? ((u0.x + u1.x) + (u2.x + u3.x)) * f : -INFINITY;
                z[1] = key + 1 <= pos && key + 1 >= key_lo ? ((u0.y + u1.y) + (u2.y + u3.y)) * f : -INFINITY;
            }
            float mx = fmaxf(z[0], z[1]);
#pragma unroll
            for (int d = 1; d < 16; d *= 2) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            const float m_new = fmaxf(m, mx), base = m_new == -INFINITY ? 0.0f : m_new, alpha = m == m_new ? 1.0f : lt_exp2(m - m_new);
            m = m_new;
            z[0] = lt_exp2(z[0] - base + LR_SHIFT); z[1] = lt_exp2(z[1] - base + LR_SHIFT);
            l = fmaf(l, alpha, z[0] + z[1]);
            *(unsigned*)&sh.p[group][row][part * 2] = lt_pack(z[0], z[1]);
            if (part == 0) sh.alpha[group][row] = alpha;
            if (lr_sync_or(group, alpha != 1.0f)) {
                const float a0 = sh.alpha[group][lane >> 2], a1 = sh.alpha[group][(lane >> 2) + 8];
#pragma unroll
                for (int i = 0; i < LR_VB; i++)
#pragma unroll
                    for (int y = 0; y < 2; y++) { o[i][y][0] *= a0; o[i][y][1] *= a0; o[i][y][2] *= a1; o[i][y][3] *= a1; }
            }
#pragma unroll
            for (int kk = 0; kk < LR_KEYS / 16; kk++) {
                unsigned p[4];
                lt_ldsm(p, p_at + kk * 32);
#pragma unroll
                for (int i = 0; i < LR_VB; i++)
                    if (warp + 8 * i < v_blocks) {
                        unsigned v[4];
                        lt_ldsm_t(v, at + v_lane + kk * 2048 + i * 2 * LR_BLOCK);
                        lt_mma(o[i][0], p, v[0], v[1]);
                        lt_mma(o[i][1], p, v[2], v[3]);
                    }
            }
            last = here;
        }
        n += k1 - k0;
        // both groups' sums: group 1 gives the first half of its columns' blocks, group 0 the second.  A cut segment leaves its sums, the others their result
#pragma unroll
        for (int d = 1; d < 16; d *= 2) l += __shfl_xor_sync(0xffffffffu, l, d);
        if (part == 0) { sh.top[group][row] = m; sh.sum[group][row] = l; }
        float4* box = (float4*)&sh.sums[0][0][0][0] + in_group;
        auto give = [&](int half) {
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int y = 0; y < 2; y++) {
                    const float* v = o[half * 2 + i][y];
                    box[(i * 2 + y) * (LR_THREADS / LR_GROUPS)] = make_float4(v[0], v[1], v[2], v[3]);
                }
        };
        __syncthreads();                                              // scores and weights are read
        again();
        if (group == 1) give(0);
        const int place = 2 * blockIdx.x + (first ? 0 : 1);
        const bool any = k1 > k0 || !cut;
        float* lat = cut ? a.part + (size_t)place * LR_ROWS * a.rank : a.lat + ((int64_t)s.first * a.H + row0) * a.rank;
        float mine[2], other[2], by[2], both[2];                      // of the rows lane / 4 and that + 8: factors of the groups' sums, then of the result; the largest score
        unsigned wild = 0;
#pragma unroll
        for (int y = 0; y < 2; y++) {
            const int r = (lane >> 2) + y * 8;
            const float m0 = sh.top[0][r], m1 = sh.top[1][r], l0 = sh.sum[0][r], l1 = sh.sum[1][r], mm = fmaxf(m0, m1);
            const float f0 = m0 == -INFINITY ? (l0 == 0.0f ? 0.0f : 1.0f) : lt_exp2(m0 - mm), f1 = m1 == -INFINITY ? (l1 == 0.0f ? 0.0f : 1.0f) : lt_exp2(m1 - mm);
            float total = f0 * l0 + f1 * l1, g = 1.0f;
            if (cut) {
                by[y] = 1.0f;
                if (any && group == 0 && warp == 0 && (lane & 3) == 0) a.ml[(size_t)place * LR_ROWS + r] = make_float2(mm, total);
            } else {
                float all = total;
                if (a.sink && r < n_rows) {
                    const float sk = a.sink[(row0 + r) % a.H] * LR_LOG2E, m2 = fmaxf(mm, sk);
                    g = mm == -INFINITY ? (total == 0.0f ? 0.0f : 1.0f) : exp2f(mm - m2);
                    all = g * total + (sk == -INFINITY ? 0.0f : exp2f(sk - m2 + LR_SHIFT));
                }
                by[y] = g / all;
            }
            mine[y] = group ? f1 : f0; other[y] = group ? f0 : f1;
            both[y] = fabsf(total) < INFINITY ? mm : NAN;
        }
        auto finish = [&](int half) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int b = warp + 8 * (half * 2 + i);
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const float4 u = box[(i * 2 + c) * (LR_THREADS / LR_GROUPS)];
                    const float theirs[4] = {u.x, u.y, u.z, u.w};
                    if (b < v_blocks && any) {
#pragma unroll
                        for (int y = 0; y < 2; y++) {
                            const int r = (lane >> 2) + y * 8;
                            if (r >= n_rows) continue;
                            // (a group without keys has sums of 0 and the factor 0)
                            const float v0 = fmaf(o[half * 2 + i][c][2 * y], mine[y], theirs[2 * y] * other[y]), v1 = fmaf(o[half * 2 + i][c][2 * y + 1], mine[y], theirs[2 * y + 1] * other[y]);
                            if (!(fabsf(v0) < INFINITY && fabsf(v1) < INFINITY) && both[y] == both[y]) wild |= 1u << r;
                            *(float2*)(lat + (int64_t)r * a.rank + b * 16 + c * 8 + (lane & 3) * 2) = make_float2(v0 * by[y], v1 * by[y]);
                        }
                    }
                }
            }
        };
        __syncthreads();
        if (group == 0) finish(0);
        __syncthreads();
        if (group == 0) give(1);
        __syncthreads();
        if (group == 1) finish(1);
        if (wild) atomicOr(&sh.wild, wild);
        if (__syncthreads_or(wild != 0)) {
            for (unsigned left = sh.wild; left; left &= left - 1) {
                const int r = __ffs(left) - 1;
                float m, l, g = 1.0f;
                const float sum = lr_again(a, sh, s, seq, row0, from + k0 * LR_KEYS, min(to, from + k1 * LR_KEYS), r, m, l);
                if (cut) {
                    if (tid == 0) a.ml[(size_t)place * LR_ROWS + r] = make_float2(m, l);
                } else {
                    if (a.sink) {
                        const float sk = a.sink[(row0 + r) % a.H] * LR_LOG2E, m2 = fmaxf(m, sk);
                        g = m == -INFINITY ? 0.0f : exp2f(m - m2);
                        l = g * l + (sk == -INFINITY ? 0.0f : exp2f(sk - m2 + LR_SHIFT));
                    }
                    g /= l;
                }
                if (tid < a.rank) lat[(int64_t)r * a.rank + tid] = sum * g;
            }
            __syncthreads();
        }
        first = false;
    })) {}
    // no copy is under way when the CTA ends: all steps of the run have been waited for, but where a wait ran out
    if (*(volatile int*)&sh.fail)
        for (int i = 0; i < 1000; i++) __nanosleep(1000);
    if (tid == 0 && *(volatile int*)&sh.fail) {
        if (err_dev) atomicExch(err_dev, 5u);
        if (err_host) { *(volatile unsigned*)err_host = 5u; __threadfence_system(); }
    }
}
// segments in several runs: grid (segments, rows, COLS columns); a thread 4 columns of every SLICES-th slice.  Many slices, few segments: 64 columns a CTA, 16 slices at a time (one thread a column,
// one slice after another: 43 us for the 148 slices of a long cache, so 4); many segments of a few slices: all columns (64 sequences: 57 us a call, in columns of 64 77)
#define LJ_THREADS 256
template <int COLS>
__global__ void __launch_bounds__(LJ_THREADS) latent_join_kernel(const __grid_constant__ LrArgs a, const __grid_constant__ LrCuts cuts) {
    constexpr int SLICES = LJ_THREADS / (COLS / 4), TURNS = COLS == 64 ? (LR_CTAS + SLICES - 1) / SLICES : LJ_FEW / SLICES;
    __shared__ float factor[LR_CTAS], red[2][LJ_THREADS / 32];
    __shared__ float4 sums[SLICES][COLS / 4];
    pdl_enter();
    const auto cut = cuts.at[blockIdx.x];
    const PgSeq s = lr_clip(a.seqs[cut.seq], a);
    const int x = threadIdx.x, y = blockIdx.y, row = cut.tile * LR_ROWS + y, lane = x & 31, w = x >> 5, c = blockIdx.z * COLS + x % (COLS / 4) * 4, which = x / (COLS / 4);
    if (row >= s.count * a.H) return;
    auto place = [&](int i) { return (size_t)(i == 0 ? cut.slot : 2 * (cut.cta + i - 1)) * LR_ROWS + y; };
    static_assert(LR_CTAS <= LJ_THREADS, "a thread a slice");
    const float2 z = x < cut.n ? a.ml[place(x)] : make_float2(-INFINITY, 0.0f);
    float4 v[TURNS];
#pragma unroll
    for (int i = 0; i < TURNS; i++) {
        const int at = i * SLICES + which;
        v[i] = at < cut.n && c < a.rank ? *(const float4*)(a.part + place(at) * a.rank + c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    float m = warp_max(z.x);
    if (lane == 0) red[0][w] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LJ_THREADS / 32; i++) m = fmaxf(m, red[0][i]);
    const float f = z.x == -INFINITY ? (z.y == 0.0f ? 0.0f : 1.0f) : exp2f(z.x - m);
    if (x < LR_CTAS) factor[x] = f;
    float l = warp_sum(f * z.y);
    if (lane == 0) red[1][w] = l;
    __syncthreads();
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
    for (int i = 0; i < TURNS; i++) {
        const int at = i * SLICES + which;
        const float by = at < LR_CTAS ? factor[at] : 0.0f;
        if (by != 0.0f) { o.x = fmaf(by, v[i].x, o.x); o.y = fmaf(by, v[i].y, o.y); o.z = fmaf(by, v[i].z, o.z); o.w = fmaf(by, v[i].w, o.w); }
    }
    sums[which][x % (COLS / 4)] = o;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < LJ_THREADS / 32; i++) l += red[1][i];
    __syncthreads();
    float g = 1.0f;
    if (a.sink) {
        const float sk = a.sink[row % a.H] * LR_LOG2E, m2 = fmaxf(m, sk);
        g = m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : exp2f(m - m2);
        l = g * l + (sk == -INFINITY ? 0.0f : exp2f(sk - m2 + LR_SHIFT));
    }
    for (int col = x; col < COLS && blockIdx.z * COLS + col < a.rank; col += LJ_THREADS) {
        float t = 0.0f;
#pragma unroll
        for (int i = 0; i < SLICES; i++) t += ((const float*)sums[i])[col];
        a.lat[((int64_t)s.first * a.H + row) * a.rank + blockIdx.z * COLS + col] = t * (g / l);
    }
}

// the runs of deal.ctas CTAs over all steps, and the segments that are in several of them (returned: how many)
static int lr_deal(const cc_page_plan* plan, const LrArgs& a, int64_t steps, LrDeal& deal, LrCuts& cuts) {
    deal.run_lo = (int)(steps / deal.ctas); deal.run_more = (int)(steps % deal.ctas);
    int64_t before = 0, next = 0;                                  // steps in front of the sequence, and of run c
    int c = 0, n_cuts = 0;
    for (int seq = 0; seq < (int)plan->seqs.size() && c < deal.ctas; seq++) {
        const PgSeq s = lr_clip(plan->seqs[seq], a);
        const int n = lr_tiles(s, a), all = n ? lr_steps(s, a) : 0;
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
// the tokens a.token0 .. a.token1 - 1
static int lr_portion(cc_device* dev, const cc_page_plan* plan, LrArgs a) {
    int64_t steps = 0, tiles = 0;
    LtRuns runs{};
    for (const PgSeq& whole : plan->seqs) {
        const PgSeq s = lr_clip(whole, a);
        if (!s.count) continue;
        const int n = lr_tiles(s, a);
        tiles += n;
        steps += (int64_t)n * lr_steps(s, a);
        // many runs: the last one takes all that lies behind (results of other tokens are overwritten)
        if (runs.n && (runs.hi[runs.n - 1] == s.first || runs.n == LT_RUNS)) runs.hi[runs.n - 1] = s.first + s.count;
        else { runs.lo[runs.n] = s.first; runs.hi[runs.n++] = s.first + s.count; }
    }
    if (!tiles) return CC_OK;
    for (int i = 0; i < runs.n; i++) { runs.tile0[i] = runs.tiles; runs.tiles += (runs.hi[i] - runs.lo[i] + LT_TOKENS - 1) / LT_TOKENS; }
    LrDeal deal;
    LrCuts cuts;
    deal.ctas = (int)std::min<int64_t>(std::min(LR_CTAS, dev->sm_count), (steps + LR_BEGIN + 1) / (LR_BEGIN + 2));
    CC_REQUIRE(dev, steps / deal.ctas < 0x7ffffffe, "paged_latent_attention: too many rows");
    const int n_cuts = lr_deal(plan, a, steps, deal, cuts);
    const int64_t tokens = a.token1 - a.token0;
    const size_t qf = (size_t)tokens * a.H * a.cols * 4, lat = (size_t)tokens * a.H * a.rank * 4, part = n_cuts ? (size_t)2 * deal.ctas * LR_ROWS * a.rank * 4 : 0,
                 ml = (size_t)2 * deal.ctas * LR_ROWS * sizeof(float2), list = (size_t)deal.ctas * (deal.run_lo + 1) * sizeof(int4);
    void* ws = nullptr; size_t cls = 0;
    int rc = cc_pool_alloc(dev, qf + lat + part + ml + list, &ws, &cls);
    if (rc) return rc;
    // rows count from the call's first token
    a.qf = (float*)((uintptr_t)ws - (uintptr_t)a.token0 * a.H * a.cols * 4); a.lat = (float*)((uintptr_t)ws + qf - (uintptr_t)a.token0 * a.H * a.rank * 4); a.part = (float*)((uint8_t*)ws + qf + lat); a.ml = (float2*)((uint8_t*)ws + qf + lat + part);
    a.steps = (int4*)((uint8_t*)ws + qf + lat + part + ml);
    const int slot = (a.cols + 63) / 64 * LR_BLOCK;
    a.slots = std::min(LR_SLOTS, (LR_SMEM - (int)sizeof(LrShared) - 1024) / slot);
    // of a block of 64 columns: those behind a row's last whole one, and of pages shorter than a step all; of all whole ones
    CUtensorMap map, whole;
    const int box = std::min(plan->page, LR_KEYS);
    const bool by_blocks = a.cols % 64 || box < LR_KEYS, at_once = a.cols >= 64 && box == LR_KEYS;
    if (by_blocks) rc = cc_make_tmap_pages(dev, &map, a.rows, plan->n_pages, plan->page, a.cols, box, 0);
    if (!rc && at_once) rc = cc_make_tmap_pages(dev, &whole, a.rows, plan->n_pages, plan->page, a.cols, box, a.cols / 64);
    if (!by_blocks) map = whole;
    if (!at_once) whole = map;
    if (rc) { cc_pool_free(dev, ws, cls); return rc; }
    const unsigned z = (unsigned)std::min(runs.tiles, 64);
    const size_t fold = (size_t)a.dim * (LF_COLS + 8) * 2 + LT_TOKENS * (a.dim + 8) * 2;
    cudaError_t e = cc_smem_limit(dev, CC_LIMIT_LATENT, latent_fold_kernel, LT_DIM * (LF_COLS + 8) * 2 + LT_TOKENS * (LT_DIM + 8) * 2);
    if (e == cudaSuccess) e = cc_smem_limit(dev, CC_LIMIT_LATENT + 1, latent_rows_kernel, LR_SMEM - (int)sizeof(LrShared));
    if (e == cudaSuccess) e = cc_smem_limit(dev, CC_LIMIT_LATENT + 2, latent_unfold_kernel, lu_smem(LT_RANK));
    if (e == cudaSuccess) e = cc_launch_pdl(dev, latent_fold_kernel, dim3((unsigned)a.H, (unsigned)((a.rank + LF_COLS - 1) / LF_COLS + 1 + (deal.ctas + 4 * a.H - 1) / (4 * a.H)), z), 128, fold, a, runs, deal);
    if (e == cudaSuccess) e = cc_launch_pdl(dev, latent_rows_kernel, (unsigned)deal.ctas, LR_THREADS, (size_t)a.slots * slot + 1024, whole, map, a, deal, dev->err_dev, dev->err_host);
    if (e == cudaSuccess && n_cuts) {
        int most = 0;
        for (int i = 0; i < n_cuts; i++) most = std::max(most, cuts.at[i].n);
        e = most <= LJ_FEW ? cc_launch_pdl(dev, latent_join_kernel<LT_RANK>, dim3((unsigned)n_cuts, LR_ROWS, 1), LJ_THREADS, 0, a, cuts)
                           : cc_launch_pdl(dev, latent_join_kernel<64>, dim3((unsigned)n_cuts, LR_ROWS, (unsigned)(a.rank + 63) / 64), LJ_THREADS, 0, a, cuts);
        dev->launches++;
    }
    if (e == cudaSuccess) e = cc_launch_pdl(dev, latent_unfold_kernel, dim3((unsigned)a.H, (unsigned)((a.vdim + LU_COLS - 1) / LU_COLS), z), LU_THREADS, lu_smem(a.rank), a, runs);
    dev->launches += 3;
    cc_pool_free(dev, ws, cls);
    if (e != cudaSuccess) return cc_fail(dev, CC_ERR_CUDA, "paged_latent_attention: %s", cudaGetErrorString(e));
    return CC_OK;
}

// as many tokens at a time as have their queries and sums over the latents in LT_WORKSPACE
#define LT_WORKSPACE ((int64_t)256 << 20)
static int lr_run(cc_device* dev, const cc_page_plan* plan, LrArgs a) {
    const int64_t each = std::max<int64_t>(LT_TOKENS, LT_WORKSPACE / ((int64_t)a.H * (a.cols + a.rank) * 4) / LT_TOKENS * LT_TOKENS);
    for (int64_t t = 0; t < plan->tokens; t += each) {
        a.token0 = (int)t; a.token1 = (int)std::min(plan->tokens, t + each);
        const int rc = lr_portion(dev, plan, a);
        if (rc) return rc;
    }
    return CC_OK;
}
#include "latent_tile.cuh"

// New tokens of a sequence; with more its keys and values are laid out.  us, absorbed / expanded, of 8, 16, 24, 32, 64 tokens of one sequence:
// 16 heads of 128, rank 512, behind 1000 rows: 27 / 37, 29 / 37, 30 / 37, 34 / 42, 42 / 42; behind 8000: 34 / 77, 53 / 76, 63 / 76, 79 / 76, 133 / 77; behind 32000: 75 / 228, 131 / 229, 183 / 228, 236 / 229, 446 / 227;
// 32 heads of 64, rank 512, behind 8000: 53 / 104, 75 / 104, 105 / 102, 131 / 102, 243 / 103; of 8 sequences behind 1000: 60 / 103, 91 / 103, 130 / 104, 168 / 110, 324 / 111;
// 64 heads of 128, rank 512, 16 sequences behind 3000: 392 / 1734, 772 / 1736, 1145 / 1736, 1518 / 1734, 3041 / 1736
#define LT_FEW 24

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
    const bool expands = dim <= TL_DIM && vdim <= TL_DIM;
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
        rc = lr_run(dev, plan, a);
        if (!rc && a.most < 0x7fffffff) rc = tl_run(dev, plan, a);      // behind the others: their last products may run over tokens of these
    }
    if (rc) { cc_tensor_release(o); return rc; }
    *out = o;
    return CC_OK;
}
