// paged_attn.cu -- attention over the pages of a cache (include/crabml_paged.h).
//
// 32-bit results from 16-bit tensor-core products.  Codes and 16-bit numbers are exact as f16 operands; a query or weight x is two of them, h = f16(x) and
// l = f16(x - h), 22 bits together.  A query row is first brought near 2^14 by a power of two, weights go up to 2^14, so that l keeps its bits.
//
// Few rows (paged_few_kernel; a row is a query of one head).  mma.sync.m16n8k16 has room for 16 rows: eight rows' h above, the same rows' l below, and both
// products are one instruction whose accumulators a thread adds up itself.  A warp takes 16 keys at a time.  Its lanes keep, read and convert the pieces of the
// cache that the instruction's layout gives them and no others: which four columns of a row a lane puts into a step is free as long as queries and keys agree, and so
// is the order of the value columns, so a lane takes 16 neighbouring bytes of a row, and the way through shared memory (cp.async, a ring per warp) needs no barrier.
// Keys and values are read once, so memory bounds it: 64 sequences of up to 4000 tokens (268 MB, 41 us) take 79 us, 16 sequences in 16-bit pages (311 MB, 47 us) 75.  While all CTAs
// stream they read 5.6 to 6 TB/s; the rest is what a CTA does before and behind each segment (7 us to its first rows), and the kernel that adds up cut segments (5 us).
#include <math.h>

#include <algorithm>

#include "paged.cuh"

#define PT_WARPS 4
#define PT_THREADS (PT_WARPS * 32)
#define PT_SHIFT 9.0f                         // weights are exp2(score - base + PT_SHIFT), base the largest score so far, or up to PT_LAG less, so that the sums of a row are not scaled
#define PT_LAG 5.0f                           // again for every score that is a little larger.  Weights stay at 2^14, times a value factor's mantissa (below 2) below 2^15: f16 ends at 65504
#define PT_FAR 64.0f                          // 8-bit pages: products of a weight and its value's factor keep their bits down to 2^-64 of the largest weight (exp2 ends at 2^-126)
#define PT_STEP 64                            // keys that few rows are dealt out by
#define PT_BEGIN 5                            // what a segment's begin and end cost, in steps (finding it, the queries, the sums: 13 thousand cycles)
#define PT_CHUNK 4096                         // keys whose page numbers and factors a CTA holds at a time
#define PT_FEW 32                             // rows of a sequence and key head, 8 at a time; more go to tiles of 128.  16 sequences at 2000 tokens, 32 heads on 8, 8-bit pages, us by 8 and by 128:
                                              // 16 rows 52 and 118, 32 rows 86 and 123, 64 rows 149 and 135; one sequence at 4000: 25 and 39 with 32 rows, 49 and 42 with 128
#define PT_TILE 72                            // floats from one tile of 8 x 8 sums to the next
#define PT_LOG2E 1.4426950408889634f

struct TiInfo;
struct PtArgs {
    const PgSeq* seqs;
    const int* table;
    const uint8_t *k, *v;
    const float *ks, *vs, *q, *sink;
    const __half *ko, *vo;
    float *out, *part;                        // part: [item][head][tile_rows][dv] sums of a slice (few rows: [2 x CTA][8][dv], of its first and its last segment)
    float2* ml;                               // [item][head][tile_rows]: largest score (base 2) and sum of weights
    float scale, softcap;
    int n_seqs, table_cols, page, shift, H, G, R, dk, dv, window, split, rows_lo, rows_hi;
    int tile_rows, align;                     // of an item: 8 (paged_few_kernel) or 128 (paged_tile_kernel); what keys count from is a multiple of align
    int head0, heads;                         // key heads of this launch
    uint8_t *k_image, *v_image;               // paged_tile.cuh
    struct TiInfo* info;
};
// few rows: segments are (sequence, 8 rows, key head), of steps of PT_STEP keys behind PT_BEGIN more for the segment itself.  `ctas` CTAs take equal runs of them: where the run of CTA c
// begins, dealt out on the host (a search by each CTA took 3 to 5 us at the start); ctas 0: a CTA a segment
#define PT_CTAS 592
struct PtDeal { int ctas, run_lo, run_more; struct { int seq, seg, off; } at[PT_CTAS]; };      // the first run_more runs are of run_lo + 1 steps
struct PtCuts { struct { int seq, seg, slot, cta, n; } at[PT_CTAS]; };      // segments that are in several runs: the place of the first one's sums, the next CTA, how many
struct PtItem { int seq, split, tile, n_split; };

// keys [from, to) that the sequence's new tokens see together
__host__ __device__ __forceinline__ void pt_range(const PgSeq& s, const PtArgs& a, int* from, int* to) {
    *to = s.pos0 + s.count;
    *from = a.window > 0 && s.pos0 - a.window + 1 > 0 ? (s.pos0 - a.window + 1) & ~(a.align - 1) : 0;
}
__host__ __device__ __forceinline__ int pt_splits(const PgSeq& s, const PtArgs& a) {
    const int64_t rows = (int64_t)s.count * a.R;
    if (rows < a.rows_lo || rows > a.rows_hi) return 0;
    int from, to;
    pt_range(s, a, &from, &to);
    return (to - from - 1) / a.split + 1;
}
// keys of a slice: the sequence's in equal parts
__host__ __device__ __forceinline__ int pt_each(int keys, int n_split) { return ((keys + n_split - 1) / n_split + 127) / 128 * 128; }
// few rows: a segment is (sequence, 8 rows, key head); a sequence's segments, and the steps of each
__host__ __device__ __forceinline__ int pt_segments(const PgSeq& s, const PtArgs& a) {
    const int64_t rows = (int64_t)s.count * a.R;
    return rows < a.rows_lo || rows > a.rows_hi ? 0 : (int)((rows + 7) / 8) * a.G;
}
__host__ __device__ __forceinline__ int pt_steps(const PgSeq& s, const PtArgs& a) {
    int from, to;
    pt_range(s, a, &from, &to);
    return PT_BEGIN + (to - from + PT_STEP - 1) / PT_STEP;
}
// the place of number n in the sequences' counts: every lane gets the sequence and what is left of n
template <class Count>
__device__ __forceinline__ int pt_find(const PtArgs& a, int n, Count count, int* rest) {
    const int lane = threadIdx.x & 31;
    for (int s0 = 0; s0 < a.n_seqs; s0 += 32) {
        const int s = s0 + lane, mine = s < a.n_seqs ? count(a.seqs[s]) : 0;
        int sum = mine;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, n < sum);
        if (hit) {
            const int l = __ffs(hit) - 1;
            *rest = n - __shfl_sync(0xffffffffu, sum - mine, l);
            return s0 + l;
        }
        n -= __shfl_sync(0xffffffffu, sum, 31);
    }
    return -1;
}

__device__ __forceinline__ void pt_copy4(unsigned dst, const void* src) { asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory"); }
__device__ __forceinline__ void pt_copy16(unsigned dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void pt_copy8(unsigned dst, const void* src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(there ? 8 : 0) : "memory");
}
__device__ __forceinline__ void pt_mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// two 8-bit numbers, 128 added to each, in the bytes that `pick` takes, as f16: 1024 + 128 + x is 0x6400 | byte, and 1152 leaves exactly
__device__ __forceinline__ unsigned pt_half2(unsigned biased, unsigned pick) {
    const unsigned u = __byte_perm(biased, 0x64646464u, pick);
    const __half2 h = __hsub2(*(const __half2*)&u, __floats2half2_rn(1152.0f, 1152.0f));
    return *(const unsigned*)&h;
}
__device__ __forceinline__ unsigned pt_pack(float x, float y) {
    const __half2 h = __floats2half2_rn(x, y);
    return *(const unsigned*)&h;
}
// 2^x; what is below 2^-126 is 0
__device__ __forceinline__ float pt_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// x, y as f16 (h) and what is left of them as f16 (l)
__device__ __forceinline__ void pt_cut(float x, float y, unsigned& h, unsigned& l) {
    const __half2 a = __floats2half2_rn(x, y);
    const float2 b = __half22float2(a);
    h = *(const unsigned*)&a;
    l = pt_pack(x - b.x, y - b.y);
}
// halves that are an infinity or a NaN: as a mask of 16 ones each
__device__ __forceinline__ unsigned pt_wild(unsigned u) {
    return ((u & 0x7c00u) == 0x7c00u ? 0xffffu : 0u) | ((u & 0x7c000000u) == 0x7c000000u ? 0xffff0000u : 0u);
}

// what a warp keeps of its eight rows
template <int D>
struct PtRows {
    unsigned q[D / 16][4];                    // h and l of the lane's columns, as the instruction takes them
    float o[D / 8][4];                        // sums of weighted values: tile i, columns 2 t and 2 t + 1 of its eight, rows h and l
    float inv, m, l, n, c;                    // power of two that q was divided by; base of the weights; the lane's sum of weights; base of the products of a weight and its value's factor, which o is in; 2^(m - n)
    int pos, lo;                              // the row's position and the first key it sees (pos -1: no row)
};
// 2^x of a whole number; 0 below 2^-126 and for NaN
__device__ __forceinline__ float pt_pow2(float x) { return __int_as_float(((int)fminf(fmaxf(x, -127.0f), 128.0f) + 127) << 23); }
// the power of two below a factor, as a score: what it adds to the scores of its block; -inf for a block of zeros
__device__ __forceinline__ float pt_log2(float vf) { return vf > 0.0f ? (float)((__float_as_int(vf) >> 23) - 127) : -INFINITY; }
// 16 scores of the row -> weights; x: raw sums of keys 2 t, 2 t + 1, 8 + 2 t, 9 + 2 t.  kf, vf: the keys' and values' factors.  edge: some row does not see some key.
// FACTORS (8-bit pages): a row's largest weight and its largest product of a weight and a factor may lie in blocks whose factors are far apart; the weights' sum counts from the one (m), the
// operands of the values' product from the other (n), so that the product that counts keeps its bits whatever the factors of others.  Both are whole numbers: what is scaled is exact
template <int D, bool FACTORS>
__device__ __forceinline__ void pt_weights(PtRows<D>& r, float (&x)[4], int key0, float kf, float vf, bool edge, const PtArgs& a, unsigned (&p)[4], unsigned& seen) {
    const int t = threadIdx.x & 3;
    const float f = a.softcap > 0.0f ? r.inv * kf * a.scale : r.inv * kf * (a.scale * PT_LOG2E);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[i] *= f;
        if (a.softcap > 0.0f) x[i] = a.softcap * tanhf(x[i] / a.softcap) * PT_LOG2E;
    }
    seen = 15u;
    if (edge) {
        seen = 0u;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int key = key0 + (i >> 1) * 8 + 2 * t + (i & 1);
            if (key <= r.pos && key >= r.lo) seen |= 1u << i;
            else x[i] = -INFINITY;
        }
    }
    float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    // differences of scores before anything is added to them: from 2^27 on a score's last place is more than PT_LAG or PT_SHIFT, which the sum would round to more than f16 has room for
    const float top = FACTORS ? mx + pt_log2(vf) : mx;
    const bool up = mx - r.m > PT_LAG, more = FACTORS && top - r.n > PT_LAG;      // (r.m, r.n -inf: every score is more)
    if (__any_sync(0xffffffffu, up || more)) {
        float alpha = 1.0f;
        if (up) {
            const float m = FACTORS ? ceilf(mx) : mx;
            alpha = r.m == -INFINITY ? 0.0f : FACTORS ? pt_pow2(r.m - m) : pt_exp2(r.m - m);
            r.m = m;
            r.l *= alpha;
        }
        if (FACTORS) {
            const float n = fmaxf(more ? ceilf(top) : r.n, r.m - PT_FAR);
            alpha = n == r.n || r.n == -INFINITY ? 1.0f : pt_pow2(r.n - n);      // (nothing in o so far but zeros)
            r.n = n;
            r.c = pt_pow2(r.m - n);
        }
#pragma unroll
        for (int i = 0; i < D / 8; i++) { r.o[i][0] *= alpha; r.o[i][1] *= alpha; r.o[i][2] *= alpha; r.o[i][3] *= alpha; }
    }
    const float base = r.m == -INFINITY ? 0.0f : r.m, vr = FACTORS ? vf * r.c : vf;
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = pt_exp2((x[i] - base) + PT_SHIFT);
    r.l += (x[0] + x[1]) + (x[2] + x[3]);
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = seen & (1u << i) ? x[i] * vr : 0.0f;
    pt_cut(x[0], x[1], p[0], p[1]);
    pt_cut(x[2], x[3], p[2], p[3]);
}

// ---- 16 keys of 8-bit codes ----------------------------------------------------------------------------------------------------------------
template <int D>
struct PtI8 {
    static constexpr int KC = D / 64, VB = D == 64 ? 8 : 16, VC = D == 64 ? 1 : D / 128, BYTES = 32 * D;
    static __device__ __forceinline__ void load(unsigned st, const uint8_t* k, const uint8_t* v, const PtArgs& a) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int c = 0; c < KC; c++) {
                const bool in = c * 64 + t * 16 < a.dk;
                pt_copy16(st + (j * KC + c) * 512 + lane * 16, in ? k + (8 * j + g) * a.dk + c * 64 + t * 16 : k, in);
            }
        st += 2 * KC * 512;
#pragma unroll
        for (int x = 0; x < 4; x++)
#pragma unroll
            for (int c = 0; c < VC; c++) {
                const int col = c * 128 + g * VB, key = 2 * t + (x & 1) + (x >> 1) * 8;
                const bool in = col < a.dv;
                if (VB == 8) pt_copy8(st + x * 256 + lane * 8, in ? v + key * a.dv + col : v, in);
                else pt_copy16(st + (x * VC + c) * 512 + lane * 16, in ? v + key * a.dv + col : v, in);
            }
    }
    static __device__ __forceinline__ void use(PtRows<D>& r, const uint8_t* st, int key0, float kf, float vf, bool edge, const PtArgs& a) {
        const int lane = threadIdx.x & 31;
        float s[2][4];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
#pragma unroll
            for (int c = 0; c < KC; c++) {
                const uint4 w4 = *(const uint4*)(st + (j * KC + c) * 512 + lane * 16);
                const unsigned w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const unsigned u = w[e] ^ 0x80808080u;
                    pt_mma(s[j], r.q[c * 4 + e], pt_half2(u, 0x4140), pt_half2(u, 0x4342));
                }
            }
        }
        float x[4] = {s[0][0] + s[0][2], s[0][1] + s[0][3], s[1][0] + s[1][2], s[1][1] + s[1][3]};
        unsigned p[4], seen;
        pt_weights<D, true>(r, x, key0, kf, vf, edge, a, p, seen);
        st += 2 * KC * 512;
#pragma unroll
        for (int c = 0; c < VC; c++) {
            unsigned w[4][4];
#pragma unroll
            for (int y = 0; y < 4; y++) {
                if (VB == 8) {
                    const uint2 v = *(const uint2*)(st + y * 256 + lane * 8);
                    w[y][0] = v.x ^ 0x80808080u; w[y][1] = v.y ^ 0x80808080u;
                } else {
                    const uint4 v = *(const uint4*)(st + (y * VC + c) * 512 + lane * 16);
                    w[y][0] = v.x ^ 0x80808080u; w[y][1] = v.y ^ 0x80808080u; w[y][2] = v.z ^ 0x80808080u; w[y][3] = v.w ^ 0x80808080u;
                }
            }
#pragma unroll
            for (int e = 0; e < VB / 4; e++) {
                const unsigned a01 = __byte_perm(w[0][e], w[1][e], 0x5140), a23 = __byte_perm(w[0][e], w[1][e], 0x7362);
                const unsigned b01 = __byte_perm(w[2][e], w[3][e], 0x5140), b23 = __byte_perm(w[2][e], w[3][e], 0x7362);
                float(*o)[4] = r.o + c * 16 + e * 4;
                pt_mma(o[0], p, pt_half2(a01, 0x4140), pt_half2(b01, 0x4140));
                pt_mma(o[1], p, pt_half2(a01, 0x4342), pt_half2(b01, 0x4342));
                pt_mma(o[2], p, pt_half2(a23, 0x4140), pt_half2(b23, 0x4140));
                pt_mma(o[3], p, pt_half2(a23, 0x4342), pt_half2(b23, 0x4342));
            }
        }
    }
};
// ---- 16 keys of 16-bit numbers.  WIDE: with the columns dealt out as for codes (a block that is open beside pages of codes) ------------------------------
template <int D, bool WIDE>
struct PtF16 {
    static constexpr int EK = WIDE ? 16 : 8, KC = D / (4 * EK), KP = EK / 8;          // elements of a lane and chunk of a key row; 16-byte pieces of them
    static constexpr int CW = WIDE && D >= 128 ? 128 : 64, VC = D / CW, VP = CW / 64, BYTES = 64 * D;
    // rows from `there` on are zeros
    static __device__ __forceinline__ void load(unsigned st, const __half* k, const __half* v, int there, const PtArgs& a) {
        const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int c = 0; c < KC; c++)
#pragma unroll
                for (int h = 0; h < KP; h++) {
                    const int col = c * 4 * EK + t * EK + h * 8, key = 8 * j + g;
                    const bool in = col < a.dk && key < there;
                    pt_copy16(st + ((j * KC + c) * KP + h) * 512 + lane * 16, in ? k + key * a.dk + col : k, in);
                }
        st += 2 * KC * KP * 512;
#pragma unroll
        for (int x = 0; x < 4; x++)
#pragma unroll
            for (int c = 0; c < VC; c++)
#pragma unroll
                for (int h = 0; h < VP; h++) {
                    const int col = c * CW + g * (CW / 8) + h * 8, key = 2 * t + (x & 1) + (x >> 1) * 8;
                    const bool in = col < a.dv && key < there;
                    pt_copy16(st + ((x * VC + c) * VP + h) * 512 + lane * 16, in ? v + key * a.dv + col : v, in);
                }
    }
    static __device__ __forceinline__ void use(PtRows<D>& r, const uint8_t* st, int key0, bool edge, const PtArgs& a) {
        const int lane = threadIdx.x & 31;
        float s[2][4];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
#pragma unroll
            for (int c = 0; c < KC * KP; c++) {
                const uint4 w = *(const uint4*)(st + (j * KC * KP + c) * 512 + lane * 16);
                pt_mma(s[j], r.q[c * 2], w.x, w.y);
                pt_mma(s[j], r.q[c * 2 + 1], w.z, w.w);
            }
        }
        float x[4] = {s[0][0] + s[0][2], s[0][1] + s[0][3], s[1][0] + s[1][2], s[1][1] + s[1][3]};
        unsigned p[4], seen;
        pt_weights<D, WIDE>(r, x, key0, 1.0f, 1.0f, edge, a, p, seen);
        st += 2 * KC * KP * 512;
        // a value that is not finite must not meet a weight of zero in the sums of a row that does not see it
        bool wild = false;
        if (edge) {
#pragma unroll 1
            for (int y = 0; y < 4 * VC * VP; y++) {
                const uint4 v = *(const uint4*)(st + y * 512 + lane * 16);
                wild |= (pt_wild(v.x) | pt_wild(v.y) | pt_wild(v.z) | pt_wild(v.w)) != 0u;
            }
            wild = __any_sync(0xffffffffu, wild);
        }
#pragma unroll
        for (int c = 0; c < VC * VP; c++) {
            unsigned w[4][4];
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const uint4 v = *(const uint4*)(st + (y * VC * VP + c) * 512 + lane * 16);
                w[y][0] = v.x; w[y][1] = v.y; w[y][2] = v.z; w[y][3] = v.w;
            }
#pragma unroll
            for (int e = 0; e < 8; e++) {
                unsigned b0 = __byte_perm(w[0][e / 2], w[1][e / 2], e & 1 ? 0x7632 : 0x5410), b1 = __byte_perm(w[2][e / 2], w[3][e / 2], e & 1 ? 0x7632 : 0x5410);
                if (wild) {                                        // how many of them each row sees, by a product of ones; the sums of those that do are NaN
                    const unsigned w0 = pt_wild(b0), w1 = pt_wild(b1);
                    const unsigned ones[4] = {(seen & 1u ? 0x3c00u : 0u) | (seen & 2u ? 0x3c000000u : 0u), 0u, (seen & 4u ? 0x3c00u : 0u) | (seen & 8u ? 0x3c000000u : 0u), 0u};
                    float n[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    pt_mma(n, ones, w0 & 0x3c003c00u, w1 & 0x3c003c00u);
                    if (n[0] > 0.0f) r.o[c * 8 + e][0] = NAN;
                    if (n[1] > 0.0f) r.o[c * 8 + e][1] = NAN;
                    b0 &= ~w0; b1 &= ~w1;
                }
                pt_mma(r.o[c * 8 + e], p, b0, b1);
            }
        }
    }
};

template <int D, bool I8>
__global__ void __launch_bounds__(PT_THREADS, D <= 64 ? 4 : D <= 128 ? 3 : 1) paged_few_kernel(const PtArgs a, const __grid_constant__ PtDeal deal) {
    using Mine = PtF16<D, I8>;                                     // 16-bit rows: pages, or the open block beside codes
    constexpr int RING = 128 * D, STAGES = RING / Mine::BYTES, STAGES8 = RING / PtI8<D>::BYTES, CW = I8 && D >= 128 ? 128 : 64;
    extern __shared__ __align__(16) uint8_t pt_sm[];
    __shared__ int pid[PT_CHUNK / 16 + 1];
    __shared__ float kfs[PT_CHUNK / 16 + 1], vfs[PT_CHUNK / 16 + 1];
    __shared__ float2 ml[PT_WARPS][8];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    uint8_t* ring = pt_sm + w * RING;
    const unsigned ring_at = (unsigned)__cvta_generic_to_shared(ring);
    pdl_enter();
    // this CTA's run of steps; pieces of it, a segment each
    const int c = blockIdx.x, run = deal.ctas ? deal.run_lo + (c < deal.run_more ? 1 : 0) : 1;
    int seq, seg, off = 0, more = 0;                               // more: segments of the sequence behind this one
    if (deal.ctas) {
        seq = deal.at[c].seq; seg = deal.at[c].seg; off = deal.at[c].off;
        more = pt_segments(a.seqs[seq], a) - 1 - seg;
    } else if ((seq = pt_find(a, c, [&](const PgSeq& s) { return pt_segments(s, a); }, &seg)) < 0) return;
    for (int at = 0; at < run;) {
    int from, to;
    if (at > 0) {
        off = 0;
        if (more-- > 0) seg++;
        else {
            do if (++seq >= a.n_seqs) return;
            while ((more = pt_segments(a.seqs[seq], a) - 1) < 0);
            seg = 0;
        }
    }
    const PgSeq s = a.seqs[seq];
    pt_range(s, a, &from, &to);
    const int all = pt_steps(s, a), upto = deal.ctas ? min(all, off + run - at) : all;
    const int rows = s.count * a.R, nth = seg / a.G, kvh = seg - nth * a.G, tile = deal.ctas ? nth : (rows + 7) / 8 - 1 - nth, slot = 2 * c + (at == 0 ? 0 : 1);
    const bool whole = off <= PT_BEGIN && upto == all;
    at += upto - off;
    if (upto <= PT_BEGIN) break;                                   // the next CTA has all its keys
    const int row = tile * 8 + g, tok = row / a.R, pos_first = s.pos0 + tile * 8 / a.R, pos_last = s.pos0 + (min(rows, tile * 8 + 8) - 1) / a.R;
    const int k0 = from + max(off - PT_BEGIN, 0) * PT_STEP, k1 = min(min(to, from + (upto - PT_BEGIN) * PT_STEP), pos_last + 1);       // keys of the piece that some row of the tile may see
    const int lo0 = a.window > 0 ? max(k0, (pos_first - a.window + 1) & ~15) : k0, opens = I8 ? to >> a.shift << a.shift : 0;      // opens: the first key that is not in a page of codes
    // the lane's columns of its row
    const bool in = row < rows;
    constexpr int E = I8 ? 16 : 8;
    PtRows<D> r;
    float v[D / 4];
    {
        const float* q = a.q + ((int64_t)(s.first + (in ? tok : 0)) * a.H + kvh * a.R + (in ? row - tok * a.R : 0)) * a.dk;
#pragma unroll
        for (int i = 0; i < D / 4; i++) {
            const int col = i / E * 4 * E + t * E + i % E;
            v[i] = in && col < a.dk ? q[col] : 0.0f;
        }
    }
    for (int lo = lo0;; lo += PT_CHUNK) {                          // (once, but for the longest pieces)
    const int hi = min(k1, lo + PT_CHUNK), units = hi > lo ? (hi - lo + 15) >> 4 : 0, p0 = lo >> a.shift;
    const int n_pages = units > 0 ? ((hi - 1) >> a.shift) - p0 + 1 : 0, units8 = I8 ? max(0, min(units, (opens - lo) >> 4)) : 0;
    for (int i = threadIdx.x; i < n_pages; i += PT_THREADS) pid[i] = a.table[(int64_t)seq * a.table_cols + p0 + i];
    __syncthreads();
    // 16 keys' rows on their way into a place of the ring: codes, and 16-bit rows (`first` on: this warp's units behind the codes)
    auto load8 = [&](int u) {
        if (I8 && u < units8) {
            const int key0 = lo + u * 16;
            const size_t at = ((size_t)pid[(key0 >> a.shift) - p0] * a.G + kvh) * a.page + (key0 & (a.page - 1));
            PtI8<D>::load(ring_at + (u / PT_WARPS % STAGES8) * PtI8<D>::BYTES, a.k + at * a.dk, a.v + at * a.dv, a);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const __half *kb = I8 ? a.ko : (const __half*)a.k, *vb = I8 ? a.vo : (const __half*)a.v;
    auto load16 = [&](int u) {
        if (u < units) {
            const int key0 = lo + u * 16;
            const size_t block = I8 ? (size_t)(2 * s.slot + ((to >> a.shift) & 1)) : (size_t)pid[(key0 >> a.shift) - p0], at = (block * a.G + kvh) * a.page + (key0 & (a.page - 1));
            Mine::load(ring_at + (u / PT_WARPS % STAGES) * Mine::BYTES, kb + at * a.dk, vb + at * a.dv, to - key0, a);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    const int first = units8 + (w - units8 % PT_WARPS + PT_WARPS) % PT_WARPS;
    if (I8)
        for (int i = threadIdx.x; i < n_pages; i += PT_THREADS) {     // (copies too, that the first rows bring with them)
            const size_t at = (size_t)pid[i] * a.G + kvh;
            pt_copy4((unsigned)__cvta_generic_to_shared(kfs + i), a.ks + at);
            pt_copy4((unsigned)__cvta_generic_to_shared(vfs + i), a.vs + at);
        }
    // the first rows come while the queries are cut
    if (I8) {
#pragma unroll
        for (int i = 0; i < STAGES8 - 1; i++) load8(w + i * PT_WARPS);
    } else load16(first);
    if (lo == lo0) {
        float top = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 4; i++) top = fmaxf(top, fabsf(v[i]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        int ex = 14;
        if (top > 0.0f && top < INFINITY) frexpf(top, &ex);
        ex = max(ex, -100);
        const float f = ldexpf(1.0f, 14 - ex);
        r.inv = ldexpf(1.0f, ex - 14);
#pragma unroll
        for (int i = 0; i < D / 16; i++) {
            pt_cut(v[4 * i] * f, v[4 * i + 1] * f, r.q[i][0], r.q[i][1]);
            pt_cut(v[4 * i + 2] * f, v[4 * i + 3] * f, r.q[i][2], r.q[i][3]);
        }
        r.pos = in ? s.pos0 + tok : -1;
        r.lo = a.window > 0 ? r.pos - a.window + 1 : 0;
        r.m = r.n = -INFINITY; r.l = r.c = 0.0f;
#pragma unroll
        for (int i = 0; i < D / 8; i++) r.o[i][0] = r.o[i][1] = r.o[i][2] = r.o[i][3] = 0.0f;
    }
    if (I8) asm volatile("cp.async.wait_group %0;" ::"n"(STAGES8 - 2) : "memory");
    __syncthreads();
    auto edge = [&](int key0) { return key0 + 15 > pos_first || (a.window > 0 && key0 < pos_last - a.window + 1); };
    if constexpr (I8) {
        for (int u = w; u < units8; u += PT_WARPS) {
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES8 - 2) : "memory");
            load8(u + (STAGES8 - 1) * PT_WARPS);
            const int key0 = lo + u * 16, i = (key0 >> a.shift) - p0;
            PtI8<D>::use(r, ring + (u / PT_WARPS % STAGES8) * PtI8<D>::BYTES, key0, kfs[i], vfs[i], edge(key0), a);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
        load16(first);
    }
    for (int u = first; u < units; u += PT_WARPS) {
        load16(u + PT_WARPS);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
        const int key0 = lo + u * 16;
        Mine::use(r, ring + (u / PT_WARPS % STAGES) * Mine::BYTES, key0, edge(key0), a);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();                                               // the rings, page numbers and factors are free
    if (hi >= k1) break;
    }
    // the warps' sums, in the order of the warps
    r.l += __shfl_xor_sync(0xffffffffu, r.l, 1);
    r.l += __shfl_xor_sync(0xffffffffu, r.l, 2);
    // [warp][tile of 8 columns][row][column], tiles PT_TILE floats apart: no two lanes in one bank, neither here nor below
    float* sums = (float*)pt_sm;
    const float back = I8 ? pt_pow2(r.n - r.m) : 1.0f;             // (no key: both -inf, all 0)
#pragma unroll
    for (int i = 0; i < D / 8; i++)
        *(float2*)(sums + (w * (D / 8) + i) * PT_TILE + g * 8 + 2 * t) = make_float2((r.o[i][0] + r.o[i][2]) * back, (r.o[i][1] + r.o[i][3]) * back);
    if (t == 0) ml[w][g] = make_float2(r.m, r.l);
    __syncthreads();
    const int n = min(8, rows - tile * 8);
    for (int e = threadIdx.x; e < n * D; e += PT_THREADS) {
        const int y = e / D, i = e % D >> 3, x8 = e & 7, col = i / (CW / 8) * CW + x8 * (CW / 8) + i % (CW / 8);      // column x8 of tile i
        if (col >= a.dv) continue;
        float m = -INFINITY, l = 0.0f, o = 0.0f;
#pragma unroll
        for (int x = 0; x < PT_WARPS; x++) m = fmaxf(m, ml[x][y].x);
#pragma unroll
        for (int x = 0; x < PT_WARPS; x++) {
            const float f = ml[x][y].x == -INFINITY ? (ml[x][y].y == 0.0f ? 0.0f : 1.0f) : exp2f(ml[x][y].x - m);
            l = fmaf(f, ml[x][y].y, l);
            o = fmaf(f, sums[(x * (D / 8) + i) * PT_TILE + y * 8 + x8], o);
        }
        if (!whole) {
            a.part[((size_t)slot * 8 + y) * a.dv + col] = o;
            if (col == 0) a.ml[slot * 8 + y] = make_float2(m, l);
            continue;
        }
        const int rr = tile * 8 + y, tk = rr / a.R, head = kvh * a.R + rr - tk * a.R;
        if (a.sink) {
            const float sk = a.sink[head] * PT_LOG2E, m2 = fmaxf(m, sk), f = m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : exp2f(m - m2);
            l = f * l + (sk == -INFINITY ? 0.0f : exp2f(sk - m2 + PT_SHIFT));
            o *= f;
        }
        a.out[((int64_t)(s.first + tk) * a.H + head) * a.dv + col] = o / l;
    }
    __syncthreads();                                               // the sums, before the next piece's rows
    }
}
#define PT_JOIN 4                             // warps
// n slices of a row added up by a CTA: a warp takes every PT_JOINth of them, a lane 4 neighbouring columns; part and ml of slice x at place(x)
template <class Place>
__device__ __forceinline__ void pt_join(const PtArgs& a, int n, Place place, float* out, int head) {
    __shared__ float so[PT_JOIN][256];
    __shared__ float2 sm[PT_JOIN];
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    float m = -INFINITY;
    for (int x = lane; x < n; x += 32) m = fmaxf(m, a.ml[place(x)].x);
    m = warp_max(m);
    float l = 0.0f;
    for (int c0 = 0; c0 < a.dv; c0 += 128) {
        const int col = c0 + lane * 4;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float sum = 0.0f;
#pragma unroll 4
        for (int x = w; x < n; x += PT_JOIN) {
            const float2 z = a.ml[place(x)];
            const float f = z.x == -INFINITY ? (z.y == 0.0f ? 0.0f : 1.0f) : exp2f(z.x - m);
            sum = fmaf(f, z.y, sum);
            if (col < a.dv) {
                const float4 v = *(const float4*)(a.part + place(x) * a.dv + col);
                o.x = fmaf(f, v.x, o.x); o.y = fmaf(f, v.y, o.y); o.z = fmaf(f, v.z, o.z); o.w = fmaf(f, v.w, o.w);
            }
        }
        l = sum;
        if (col < a.dv) *(float4*)&so[w][col] = o;
    }
    if (lane == 0) sm[w] = make_float2(m, l);
    __syncthreads();
    l = 0.0f;
#pragma unroll
    for (int x = 0; x < PT_JOIN; x++) l += sm[x].y;
    float f = 1.0f;
    if (a.sink) {
        const float sk = a.sink[head] * PT_LOG2E, m2 = fmaxf(m, sk);
        f = m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : exp2f(m - m2);
        l = f * l + (sk == -INFINITY ? 0.0f : exp2f(sk - m2 + PT_SHIFT));
    }
    for (int c = threadIdx.x; c < a.dv; c += 32 * PT_JOIN) {
        float o = 0.0f;
#pragma unroll
        for (int x = 0; x < PT_JOIN; x++) o += so[x][c];
        out[c] = o * f / l;
    }
}
// few rows: grid (segments in several runs, 8 rows)
__global__ void __launch_bounds__(32 * PT_JOIN) paged_join_kernel(const PtArgs a, const __grid_constant__ PtCuts cuts) {
    pdl_enter();
    const auto cut = cuts.at[blockIdx.x];
    const PgSeq s = a.seqs[cut.seq];
    const int y = blockIdx.y, tile = cut.seg / a.G, kvh = cut.seg - tile * a.G, row = tile * 8 + y;
    if (row >= s.count * a.R) return;
    const int tok = row / a.R, head = kvh * a.R + row - tok * a.R;
    pt_join(a, cut.n, [&](int x) { return (size_t)(x == 0 ? cut.slot : 2 * (cut.cta + x - 1)) * 8 + y; }, a.out + ((int64_t)(s.first + tok) * a.H + head) * a.dv, head);
}
// tiles of 128 rows: the slices of a row, grid (PT_SUM rows of a sequence, key heads); a warp a row, four times, a lane 4 neighbouring columns.  (A CTA a row, which finds its place by itself: 6600
// rows of 8 key heads took 107 us longer in two slices than in one, 42 so)
#define PT_SUM 32
__global__ void __launch_bounds__(256) paged_sum_kernel(const PtArgs a) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, kvh = a.head0 + blockIdx.y, col = lane * 4;
    pdl_enter();
    int group, items = 0;
    const int seq = pt_find(a, blockIdx.x, [&](const PgSeq& s) { return pt_splits(s, a) > 1 ? (s.count * a.R + PT_SUM - 1) / PT_SUM : 0; }, &group);
    if (seq < 0) return;
    for (int x = lane; x < seq; x += 32) items += pt_splits(a.seqs[x], a) * ((a.seqs[x].count * a.R + a.tile_rows - 1) / a.tile_rows);
    items = warp_sum_i(items);
    const PgSeq s = a.seqs[seq];
    const int tiles = (s.count * a.R + a.tile_rows - 1) / a.tile_rows, n = pt_splits(s, a), end = min(s.count * a.R, (group + 1) * PT_SUM);
    for (int row = group * PT_SUM + w; row < end; row += 8) {
        const int tile = row / a.tile_rows, y = row - tile * a.tile_rows, tok = row / a.R, head = kvh * a.R + row - tok * a.R, first = items + (tiles - 1 - tile) * n;      // tile by tile from the last one on
        auto place = [&](int x) { return ((size_t)(first + x) * a.heads + blockIdx.y) * a.tile_rows + y; };
        float m = -INFINITY, l = 0.0f;
        for (int x = lane; x < n; x += 32) m = fmaxf(m, a.ml[place(x)].x);
        m = warp_max(m);
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int x0 = 0; x0 < n; x0 += 32) {
            const float2 z = x0 + lane < n ? a.ml[place(x0 + lane)] : make_float2(-INFINITY, 0.0f);
            const float f = z.x == -INFINITY ? (z.y == 0.0f ? 0.0f : 1.0f) : exp2f(z.x - m);
            l = fmaf(f, z.y, l);
#pragma unroll 4
            for (int x = x0; x < min(n, x0 + 32); x++) {
                const float by = __shfl_sync(0xffffffffu, f, x - x0);
                if (col < a.dv) {
                    const float4 v = *(const float4*)(a.part + place(x) * a.dv + col);
                    o.x = fmaf(by, v.x, o.x); o.y = fmaf(by, v.y, o.y); o.z = fmaf(by, v.z, o.z); o.w = fmaf(by, v.w, o.w);
                }
            }
        }
        l = warp_sum(l);
        float f = 1.0f;
        if (a.sink) {
            const float sk = a.sink[head] * PT_LOG2E, m2 = fmaxf(m, sk);
            f = m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : exp2f(m - m2);
            l = f * l + (sk == -INFINITY ? 0.0f : exp2f(sk - m2 + PT_SHIFT));
        }
        if (col < a.dv) *(float4*)(a.out + ((int64_t)(s.first + tok) * a.H + head) * a.dv + col) = make_float4(o.x * f / l, o.y * f / l, o.z * f / l, o.w * f / l);
    }
}

template <int D, bool I8>
static cudaError_t pt_launch_few(cc_device* dev, const PtArgs& a, const PtDeal& deal, unsigned ctas) {
    constexpr int smem = PT_WARPS * 128 * D;
    cudaError_t e = cudaFuncSetAttribute(paged_few_kernel<D, I8>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = cc_launch_pdl(dev, paged_few_kernel<D, I8>, ctas, PT_THREADS, smem, a, deal);
    dev->launches++;
    return e;
}
// the runs of deal.ctas CTAs over all steps, and the segments that are in several of them (returned: how many; `rows` of the longest)
static int pt_deal(const cc_page_plan* plan, const PtArgs& a, int64_t steps, PtDeal& deal, PtCuts& cuts) {
    deal.run_lo = (int)(steps / deal.ctas); deal.run_more = (int)(steps % deal.ctas);
    int64_t before = 0, next = 0;                                  // steps in front of the sequence, and of run c
    int c = 0, n_cuts = 0;
    for (int seq = 0; seq < (int)plan->seqs.size() && c < deal.ctas; seq++) {
        const int n = pt_segments(plan->seqs[seq], a), all = n ? pt_steps(plan->seqs[seq], a) : 0;
        for (; c < deal.ctas && next < before + (int64_t)n * all; next += deal.run_lo + (c < deal.run_more ? 1 : 0), c++) {
            const int seg = (int)((next - before) / all), off = (int)((next - before) - (int64_t)seg * all);
            deal.at[c] = {seq, seg, off};
            if (off <= PT_BEGIN) continue;                         // the segment's keys are all this run's, or there are none of them in front
            auto& cut = cuts.at[n_cuts ? n_cuts - 1 : 0];
            if (n_cuts && cut.seq == seq && cut.seg == seg) { cut.n++; continue; }
            const auto& last = deal.at[c - 1];                     // the run in front begins with the segment, or within its first PT_BEGIN steps, or ends with it
            cuts.at[n_cuts++] = {seq, seg, 2 * (c - 1) + (last.seq == seq && last.seg == seg ? 0 : 1), c, 2};
        }
        before += (int64_t)n * all;
    }
    return n_cuts;
}
// Sequences of few rows, or of any where heads are too wide for tiles of 128.  All steps in equal runs, as many CTAs as the device holds at a time, so that none waits for a last wave and few
// begin anew.  (Slices of up to 1024 keys, a CTA each: 64 sequences of up to 4000 tokens, 32 heads on 8, 8-bit pages: 90 us, in runs 82; 16-bit pages 77 and 75.)
// Segments of up to PT_WHOLE steps: a CTA each, nothing to add up (64 sequences at 250 tokens 28 us, in runs 35; at 500 38 and 39, at 1000 57 and 52; 16 at 500 15 and 22, at 1000 32 and 25).
// Prompts of wide heads likewise, late rows first: their early rows see less than a run counts (1000 tokens, 16 heads of 256 on 4: 346 us, in runs 561)
#define PT_WHOLE 8
static int pt_run_few(cc_device* dev, const cc_page_plan* plan, PtArgs a, bool i8) {
    int64_t segments = 0, steps = 0;
    int most = 0;
    for (const PgSeq& s : plan->seqs) {
        const int n = pt_segments(s, a);
        if (!n) continue;
        const int all = pt_steps(s, a);
        segments += n;
        steps += (int64_t)n * all;
        most = std::max(most, all - PT_BEGIN);
    }
    if (!segments) return CC_OK;
    CC_REQUIRE(dev, segments < ((int64_t)1 << 31), "paged_attention: too many rows");
    const int d = std::max(a.dk, a.dv), per_sm = d <= 64 ? 4 : d <= 128 ? 3 : 1;
    const int64_t slots = std::min<int64_t>(PT_CTAS, (int64_t)per_sm * dev->sm_count);
    PtDeal deal;
    PtCuts cuts;
    deal.ctas = most <= PT_WHOLE || (a.rows_hi > PT_FEW && segments >= 8 * slots) ? 0 : (int)std::min<int64_t>(slots, (steps + PT_BEGIN + 1) / (PT_BEGIN + 2));
    const int n_cuts = deal.ctas ? pt_deal(plan, a, steps, deal, cuts) : 0;
    void* ws = nullptr; size_t cls = 0;
    if (n_cuts) {
        const size_t part = (size_t)2 * deal.ctas * 8 * a.dv * sizeof(float);
        const int rc = cc_pool_alloc(dev, part + (size_t)2 * deal.ctas * 8 * sizeof(float2), &ws, &cls);
        if (rc) return rc;
        a.part = (float*)ws; a.ml = (float2*)((uint8_t*)ws + part);
    }
    const unsigned ctas = deal.ctas ? (unsigned)deal.ctas : (unsigned)segments;
    cudaError_t e = i8 ? (d <= 64 ? pt_launch_few<64, true>(dev, a, deal, ctas) : d <= 128 ? pt_launch_few<128, true>(dev, a, deal, ctas) : pt_launch_few<256, true>(dev, a, deal, ctas))
                       : (d <= 64 ? pt_launch_few<64, false>(dev, a, deal, ctas) : d <= 128 ? pt_launch_few<128, false>(dev, a, deal, ctas) : pt_launch_few<256, false>(dev, a, deal, ctas));
    if (e == cudaSuccess && n_cuts) {
        e = cc_launch_pdl(dev, paged_join_kernel, dim3((unsigned)n_cuts, 8), 32 * PT_JOIN, 0, a, cuts);
        dev->launches++;
    }
    if (ws) cc_pool_free(dev, ws, cls);
    if (e != cudaSuccess) return cc_fail(dev, CC_ERR_CUDA, "paged_attention: %s", cudaGetErrorString(e));
    return CC_OK;
}
#include "paged_tile.cuh"

#define TI_WORKSPACE ((int64_t)256 << 20)     // bytes of images that a call has at a time, as long as those of one sequence and head are no more; and of sums of slices

// How long a call takes with slices of a.split keys, in cycles.  An item's start and end 18000, a step of 128 keys 3900; CTAs take items in turn, so that the SMs end half of the longest one apart;
// sums of slices are written and read at 3 TB/s (1600 bytes a cycle), 10000 cycles for the kernel that adds them up
static double pt_guess(const PgSeq* seqs, const PtArgs& a, int sms) {
    double all = 0.0, longest = 0.0, sums = 0.0, items = 0.0;
    for (int i = 0; i < a.n_seqs; i++) {
        const PgSeq& s = seqs[i];
        const int n = pt_splits(s, a);
        if (!n) continue;
        int from, to;
        pt_range(s, a, &from, &to);
        const double rows = (double)s.count * a.R, heads = std::ceil(rows / TI_ROWS) * a.G;
        all += heads * (18000.0 * n + 3900.0 / TI_KEYS * (std::max(to - from - 0.5 * s.count, 0.5 * TI_KEYS)));
        items += heads * n;
        longest = std::max(longest, 18000.0 + 3900.0 / TI_KEYS * std::min(pt_each(to - from, n), to - from));
        if (n > 1) sums += rows * a.G * (2 * n + 1) * a.dv * 4 / 1600.0;
    }
    return (items <= sms ? longest : std::max(longest, all / sms + 0.5 * longest)) + (sums > 0.0 ? sums + 10000.0 : 0.0);
}
// slices of a.split keys: the items of a head, and the groups of PT_SUM rows whose slices are to be added up
static void pt_count(const PgSeq* seqs, const PtArgs& a, int64_t* items, int64_t* split_rows) {
    *items = *split_rows = 0;
    for (int i = 0; i < a.n_seqs; i++) {
        const int n = pt_splits(seqs[i], a);
        *items += (int64_t)n * (((int64_t)seqs[i].count * a.R + a.tile_rows - 1) / a.tile_rows);
        if (n > 1) *split_rows += ((int64_t)seqs[i].count * a.R + PT_SUM - 1) / PT_SUM;
    }
}
// Sequences of many rows: of some lengths of slices the one that should take least time.  (As many as give every SM one, against this, 32 heads on 8: 4 sequences of 3000 to 6000 tokens
// with 16 to 128 new ones 120 us and 92, 8 of 3000 with 64 106 and 93, 16 of 500 to 3000 with 16 to 64 146 and 132; 256 tokens over 8000 149 and 148, where slices of 2560 take 130.)
// A row that is cut leaves its sums for each slice: those of a long prompt would be gigabytes, while it has rows enough for every SM without; so not beyond TI_WORKSPACE
static int pt_tiles(cc_device* dev, const PgSeq* seqs, PtArgs a, int64_t key_tiles, bool i8) {
    const size_t kb = (size_t)((a.dk + 63) / 64) * TI_BLOCK, vb = (size_t)((a.dv + 63) / 64) * TI_BLOCK, per_head = (size_t)key_tiles * (kb + vb + sizeof(TiInfo));
    const size_t per_row = (size_t)a.dv * sizeof(float) + sizeof(float2);
    int best = 0;
    double least = 0.0;
    int64_t items, split_rows;
    for (int split : {TI_WHOLE, 4096, 2560, 2048, 1536, 1024, 768, 512}) {
        a.split = split;
        pt_count(seqs, a, &items, &split_rows);
        if (split_rows && (double)items * a.G * a.tile_rows * per_row > (double)TI_WORKSPACE) continue;
        const double t = pt_guess(seqs, a, dev->sm_count);
        if (!best || t < 0.97 * least) { best = split; least = t; }
    }
    a.split = best;
    pt_count(seqs, a, &items, &split_rows);
    CC_REQUIRE(dev, items * a.G < ((int64_t)1 << 31) && split_rows < ((int64_t)1 << 31) && key_tiles < ((int64_t)1 << 31), "paged_attention: too many rows");
    a.heads = (int64_t)per_head * a.G <= TI_WORKSPACE ? a.G : (int)std::max<int64_t>(1, TI_WORKSPACE / (int64_t)per_head);
    const size_t part = split_rows ? (size_t)items * a.heads * a.tile_rows * a.dv * sizeof(float) : 0, ml = split_rows ? (size_t)items * a.heads * a.tile_rows * sizeof(float2) : 0;
    void* ws = nullptr; size_t cls = 0;
    const int rc = cc_pool_alloc(dev, part + ml + per_head * a.heads + 256, &ws, &cls);
    if (rc) return rc;
    a.k_image = (uint8_t*)ws; a.v_image = a.k_image + key_tiles * a.heads * kb;
    a.part = (float*)(a.v_image + key_tiles * a.heads * vb);
    a.ml = (float2*)((uint8_t*)a.part + part); a.info = (TiInfo*)((uint8_t*)a.ml + ml);
    const int all = a.heads;
    const bool cap = a.softcap > 0.0f;
    auto kernel = i8 ? (cap ? paged_tile_kernel<true, true> : paged_tile_kernel<true, false>) : (cap ? paged_tile_kernel<false, true> : paged_tile_kernel<false, false>);
    cudaError_t e = cudaSuccess;
    for (a.head0 = 0; a.head0 < a.G && e == cudaSuccess; a.head0 += all) {
        a.heads = std::min(all, a.G - a.head0);
        e = cc_launch_pdl(dev, i8 ? paged_unpack_kernel<true> : paged_unpack_kernel<false>, dim3((unsigned)key_tiles, (unsigned)a.heads), TU_THREADS, 0, a);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TI_SMEM);
        if (e == cudaSuccess) e = cc_launch_pdl(dev, kernel, (unsigned)(items * a.heads), TI_THREADS, TI_SMEM, a, dev->err_dev, dev->err_host);
        dev->launches += 2;
        if (e == cudaSuccess && split_rows) {
            e = cc_launch_pdl(dev, paged_sum_kernel, dim3((unsigned)split_rows, (unsigned)a.heads), 256, 0, a);
            dev->launches++;
        }
    }
    if (ws) cc_pool_free(dev, ws, cls);
    if (e != cudaSuccess) return cc_fail(dev, CC_ERR_CUDA, "paged_attention: %s", cudaGetErrorString(e));
    return CC_OK;
}
// as many sequences at a time as have their images of one head in TI_WORKSPACE
static int pt_run_tiles(cc_device* dev, const cc_page_plan* plan, PtArgs a, bool i8) {
    const int64_t per_tile = (int64_t)((a.dk + 63) / 64 + (a.dv + 63) / 64) * TI_BLOCK + (int64_t)sizeof(TiInfo);
    for (int first = 0, end; first < plan->n_seqs; first = end) {
        int64_t key_tiles = 0;
        for (end = first; end < plan->n_seqs; end++) {
            const int n = ti_key_tiles(plan->seqs[end], a);
            if (key_tiles && (key_tiles + n) * per_tile > TI_WORKSPACE) break;
            key_tiles += n;
        }
        a.seqs = plan->d_seqs + first; a.n_seqs = end - first; a.table = plan->d_table + (int64_t)first * a.table_cols;
        const int rc = key_tiles ? pt_tiles(dev, plan->seqs.data() + first, a, key_tiles, i8) : CC_OK;
        if (rc) return rc;
    }
    return CC_OK;
}

extern "C" CC_API int cc_paged_attention(cc_device* dev, const cc_page_plan* plan, const cc_paged_cache* cache, const cc_view* q, int32_t H, float scale, int32_t window,
                                         float softcap, const cc_view* sink, cc_buf** out) {
    PG_ENTER(dev, plan, "paged_attention");
    if (!out) return cc_fail(dev, CC_ERR_ARG, "paged_attention: out is NULL");
    *out = nullptr;
    PgCache c;
    int rc = pg_check_cache(dev, plan, cache, "paged_attention", &c);
    if (rc) return rc;
    PG_ROWS(dev, q, "paged_attention q");
    CC_REQUIRE(dev, view_contiguous(q), "paged_attention q: not contiguous");
    const int64_t T = plan->tokens;
    CC_REQUIRE(dev, H > 0 && H <= 8192 && H % c.G == 0, "paged_attention: %d query heads over %d", H, c.G);
    CC_REQUIRE(dev, q->shape[0] == T && q->shape[1] == (int64_t)H * c.dk, "paged_attention: q is not [%lld, %d * %d]", (long long)T, H, c.dk);
    if (sink) {
        if (!view_ok(sink)) return cc_fail(dev, CC_ERR_ARG, "paged_attention: bad view of sink");
        CC_REQUIRE(dev, view_in_bounds(sink) && view_contiguous(sink) && view_len(sink) == H && sink->buf->dtype == CC_F32 && sink->buf->dev == dev,
                   "paged_attention: sink is not contiguous F32 [%d] of this device", H);
    }
    CC_REQUIRE(dev, T * H < ((int64_t)1 << 31), "paged_attention: %lld tokens of %d heads", (long long)T, H);
    cc_buf* o = nullptr;
    rc = cc_new_activation(dev, T * H * c.dv, CC_F32, false, &o);
    if (rc) return rc;
    if (T > 0) {
        PtArgs a{};
        a.seqs = plan->d_seqs; a.table = plan->d_table; a.k = c.k; a.v = c.v; a.ks = c.ks; a.vs = c.vs; a.ko = c.ko; a.vo = c.vo;
        a.q = (const float*)q->buf->plane[0]; a.sink = sink ? (const float*)sink->buf->plane[0] : nullptr; a.out = (float*)o->base;
        a.scale = scale; a.softcap = softcap; a.window = window > 0 ? window : 0;
        a.n_seqs = plan->n_seqs; a.table_cols = plan->table_cols; a.page = plan->page; a.shift = plan->shift;
        a.H = H; a.G = c.G; a.R = H / c.G; a.dk = c.dk; a.dv = c.dv;
        // up to PT_FEW rows in tiles of 8, more in tiles of 128 where a head's numbers have room there
        a.rows_lo = 1; a.rows_hi = c.dk <= TI_D && c.dv <= TI_D ? PT_FEW : 0x7fffffff; a.tile_rows = 8; a.align = 16;
        rc = pt_run_few(dev, plan, a, c.i8);
        if (!rc && a.rows_hi == PT_FEW) {
            a.rows_lo = PT_FEW + 1; a.rows_hi = 0x7fffffff; a.tile_rows = TI_ROWS; a.align = TI_KEYS;
            rc = pt_run_tiles(dev, plan, a, c.i8);
        }
    }
    if (rc) { cc_tensor_release(o); return rc; }
    *out = o;
    return CC_OK;
}
