// paged_tile.cuh -- attention of many rows over pages (prompts, drafts of many heads), on tcgen05.mma.  Included by paged_attn.cu behind its few-row kernel.
//
// paged_unpack_kernel lays out the visible keys and values once for all rows: per 128 keys and head an image of each operand as f16 (codes and 16-bit numbers are exact),
// in the order of the 128-byte swizzle, that a bulk copy brings into shared memory as it is, beside the factors of its pages.  (Converted by warps of the kernel below
// for each of its tiles instead, portions of three prompts took 285 us: 2700 of 8000 instructions of a step, and an instruction cache that did not hold all roles.)
//
// A tile is 128 rows (a row: a query of one head; the heads of a key head side by side) x the keys they see, 128 at a time:
//   S = Q_h K^T + Q_l K^T                                                                         2 x 128 x 128 x dk products
//   P = exp2(S f - largest) as f16 h and l, written over S in TMEM, the first operand of
//   O = P_h V + P_l V         in an accumulator of its own, added to 32-bit registers afterwards: the tensor core cuts its sums off at 24 bits, a chain over
//                             thousands of keys would drift (1e-5 of a result after 2000 keys of one sign)
// TMEM holds S twice, O, Q_h and Q_l (512 columns), shared memory two stages of K and V (128 KB): while 8 warps make the weights of one step, the tensor core computes the
// scores of the next and the sums of the one before.  With Q in shared memory a step's products read 192 KB there and took 3100 cycles instead of 2050.
// A row's 128 scores lie with two threads, a half each, which exchange their largest score once a step.  Warps 0-7 weights and sums, 8 the copies, 9 the products, 10 what stands beside the images.
// Portions of three prompts (3000 rows of 32 heads on 8, 8-bit pages): 12 us of images and 208 of tiles, 326 TFLOP/s of the four products' 68 GFLOP, of which the h and l of
// queries and weights make two.  A step takes 3900 cycles, its products 2050 of them, the weights' instructions 1500; the rest is the way of a step's scores through one group of warps
// in turn (wait, read, largest, meet, weights, store).  Sums of four steps left to the tensor core, fewer reads of O, took 3 % more.
// Every wait is bounded (sg_wait); where one ran out all roles run to their ends without waiting (the barrier of warps 0-7 included) and the host reports it.
#pragma once
#include <stddef.h>

#include "split_gemm.cuh"

#define TI_ROWS 128
#define TI_KEYS 128
#define TI_SPLIT 2                            // threads of a row: half of a step's keys and of the value columns each
#define TI_SOFT (TI_ROWS * TI_SPLIT)
#define TI_SOFT_WARPS (TI_SOFT / 32)
#define TI_THREADS (TI_SOFT + 128)
// 384 threads of 168 registers at launch are 256 of 216 and 128 of 72 afterwards.  A step's numbers must not spill: shared memory leaves next to no L1, and with 80 numbers
// a thread spilled (four threads a row, 96 registers) a step took twice as long.  Two of them do
#define TI_REGS 168
#define TI_REGS_SOFT 216
#define TI_REGS_REST 72
static_assert(TI_SOFT * TI_REGS_SOFT + (TI_THREADS - TI_SOFT) * TI_REGS_REST <= TI_THREADS * TI_REGS, "more registers than the block was launched with");
#define TI_XC (TI_KEYS / TI_SPLIT)
#define TI_OC (TI_D / TI_SPLIT)
#define TI_WHOLE 0x7fffff00                   // keys of a slice: all
#define TI_D 128                              // largest dk and dv
#define TI_STEPS 32                           // whose TiInfo a CTA holds at a time

// what stands beside the images of 128 keys of a head
struct __align__(16) TiInfo {
    float kf[TI_KEYS / 16], vf[TI_KEYS / 16]; // factors of 16 keys each (0 where there are none)
    float lv[TI_KEYS / 16];                   // 8-bit pages: how large the values of 16 keys are, as a score: log2 of their block's largest number / 127, down to a whole number (-inf: zeros)
    int wild;                                 // values that are not finite are zeros in the image
    unsigned bad[TI_KEYS / 32];               // keys whose factors or numbers are not finite (they count as 0): NaN for the rows that see one
    int pad[3];
};
#define TI_WORDS ((int)(sizeof(TiInfo) / 4))
static_assert(TI_WORDS == 32, "a word for each lane");
__device__ __forceinline__ bool ti_odd(int word) { return word >= (int)(offsetof(TiInfo, wild) / 4) && word < (int)(offsetof(TiInfo, pad) / 4); }      // wild, or bad
struct TiShared {
    unsigned long long k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full, drained;
    unsigned tmem_base;
    int fail;
    int odd;                                  // some TiInfo says wild or bad
    const TiInfo* first;                      // of the first step
    TiInfo info[TI_STEPS];
    float2 top[2][TI_SPLIT][TI_ROWS];         // of a step: largest score, and largest sum of a score and its block's lv
    float sum[TI_SPLIT][TI_ROWS], inv[TI_ROWS];
};
#define TI_OPERAND (TI_KEYS * TI_D * 2)       // bytes of a tile of f16: two blocks of 64 columns, rows of 128 bytes under the 128-byte swizzle
#define TI_SMEM (6 * TI_OPERAND + 1024)
#define TI_UP 30                              // the smallest numbers of f16, 2^-24, reach 2^6
#define TI_TOP 512.0f                         // the largest weight, 2^PT_SHIFT
#define TI_SFU 14                             // of 16 weights those that the special function unit makes: 214 us for the portions of three prompts; 10 of them 222, 12 216, all 217
#define TI_O 256                              // TMEM columns: S and P at 0 and 128
#define TI_Q 384
#define TI_BLOCK (TI_OPERAND / 2)             // 64 columns of an operand; an image is as many as d has

__device__ __forceinline__ unsigned ti_at(int row, int chunk) { return (unsigned)((chunk >> 3) * (TI_OPERAND / 2) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4)); }
// B whose rows are the sum's index and whose columns (64 of them in 128 bytes) are the result's: blocks of 64 columns are TI_OPERAND / 2 apart, groups of 8 rows 1024 bytes
__device__ __forceinline__ uint64_t ti_desc_mn(unsigned addr) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)(TI_OPERAND / 2 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ void ti_umma_ts(unsigned d, unsigned a, uint64_t b, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void ti_store8(unsigned addr, const unsigned (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]),
                 "r"(v[7]) : "memory");
}
// sg_wait for warps that have nothing else to do for long: the hardware holds them for up to 2 us a look, so that they leave the issue slots to others
__device__ __forceinline__ bool ti_wait(unsigned bar, unsigned parity, int* fail) {
    unsigned done = 0;
    for (unsigned it = 0; it < (1u << 21); it++) {
        asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\nselp.u32 %0, 1, 0, p;\n}\n" : "=r"(done) : "r"(bar), "r"(parity), "r"(2000u) : "memory");
        if (done) return true;
        if (*(volatile int*)fail) return false;
    }
    *(volatile int*)fail = 1;
    return false;
}
__device__ __forceinline__ bool ti_wait_warp(unsigned bar, unsigned parity, int* fail) { return __all_sync(0xffffffffu, ti_wait(bar, parity, fail)); }
// pairs of 32-bit numbers in one instruction
typedef unsigned long long ti_f2;
__device__ __forceinline__ ti_f2 ti_fma2(ti_f2 a, ti_f2 b, ti_f2 c);
__device__ __forceinline__ ti_f2 ti_add2(ti_f2 a, ti_f2 b);
__device__ __forceinline__ ti_f2 ti_two(float x, float y) {
    ti_f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 ti_one(ti_f2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ ti_f2 ti_fma2(ti_f2 a, ti_f2 b, ti_f2 c) {
    ti_f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ ti_f2 ti_mul2(ti_f2 a, ti_f2 b) {
    ti_f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ ti_f2 ti_add2(ti_f2 a, ti_f2 b) {
    ti_f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// 2^x of a pair by multiply-adds: the special function unit makes 4 results a cycle and scheduler, which alone would take half of a step.  x = n + r with |r| <= 1/2 by way
// of a number whose last place is 1; 2^r by its series up to r^6 (the first term left out is 2^-23 at |r| = 1/2; with the roundings the result is off by up to 2^-22 of itself, as the special function
// unit's is); n goes into the exponent.  What is below -126, a hidden key's -inf and NaN count as -126
__device__ __forceinline__ ti_f2 ti_exp2_pair(float2 x) {
    const ti_f2 big = ti_two(12582912.0f, 12582912.0f), minus = ti_two(-1.0f, -1.0f);
    const ti_f2 v = ti_two(fmaxf(x.x, -126.0f), fmaxf(x.y, -126.0f)), t = ti_add2(v, big), n = ti_add2(t, ti_two(-12582912.0f, -12582912.0f)), r = ti_fma2(n, minus, v);
    ti_f2 p = ti_two(1.5403530e-4f, 1.5403530e-4f);                  // (ln 2)^i / i!, i = 6 .. 0
    p = ti_fma2(p, r, ti_two(1.3333558e-3f, 1.3333558e-3f));
    p = ti_fma2(p, r, ti_two(9.6181291e-3f, 9.6181291e-3f));
    p = ti_fma2(p, r, ti_two(5.5504109e-2f, 5.5504109e-2f));
    p = ti_fma2(p, r, ti_two(2.4022651e-1f, 2.4022651e-1f));
    p = ti_fma2(p, r, ti_two(6.9314718e-1f, 6.9314718e-1f));
    p = ti_fma2(p, r, ti_two(1.0f, 1.0f));
    const float2 q = ti_one(p), m = ti_one(t);
    return ti_two(__uint_as_float(__float_as_uint(q.x) + (__float_as_uint(m.x) << 23)), __uint_as_float(__float_as_uint(q.y) + (__float_as_uint(m.y) << 23)));
}
__device__ __forceinline__ float ti_max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ void ti_step_sync() { asm volatile("bar.sync 2, %0;" ::"n"(TI_SOFT + 32) : "memory"); }
__device__ __forceinline__ void ti_soft_sync() { asm volatile("bar.sync 1, %0;" ::"n"(TI_SOFT) : "memory"); }

// images of the sequences with a tile of 128 rows: their tiles of keys count from the first that a new token sees, sequence after sequence
__host__ __device__ __forceinline__ int ti_key_tiles(const PgSeq& s, const PtArgs& a) {
    const int64_t rows = (int64_t)s.count * a.R;
    if (rows < a.rows_lo || rows > a.rows_hi) return 0;
    int from, to;
    pt_range(s, a, &from, &to);
    return (to - from + TI_KEYS - 1) / TI_KEYS;
}
#define TU_THREADS 256
// grid (tiles of keys, heads of this call)
template <bool I8>
__global__ void __launch_bounds__(TU_THREADS) paged_unpack_kernel(const PtArgs a) {
    __shared__ int pages[TI_KEYS / 16];
    __shared__ float up[TI_KEYS / 16];                         // powers of two that the open block's values are multiplied by, 16 keys each
    __shared__ TiInfo info;
    const int tid = threadIdx.x, kvh = a.head0 + blockIdx.y;
    pdl_enter();
    int kt;
    const int seq = pt_find(a, blockIdx.x, [&](const PgSeq& s) { return ti_key_tiles(s, a); }, &kt);
    if (seq < 0) return;
    const PgSeq s = a.seqs[seq];
    int from, to;
    pt_range(s, a, &from, &to);
    const int key0 = from + kt * TI_KEYS, opens = I8 ? to >> a.shift << a.shift : 0, open = 2 * s.slot + ((to >> a.shift) & 1);
    // The open block's values are made as large as codes are, by a power of two that its 16 keys' first one sets (any query that sees one of them sees that, but for windows) as far as all
    // of them stay in range: exactly, for it only multiplies.  Their factor is the inverse.  A warp 16 keys, two lanes a key
    if (const int group = tid >> 5, key = key0 + (tid >> 1); I8 && key0 + group * 16 >= opens && key0 + group * 16 < to) {
        unsigned m = 0;
        if (key < to) {
            const uint4* p = (const uint4*)(a.vo + (((size_t)open * a.G + kvh) * a.page + (key & (a.page - 1))) * a.dv) + (tid & 1);
#pragma unroll 4
            for (int i = 0; i < a.dv / 16; i++) {
                const uint4 x = __ldg(p + 2 * i);
                m = __vmaxu2(m, __vmaxu2(__vmaxu2(x.x & 0x7fff7fffu & ~pt_wild(x.x), x.y & 0x7fff7fffu & ~pt_wild(x.y)),
                                         __vmaxu2(x.z & 0x7fff7fffu & ~pt_wild(x.z), x.w & 0x7fff7fffu & ~pt_wild(x.w))));
            }
            m = max(m & 0xffffu, m >> 16);
        }
        const unsigned most = __reduce_max_sync(0xffffffffu, m), mine = max(__shfl_sync(0xffffffffu, m, 0), __shfl_sync(0xffffffffu, m, 1)), first = mine ? mine : most;
        auto log2_of = [](unsigned h) { return (__float_as_int(__half2float(__ushort_as_half((unsigned short)h))) >> 23) - 127; };
        const int by = most ? max(0, min(TI_UP, min(6 - log2_of(first), 14 - log2_of(most)))) : 0;
        if ((tid & 31) == 0) {
            up[group] = pt_pow2((float)by); info.vf[group] = pt_pow2((float)-by);
            info.lv[group] = most ? (float)max(log2_of(first) - 6, -by) : -INFINITY;
        }
    }
    if (tid < 32) {
        float kf = 1.0f, vf = 1.0f, lv = 0.0f;
        const int key = key0 + (tid & 7) * 16;
        int page = -1;                                        // nothing there, or the open block
        if (key < to && (!I8 || key < opens)) {
            page = a.table[(int64_t)seq * a.table_cols + (key >> a.shift)];
            if (I8) { kf = a.ks[(int64_t)page * a.G + kvh]; vf = a.vs[(int64_t)page * a.G + kvh]; }
        }
        const bool bad = !(vf >= 0.0f && vf < INFINITY && kf >= 0.0f && kf < INFINITY);
        if (bad || key >= to) kf = vf = 0.0f;
        lv = pt_log2(vf);
        const unsigned nan = __ballot_sync(0xffffffffu, bad) >> 2 * (tid & 3);      // the lanes' groups repeat after 8
        if (tid < TI_KEYS / 16) {
            pages[tid] = page; info.kf[tid] = kf;
            if (!I8 || key < opens || key >= to) { info.vf[tid] = vf; info.lv[tid] = lv; }
        }
        if (tid < TI_KEYS / 32) info.bad[tid] = (nan & 1u ? 0xffffu : 0u) | (nan & 2u ? 0xffff0000u : 0u);
    }
    __syncthreads();
    const size_t at = (size_t)blockIdx.x * a.heads + blockIdx.y;
    bool wild = false;
#pragma unroll
    for (int v = 0; v < 2; v++) {
        const int d = v ? a.dv : a.dk;
        uint8_t* image = (v ? a.v_image : a.k_image) + at * ((d + 63) / 64) * TI_BLOCK;
        // a lane takes 16 numbers of a row: two chunks of its image
#pragma unroll 4
        for (int e = tid; e < TI_KEYS * (d / 16); e += TU_THREADS) {
            const int r = e / (d / 16), piece = e - r * (d / 16), key = key0 + r, page = pages[r >> 4], row = key & (a.page - 1);
            uint4 x = make_uint4(0, 0, 0, 0), y = x;
            if (I8 && page >= 0) {
                const uint4 c = __ldg((const uint4*)((v ? a.v : a.k) + (((size_t)page * a.G + kvh) * a.page + row) * d) + piece);
                const unsigned u0 = c.x ^ 0x80808080u, u1 = c.y ^ 0x80808080u, u2 = c.z ^ 0x80808080u, u3 = c.w ^ 0x80808080u;
                x = make_uint4(pt_half2(u0, 0x4140), pt_half2(u0, 0x4342), pt_half2(u1, 0x4140), pt_half2(u1, 0x4342));
                y = make_uint4(pt_half2(u2, 0x4140), pt_half2(u2, 0x4342), pt_half2(u3, 0x4140), pt_half2(u3, 0x4342));
            } else if (key < to) {
                const __half* p = I8 ? (v ? a.vo : a.ko) + (((size_t)open * a.G + kvh) * a.page + row) * d : (const __half*)(v ? a.v : a.k) + (((size_t)page * a.G + kvh) * a.page + row) * d;
                x = __ldg((const uint4*)p + 2 * piece); y = __ldg((const uint4*)p + 2 * piece + 1);
                unsigned* u[8] = {&x.x, &x.y, &x.z, &x.w, &y.x, &y.y, &y.z, &y.w}, any = 0;
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const unsigned w = pt_wild(*u[i]);
                    any |= w;
                    *u[i] &= ~w;
                }
                if (any && v) wild = true;
                if (any && !v) atomicOr(&info.bad[r >> 5], 1u << (r & 31));
                if (I8 && v) {                                 // (2^15 at a time: f16 ends there)
                    const float by = up[r >> 4];
                    const __half2 f = __float2half2_rn(fminf(by, 32768.0f)), g = __float2half2_rn(fmaxf(by / 32768.0f, 1.0f));
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const __half2 z = __hmul2(__hmul2(*(const __half2*)u[i], f), g);
                        *u[i] = *(const unsigned*)&z;
                    }
                }
            }
            *(uint4*)(image + ti_at(r, 2 * piece)) = x;
            *(uint4*)(image + ti_at(r, 2 * piece + 1)) = y;
        }
    }
    wild = __syncthreads_or(wild);
    if (tid == 0) info.wild = wild;
    __syncthreads();
    if (tid < (int)(sizeof(TiInfo) / 4)) ((int*)(a.info + at))[tid] = ((const int*)&info)[tid];
}

template <bool I8, bool CAP>
__global__ void __launch_bounds__(TI_THREADS, 1) paged_tile_kernel(const __grid_constant__ PtArgs a, unsigned* err_dev, unsigned* err_host) {
    extern __shared__ __align__(1024) uint8_t ti_raw[];
    __shared__ TiShared sh;
    uint8_t* qs = (uint8_t*)(((uintptr_t)ti_raw + 1023) & ~(uintptr_t)1023);      // 64 KB on the way: queries into TMEM, results out
    uint8_t *ks = qs + 2 * TI_OPERAND, *vs = ks + 2 * TI_OPERAND;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, item = (int)(blockIdx.x / (unsigned)a.heads), head_at = (int)(blockIdx.x - (unsigned)item * a.heads), kvh = a.head0 + head_at;      // heads fastest: the items that see most come first
    if (tid == 0) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            pg_mbar_init(pg_smem(&sh.k_full[i]), 1); pg_mbar_init(pg_smem(&sh.v_full[i]), 1); pg_mbar_init(pg_smem(&sh.k_empty[i]), 1); pg_mbar_init(pg_smem(&sh.v_empty[i]), 1);
            pg_mbar_init(pg_smem(&sh.s_full[i]), 1); pg_mbar_init(pg_smem(&sh.p_full[i]), TI_SOFT_WARPS);         }
        pg_mbar_init(pg_smem(&sh.o_full), 1);
        pg_mbar_init(pg_smem(&sh.drained), 1);
        sh.fail = 0;
        sh.odd = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == (TI_SOFT_WARPS + 1)) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(pg_smem(&sh.tmem_base)), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pdl_enter();
    pg_fence_before();
    __syncthreads();
    pg_fence_after();
    const unsigned tmem = sh.tmem_base;
    int rest;
    const int seq = pt_find(a, item, [&](const PgSeq& s) { return pt_splits(s, a) * (int)(((int64_t)s.count * a.R + TI_ROWS - 1) / TI_ROWS); }, &rest);
    const PgSeq s = a.seqs[max(seq, 0)];                              // (the grid has as many CTAs as there are items)
    const int rows = s.count * a.R, tiles = (rows + TI_ROWS - 1) / TI_ROWS, n_split = pt_splits(s, a), tile = tiles - 1 - rest / n_split, split = rest % n_split;      // late rows, which see most, first
    int from, to;
    pt_range(s, a, &from, &to);
    const int row0 = tile * TI_ROWS, n_rows = min(TI_ROWS, rows - row0), pos_first = s.pos0 + row0 / a.R, pos_last = s.pos0 + (row0 + n_rows - 1) / a.R;
    const int each = pt_each(to - from, n_split), k0 = from + split * each, k1 = min(min(to, k0 + each), pos_last + 1);
    const int lo = a.window > 0 ? max(k0, (pos_first - a.window + 1) & ~(TI_KEYS - 1)) : k0, steps = k1 > lo ? (k1 - lo + TI_KEYS - 1) / TI_KEYS : 0;
    const int opens = I8 ? to >> a.shift << a.shift : 0;
    // the images of the first step, and what stands beside those of the first TI_STEPS
    int before = 0;
    for (int x = lane; x < seq; x += 32) before += ti_key_tiles(a.seqs[x], a);
    const size_t image = (size_t)(warp_sum_i(before) + (lo - from) / TI_KEYS) * a.heads + head_at;
    if (tid == 0) sh.first = a.info + image;
    for (int i = tid; i < min(steps, TI_STEPS) * TI_WORDS; i += TI_THREADS) {
        const int x = ((const int*)(a.info + image + (size_t)(i / TI_WORDS) * a.heads))[i % TI_WORDS];
        ((int*)sh.info)[i] = x;
        if (x && ti_odd(i % TI_WORDS)) sh.odd = 1;
    }
    // the queries as h and l, near 2^14
    const int row = (warp & 3) * 32 + lane, part = warp >> 2;         // of weights and sums: TMEM lane, part of the columns
    const int tok = (row0 + row) / a.R, head = kvh * a.R + (row0 + row) - tok * a.R;
    const bool in = warp < TI_SOFT_WARPS && row < n_rows;
    const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
    const unsigned k_bytes = (unsigned)((a.dk + 63) / 64) * TI_BLOCK, v_bytes = (unsigned)((a.dv + 63) / 64) * TI_BLOCK;
    auto copy = [&](uint8_t* to_smem, const uint8_t* src, unsigned bytes, unsigned bar) {
        pg_mbar_expect_tx(bar, bytes);
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(pg_smem(to_smem)), "l"(src), "r"(bytes), "r"(bar) : "memory");
    };
    auto copy_k = [&](int k) { copy(ks + (size_t)(k & 1) * TI_OPERAND, a.k_image + (image + (size_t)k * a.heads) * k_bytes, k_bytes, pg_smem(&sh.k_full[k & 1])); };
    auto copy_v = [&](int k) { copy(vs + (size_t)(k & 1) * TI_OPERAND, a.v_image + (image + (size_t)k * a.heads) * v_bytes, v_bytes, pg_smem(&sh.v_full[k & 1])); };
    if (warp == TI_SOFT_WARPS && lane == 0)                           // the first images come while the queries are cut
        for (int k = 0; k < min(steps, 2); k++) { copy_k(k); copy_v(k); }
    if (warp < TI_SOFT_WARPS) {
        // a warp reads 16 rows, eight at a time; staged by rows of 512 bytes (h, then l; chunk j of 16 bytes at j ^ row % 8), then every thread stores its row's half to TMEM
#pragma unroll 1
        for (int r0 = warp * 16; r0 < warp * 16 + 16; r0 += 8) {
            float4 v[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int r = r0 + i, tk = (row0 + r) / a.R, hd = kvh * a.R + (row0 + r) - tk * a.R;
                v[i] = r < n_rows && lane * 4 < a.dk ? __ldg((const float4*)(a.q + ((int64_t)(s.first + tk) * a.H + hd) * a.dk) + lane) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const int r = r0 + i;
                // as bits, so that NaN is the largest of all
                const unsigned top = __reduce_max_sync(0xffffffffu, max(max(__float_as_uint(v[i].x) & 0x7fffffffu, __float_as_uint(v[i].y) & 0x7fffffffu),
                                                                        max(__float_as_uint(v[i].z) & 0x7fffffffu, __float_as_uint(v[i].w) & 0x7fffffffu)));
                // 2^(14 - e) for a largest number in [2^(e - 1), 2^e); zeros, subnormal and wild ones as they are
                int ex = (int)(top >> 23) - 126;
                if (top < 0x00800000u || top >= 0x7f800000u) ex = 14;
                ex = max(ex, -100);
                const float f = copysignf(__uint_as_float((unsigned)(14 - ex + 127) << 23), a.scale);      // (so that a larger sum is a larger score)
                uint2 h, l;
                pt_cut(v[i].x * f, v[i].y * f, h.x, l.x); pt_cut(v[i].z * f, v[i].w * f, h.y, l.y);
                uint8_t* at = qs + r * 512 + (((lane >> 1) ^ (r & 7)) << 4) + (lane & 1) * 8;
                *(uint2*)at = h; *(uint2*)(at + 256) = l;
                if (lane == 0) sh.inv[r] = top >= 0x7f800000u ? NAN : __uint_as_float((unsigned)(ex - 14 + 127) << 23);
            }
        }
        ti_soft_sync();
#pragma unroll 1
        for (int x = 0; x < 2; x++)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const uint4 u = *(const uint4*)(qs + row * 512 + x * 256 + (((part * 8 + j) ^ (row & 7)) << 4)), w = *(const uint4*)(qs + row * 512 + x * 256 + (((part * 8 + j + 1) ^ (row & 7)) << 4));
                const unsigned words[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
                ti_store8(tmem + lanes + TI_Q + x * 64 + part * 32 + j * 4, words);
            }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    }
    pg_fence_before();
    __syncthreads();
    pg_fence_after();

    if (warp >= TI_SOFT_WARPS) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TI_REGS_REST));
        if (warp == TI_SOFT_WARPS + 1) {
        // ===== products: one thread =====
        if (lane == 0) {
            const unsigned idesc_s = pg_instr_desc(128, TI_KEYS), idesc_o = pg_instr_desc(128, a.dv) | 1u << 16;
            bool ok = true;
            auto scores = [&](int k) {
                const unsigned slot = k & 1, at = pg_smem(ks + (size_t)slot * TI_OPERAND);
                if (!(ok = ti_wait(pg_smem(&sh.k_full[slot]), (k >> 1) & 1u, &sh.fail))) return;
                pg_fence_after();
                for (int x = 0; x < 2; x++)
                    for (int kk = 0; kk < a.dk / 16; kk++)
                        ti_umma_ts(tmem + slot * 128, tmem + TI_Q + x * 64 + kk * 8, pg_smem_desc(at + (unsigned)((kk >> 2) * TI_BLOCK + (kk & 3) * 32)), idesc_s, x > 0 || kk > 0);
                pg_umma_commit(pg_smem(&sh.s_full[slot]));
                pg_umma_commit(pg_smem(&sh.k_empty[slot]));
            };
            if (steps > 0) scores(0);
            for (int k = 0; k < steps && ok; k++) {
                const unsigned slot = k & 1, ph = (k >> 1) & 1u;
                if (k + 1 < steps) scores(k + 1);
                if (!ok || !(ok = ti_wait(pg_smem(&sh.p_full[slot]), ph, &sh.fail) && ti_wait(pg_smem(&sh.v_full[slot]), ph, &sh.fail))) break;
                pg_fence_after();
                const unsigned at = pg_smem(vs + (size_t)slot * TI_OPERAND);
                for (int x = 0; x < 2; x++)
                    for (int kk = 0; kk < TI_KEYS / 16; kk++)
                        ti_umma_ts(tmem + TI_O, tmem + slot * 128 + x * 64 + kk * 8, ti_desc_mn(at + kk * 2048), idesc_o, x > 0 || kk > 0);
                pg_umma_commit(pg_smem(&sh.o_full));
                pg_umma_commit(pg_smem(&sh.v_empty[slot]));
            }
            int never = 0;                                            // nothing of this CTA is in flight when its TMEM is given back
            pg_umma_commit(pg_smem(&sh.drained));
            ti_wait(pg_smem(&sh.drained), 0, &never);
        }
        __syncwarp();
        } else if (warp == TI_SOFT_WARPS) {
        // ===== copies of the images: one thread =====
        if (lane == 0) {
            int k = min(steps, 2), v = k;                             // copies begun
            for (; k < steps; k++) {
                const unsigned slot = k & 1, ph = ((k >> 1) & 1u) ^ 1u;
                if (!ti_wait(pg_smem(&sh.k_empty[slot]), ph, &sh.fail)) break;
                copy_k(k);
                if (!ti_wait(pg_smem(&sh.v_empty[slot]), ph, &sh.fail)) { k++; break; }
                copy_v(k);
                v++;
            }
            int never = 0;                                            // no copy is under way when the CTA ends
            for (int i = max(0, k - 2); i < k; i++) ti_wait(pg_smem(&sh.k_full[i & 1]), (i >> 1) & 1u, &never);
            for (int i = max(0, v - 2); i < v; i++) ti_wait(pg_smem(&sh.v_full[i & 1]), (i >> 1) & 1u, &never);
        }
        __syncwarp();
        } else if (warp == TI_SOFT_WARPS + 2) {
        // ===== what stands beside the images: the place of the step before goes to the one TI_STEPS behind it =====
            for (int k = 0; k < steps; k++) {
                ti_step_sync();                                       // the weights are through with step k - 1
                const int next = k - 1 + TI_STEPS;
                if (k == 0 || next >= steps) continue;
                const int x = ((const int*)(sh.first + (size_t)next * a.heads))[lane];
                ((int*)(sh.info + next % TI_STEPS))[lane] = x;
                if (x && ti_odd(lane)) sh.odd = 1;
            }
        }
    } else {
        // ===== weights and sums =====
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TI_REGS_SOFT));
        const int width = (a.dv + 16 * TI_SPLIT - 1) / (16 * TI_SPLIT) * 16, c_first = part * width, cols = max(0, min(width, a.dv - c_first));      // this thread's columns of O
        const int pos = in ? s.pos0 + tok : -1, key_lo = a.window > 0 ? pos - a.window + 1 : 0, key_hi = min(pos, k1 - 1);      // the last step may reach into the next slice
        const float f0 = sh.inv[row] * fabsf(a.scale) * (CAP ? 1.0f : PT_LOG2E);
        ti_f2 acc[TI_OC / 2];
        float m = -INFINITY, l = 0.0f, alpha_prev = 0.0f, unit_prev = 0.0f;
#pragma unroll
        for (int i = 0; i < TI_OC / 2; i++) acc[i] = 0ull;
        bool ok = true;
        auto add = [&](int k) {                                       // the sums of step k
            if (!(ok = ok && ti_wait_warp(pg_smem(&sh.o_full), k & 1, &sh.fail))) return;
            pg_fence_after();
            const ti_f2 alpha2 = ti_two(alpha_prev, alpha_prev), unit2 = ti_two(unit_prev, unit_prev);
#pragma unroll
            for (int c = 0; c < TI_OC; c += 32) {
                if (c >= cols) break;
                unsigned v[32];
                sg_tmem16(tmem + TI_O + lanes + c_first + c, *(unsigned(*)[16])v);
                if (c + 16 < cols) sg_tmem16(tmem + TI_O + lanes + c_first + c + 16, *(unsigned(*)[16])(v + 16));
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    if (i == 16 && c + 16 >= cols) break;
                    asm volatile("" : "+r"(v[i]), "+r"(v[i + 1]));
                    const ti_f2 o = ti_two(__uint_as_float(v[i]), __uint_as_float(v[i + 1]));
                    ti_f2& to = acc[(c + i) / 2];
                    to = I8 ? ti_fma2(o, unit2, ti_mul2(to, alpha2)) : ti_fma2(to, alpha2, o);
                }
            }
            pg_fence_before();
        };
#pragma unroll 1
        for (int k = 0; k < steps; k++) {
            const unsigned slot = k & 1;
            const int key0 = lo + k * TI_KEYS + part * TI_XC;
            float f[TI_XC / 16];                                               // factor of 16 keys' sums
#pragma unroll
            for (int g = 0; g < TI_XC / 16; g++) f[g] = f0 * sh.info[k & (TI_STEPS - 1)].kf[part * (TI_XC / 16) + g];
            ok = ok && ti_wait_warp(pg_smem(&sh.s_full[slot]), (k >> 1) & 1u, &sh.fail);
            unsigned x[TI_XC];
            if (ok) {
                pg_fence_after();
#pragma unroll
                for (int c = 0; c < TI_XC; c += 16) sg_tmem16(tmem + slot * 128 + lanes + part * TI_XC + c, *(unsigned(*)[16])(x + c));
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int c = 0; c < TI_XC; c++) asm volatile("" : "+r"(x[c]));
            }
            // scores, each rounded once, so that the largest is one of them and their differences from it end at 0.  (x f + base in one multiply-add, of a largest score and a base that
            // are rounded, makes weights beyond what f16 holds once their last places pass 8, from 2^27 on)
#pragma unroll
            for (int c = 0; c < TI_XC; c += 2) {
                if (CAP) {
                    x[c] = __float_as_uint(a.softcap * tanhf(__uint_as_float(x[c]) * f[c / 16] / a.softcap) * PT_LOG2E);
                    x[c + 1] = __float_as_uint(a.softcap * tanhf(__uint_as_float(x[c + 1]) * f[c / 16] / a.softcap) * PT_LOG2E);
                } else {
                    const float2 y = ti_one(ti_mul2(ti_two(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), ti_two(f[c / 16], f[c / 16])));
                    x[c] = __float_as_uint(y.x); x[c + 1] = __float_as_uint(y.y);
                }
            }
            if (lo + k * TI_KEYS + TI_KEYS - 1 > min(pos_first, k1 - 1) || (a.window > 0 && lo + k * TI_KEYS < pos_last - a.window + 1)) {
                const int c_lo = key_lo - key0, c_hi = key_hi - key0;
#pragma unroll
                for (int c = 0; c < TI_XC; c++)
                    if (c > c_hi || c < c_lo) x[c] = 0xff800000u;
            }
            float mx = -INFINITY, nx = -INFINITY;
#pragma unroll
            for (int g = 0; g < TI_XC / 16; g++) {
                float y = fmaxf(__uint_as_float(x[g * 16]), __uint_as_float(x[g * 16 + 1]));
#pragma unroll
                for (int c = 2; c < 16; c += 2) y = ti_max3(y, __uint_as_float(x[g * 16 + c]), __uint_as_float(x[g * 16 + c + 1]));
                mx = fmaxf(mx, y);
                if (I8) nx = fmaxf(nx, y + sh.info[k & (TI_STEPS - 1)].lv[part * (TI_XC / 16) + g]);
            }
            sh.top[slot][part][row] = make_float2(mx, nx);
            ti_step_sync();                                           // .. and all parts have read S
#pragma unroll
            for (int i = 0; i < TI_SPLIT; i++) {
                const float2 z = sh.top[slot][i][row];
                mx = fmaxf(mx, z.x); nx = fmaxf(nx, z.y);
            }
            const float* vfs = sh.info[k & (TI_STEPS - 1)].vf;
            const float m_new = fmaxf(m, mx), base = m_new == -INFINITY ? 0.0f : -m_new;
            const float alpha = m == m_new ? 1.0f : pt_exp2(m - m_new);
            m = m_new;
            // The operands of the values' product, a weight times its block's factor, are near 2^9 where that is largest for this row in this step, whatever the other factors and weights: `unit`
            // is the power of two that they are in, 2^-PT_FAR at least: a hidden key's 2^-126 stays 0
            const float unit = I8 ? pt_pow2(fmaxf(floorf(nx - m_new), -PT_FAR)) : 1.0f, per_unit = I8 ? TI_TOP * pt_pow2(-fmaxf(floorf(nx - m_new), -PT_FAR)) : TI_TOP;
            ti_f2 sum = 0ull;
            const ti_f2 base2 = ti_two(base, base), minus = ti_two(-1.0f, -1.0f);
            auto weights = [&](int g) {                               // of 16 keys: 8 words of h, 8 of l
                unsigned h[8], w[8];
                const float vr = I8 ? per_unit * vfs[part * (TI_XC / 16) + g] : per_unit;
                const ti_f2 vr2 = ti_two(vr, vr);
#pragma unroll
                for (int c = 0; c < 16; c += 2) {
                    const float2 y = ti_one(ti_add2(ti_two(__uint_as_float(x[g * 16 + c]), __uint_as_float(x[g * 16 + c + 1])), base2));
                    ti_f2 p = c % 16 >= TI_SFU ? ti_exp2_pair(y) : ti_two(pt_exp2(y.x), pt_exp2(y.y));
                    sum = ti_add2(sum, p);
                    p = ti_mul2(p, vr2);
                    const float2 q = ti_one(p);
                    const __half2 a2 = __floats2half2_rn(q.x, q.y);
                    const float2 b2 = __half22float2(a2), rest2 = ti_one(ti_fma2(ti_two(b2.x, b2.y), minus, p));
                    h[c / 2] = *(const unsigned*)&a2;
                    w[c / 2] = pt_pack(rest2.x, rest2.y);
                }
                ti_store8(tmem + slot * 128 + lanes + part * (TI_XC / 2) + g * 8, h);
                ti_store8(tmem + slot * 128 + lanes + 64 + part * (TI_XC / 2) + g * 8, w);
            };
            if (ok) {
#pragma unroll
                for (int g = 0; g < TI_XC / 32; g++) weights(g);
            }
            if (k > 0) add(k - 1);                                    // by now its products are done, and those of this step wait for the room
            if (ok) {
#pragma unroll
                for (int g = TI_XC / 32; g < TI_XC / 16; g++) weights(g);
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                pg_fence_before();
                sg_arrive(pg_smem(&sh.p_full[slot]));
            }
            const float2 sums = ti_one(sum);
            l = fmaf(l, alpha, (sums.x + sums.y) * TI_TOP);
            alpha_prev = alpha; unit_prev = unit;
        }
        if (steps > 0) add(steps - 1);
        if (isnan(f0)) l = NAN;                                       // a query that is not finite: maxima and the pairs' exponentials drop NaN
        // values and factors that are not finite were left out: NaN for the rows that see them
        unsigned long long lost = 0;
#pragma unroll 1
        for (int k = 0; sh.odd && k < steps; k++) {
            const TiInfo& info = sh.first[(size_t)k * a.heads];
            const unsigned* bad = info.bad;
            if (!(bad[0] | bad[1] | bad[2] | bad[3] | (unsigned)info.wild)) continue;
            const int key0 = lo + k * TI_KEYS;
#pragma unroll 1
            for (int key = max(key0, key_lo); key <= min(key0 + TI_KEYS - 1, key_hi); key++) {
                if (bad[(key - key0) >> 5] >> ((key - key0) & 31) & 1u) lost = ~0ull;
                if (I8 && key < opens) continue;
                const __half* p = (I8 ? a.vo + ((size_t)(2 * s.slot + ((to >> a.shift) & 1)) * a.G + kvh) * a.page * a.dv
                                      : (const __half*)a.v + ((size_t)a.table[(int64_t)seq * a.table_cols + (key >> a.shift)] * a.G + kvh) * a.page * a.dv) + (size_t)(key & (a.page - 1)) * a.dv + c_first;
#pragma unroll 1
                for (int c = 0; c < cols; c++)
                    if (((unsigned)__half_as_ushort(p[c]) & 0x7c00u) == 0x7c00u) lost |= 1ull << c;
            }
        }
        float o4[TI_OC];
#pragma unroll
        for (int c = 0; c < TI_OC; c += 2) {
            const float2 u = ti_one(acc[c / 2]);
            o4[c] = lost >> c & 1u ? NAN : u.x;
            o4[c + 1] = lost >> (c + 1) & 1u ? NAN : u.y;
        }
        sh.sum[part][row] = l;
        ti_soft_sync();
        l = 0.0f;
#pragma unroll
        for (int i = 0; i < TI_SPLIT; i++) l += sh.sum[i][row];
        float f = 1.0f;
        const size_t at = ((size_t)item * a.heads + head_at) * TI_ROWS;
        if (n_split > 1) {
            if (in && part == 0) a.ml[at + row] = make_float2(m, l);
        } else {
            if (a.sink && in) {
                const float sk = a.sink[head] * PT_LOG2E, m2 = fmaxf(m, sk);
                f = m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : exp2f(m - m2);
                l = f * l + (sk == -INFINITY ? 0.0f : exp2f(sk - m2 + PT_SHIFT));
            }
            f = f / l;
        }
        // by way of shared memory, 16 bytes j of a row at j ^ row % 8, so that whole rows are stored at a time
#pragma unroll
        for (int c = 0; c < TI_OC; c += 4)
            if (c < cols) *(float4*)(qs + row * 512 + ((((c_first + c) >> 2) ^ (row & 7)) << 4)) = make_float4(o4[c] * f, o4[c + 1] * f, o4[c + 2] * f, o4[c + 3] * f);
        ti_soft_sync();
        for (int r = warp; r < n_rows && ok; r += TI_SOFT_WARPS) {
            const int tk = (row0 + r) / a.R, hd = kvh * a.R + (row0 + r) - tk * a.R;
            float* o = n_split > 1 ? a.part + (at + r) * a.dv : a.out + ((int64_t)(s.first + tk) * a.H + hd) * a.dv;
            if (lane * 4 < a.dv) ((float4*)o)[lane] = *(const float4*)(qs + r * 512 + ((lane ^ (r & 7)) << 4));
        }
    }
    pg_fence_before();
    __syncthreads();
    if (warp == (TI_SOFT_WARPS + 1)) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
    if (tid == 0 && sh.fail) {
        if (err_dev) atomicExch(err_dev, 5u);
        if (err_host) { *(volatile unsigned*)err_host = 5u; __threadfence_system(); }
    }
}
