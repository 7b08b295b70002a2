// paged_tile.cuh -- attention of many rows over pages (prompts, drafts of many heads), on tcgen05.mma.  Included by paged_attn.cu behind its few-row kernel.
//
// A tile is 128 rows (a row: a query of one head; the heads of a key head side by side) x the keys they see, 128 at a time:
//   S = Q_h K^T + Q_l K^T     (K as f16 in shared memory: codes and 16-bit numbers are exact)     2 x 128 x 128 x dk products
//   P = exp2(S f - largest) as f16 h and l, written over S in TMEM, the first operand of
//   O = P_h V + P_l V         in an accumulator of its own, added to 32-bit registers afterwards: the tensor core cuts its sums off at 24 bits, a chain over
//                             thousands of keys would drift (1e-5 of a result after 2000 keys of one sign)
// S and O have two buffers each (512 TMEM columns), K and V two stages of f16 (128 KB beside the 64 KB of Q): while warps 0-7 make the weights of one step, the
// tensor core computes the scores of the next and the sums of the one before, and warps 8-13 read, convert and store the keys and values behind.
// A row's 128 scores lie with two threads, lane and half; they exchange their largest score once a step.
// Warps 0-7 weights and sums, 8-13 keys and values, 15 issues the products.  Every wait is bounded (sg_wait); where one ran out all roles run to their ends without
// waiting (the barrier of warps 0-7 included) and the host reports it.
#pragma once
#include "split_gemm.cuh"

#define TI_ROWS 128
#define TI_KEYS 128
#define TI_THREADS 512                        // 8 warps of weights and sums, 6 of keys and values, one that issues the products, one idle
#define TI_SOFT 256
#define TI_LOADERS 6
// 512 threads of 128 registers at launch are 256 of 200 and 256 of 56 afterwards (65536 either way)
#define TI_REGS_SOFT 200
#define TI_REGS_REST 56
static_assert(TI_SOFT * TI_REGS_SOFT + (TI_THREADS - TI_SOFT) * TI_REGS_REST <= TI_THREADS * 128, "more registers than the block was launched with");
#define TI_MOST 4096                          // keys of a slice
#define TI_D 128                              // largest dk and dv

struct TiShared {
    unsigned long long k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], o_empty[2], drained;
    unsigned tmem_base;
    int fail, wild[4];                        // wild[step % 4] == step + 1: values that are not finite were left out of the step's sums
    int page[TI_MOST / 16 + 8];              // of every 16 keys: -1 - block for the open one
    float kf[TI_MOST / 16 + 8], vf[TI_MOST / 16 + 8];      // vf: relative to vref, a power of two near a step's largest
    float vref[TI_MOST / TI_KEYS + 1];
    int lost;                                // some factor is not finite: it counts as 0, and NaN goes to the rows that see its keys (nan)
    uint8_t nan[TI_MOST / 16 + 8];
    float top[2][2][TI_ROWS], sum[2][TI_ROWS];
};
#define TI_OPERAND (TI_KEYS * TI_D * 2)       // bytes of a tile of f16: two blocks of 64 columns, rows of 128 bytes under the 128-byte swizzle
#define TI_GROUP 2048                         // bytes of a group as it lies in its page, two slots a warp
#define TI_SMEM (6 * TI_OPERAND + 2 * TI_LOADERS * TI_GROUP + 1024)

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
__device__ __forceinline__ float ti_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// pairs of 32-bit numbers in one instruction
typedef unsigned long long ti_f2;
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
__device__ __forceinline__ float ti_max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ void ti_soft_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// What hot loops do not hold: the kernel's roles share an instruction cache, and with everything in line they waited for it most of the time (285 -> TI_COLD_US us).
// 16 rows of an open block into an operand, values that are not finite as zeros: whether there were any
__device__ __noinline__ bool ti_open_rows(uint8_t* base, const __half* p, int d, int there, bool val) {
    bool wild = false;
    for (int e = threadIdx.x & 31; e < 16 * (d / 8); e += 32) {
        const int r = e / (d / 8);
        uint4 x = make_uint4(0, 0, 0, 0);
        if (r < there) x = ((const uint4*)p)[e];
        if (val) {
            const unsigned w0 = pt_wild(x.x), w1 = pt_wild(x.y), w2 = pt_wild(x.z), w3 = pt_wild(x.w);
            wild |= (w0 | w1 | w2 | w3) != 0u;
            x.x &= ~w0; x.y &= ~w1; x.z &= ~w2; x.w &= ~w3;
        }
        *(uint4*)(base + ti_at(r, e - r * (d / 8))) = x;
    }
    return wild;
}
// the columns, of `cols` from c_first on, that are not finite in a value that the row sees among the keys key0 .. key0 + TI_KEYS (all of them for a factor that is not)
template <bool I8>
__device__ __noinline__ unsigned long long ti_lost(const PtArgs& a, const int* page, const uint8_t* nan, int kvh, int key0, int key_lo, int key_hi, int c_first, int cols) {
    unsigned long long lost = 0;
    for (int key = max(key0, key_lo); key <= min(key0 + TI_KEYS - 1, key_hi); key++) {
        const int g = (key - key0) >> 4;
        if (nan[g]) lost = ~0ull;
        if (I8 && page[g] >= 0) continue;
        const __half* p = (I8 ? a.vo : (const __half*)a.v) + (((size_t)(I8 ? -1 - page[g] : page[g]) * a.G + kvh) * a.page + (key & (a.page - 1))) * a.dv + c_first;
        for (int c = 0; c < cols; c++)
            if (((unsigned)__half_as_ushort(p[c]) & 0x7c00u) == 0x7c00u) lost |= 1ull << c;
    }
    return lost;
}
template <bool I8, bool CAP>
__global__ void __launch_bounds__(TI_THREADS, 1) paged_tile_kernel(const __grid_constant__ PtArgs a, unsigned* err_dev, unsigned* err_host) {
    extern __shared__ __align__(1024) uint8_t ti_raw[];
    __shared__ TiShared sh;
    uint8_t* qs = (uint8_t*)(((uintptr_t)ti_raw + 1023) & ~(uintptr_t)1023);      // Q_h, Q_l
    uint8_t *ks = qs + 2 * TI_OPERAND, *vs = ks + 2 * TI_OPERAND;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kvh = blockIdx.y;
    if (tid == 0) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            pg_mbar_init(pg_smem(&sh.k_full[i]), I8 ? TI_KEYS / 16 : TI_KEYS / 8); pg_mbar_init(pg_smem(&sh.v_full[i]), I8 ? TI_KEYS / 16 : TI_KEYS / 8); pg_mbar_init(pg_smem(&sh.k_empty[i]), 1); pg_mbar_init(pg_smem(&sh.v_empty[i]), 1);
            pg_mbar_init(pg_smem(&sh.s_full[i]), 1); pg_mbar_init(pg_smem(&sh.p_full[i]), 8); pg_mbar_init(pg_smem(&sh.o_full[i]), 1); pg_mbar_init(pg_smem(&sh.o_empty[i]), 8);
            sh.wild[i] = sh.wild[i + 2] = 0;
        }
        pg_mbar_init(pg_smem(&sh.drained), 1);
        sh.fail = sh.lost = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_enter();
    __syncthreads();
    int rest;
    const int seq = pt_find(a, blockIdx.x, [&](const PgSeq& s) { return pt_splits(s, a) * (int)(((int64_t)s.count * a.R + TI_ROWS - 1) / TI_ROWS); }, &rest);
    if (seq < 0) return;                                              // (the grid has as many CTAs as there are items)
    const PgSeq s = a.seqs[seq];
    const int rows = s.count * a.R, tiles = (rows + TI_ROWS - 1) / TI_ROWS, n_split = pt_splits(s, a), tile = tiles - 1 - rest / n_split, split = rest % n_split;      // late rows, which see most, first
    int from, to;
    pt_range(s, a.window, &from, &to);
    const int row0 = tile * TI_ROWS, n_rows = min(TI_ROWS, rows - row0), pos_first = s.pos0 + row0 / a.R, pos_last = s.pos0 + (row0 + n_rows - 1) / a.R;
    const int k0 = from + split * a.split, k1 = min(min(to, k0 + a.split), pos_last + 1);
    const int lo = a.window > 0 ? max(k0, (pos_first - a.window + 1) & ~15) : k0, steps = k1 > lo ? (k1 - lo + TI_KEYS - 1) / TI_KEYS : 0;
    const int opens = I8 ? to >> a.shift << a.shift : 0;
    for (int i = tid; i < steps * (TI_KEYS / 16); i += TI_THREADS) {
        const int key = lo + i * 16;
        float kf = 1.0f, vf = 1.0f;
        int page = 0;
        if (key < to) {
            page = a.table[(int64_t)seq * a.table_cols + (key >> a.shift)];
            if (I8 && key >= opens) page = -1 - (2 * s.slot + ((to >> a.shift) & 1));
            else if (I8) { kf = a.ks[(int64_t)page * a.G + kvh]; vf = a.vs[(int64_t)page * a.G + kvh]; }
        }
        const bool bad = !(vf >= 0.0f && vf < INFINITY && kf >= 0.0f && kf < INFINITY);
        sh.page[i] = page; sh.kf[i] = bad ? 0.0f : kf; sh.vf[i] = bad ? 0.0f : vf; sh.nan[i] = bad;
        if (bad) sh.lost = 1;
    }
    __syncthreads();
    for (int k = tid; k < steps; k += TI_THREADS) {
        float most = 0.0f;
#pragma unroll
        for (int g = 0; g < TI_KEYS / 16; g++) most = fmaxf(most, sh.vf[k * (TI_KEYS / 16) + g]);
        const float vref = fminf(fmaxf(__uint_as_float(__float_as_uint(most) & 0x7f800000u), 0x1p-100f), 0x1p100f);
        sh.vref[k] = vref;
#pragma unroll
        for (int g = 0; g < TI_KEYS / 16; g++) sh.vf[k * (TI_KEYS / 16) + g] /= vref;
    }
    if (warp == 15) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(pg_smem(&sh.tmem_base)), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // the queries as h and l, near 2^14
    const int row = (warp & 3) * 32 + lane, half = (warp >> 2) & 1;   // warps 0-7: TMEM lane and half of the columns
    const int tok = (row0 + row) / a.R, head = kvh * a.R + (row0 + row) - tok * a.R;
    const bool in = warp < 8 && row < n_rows;
    float inv = 1.0f;
    if (warp < 8) {
        const float* q = a.q + ((int64_t)(s.first + tok) * a.H + head) * a.dk;
        float top = 0.0f;
        for (int c = half * 4; c < a.dk; c += 8) {
            const float4 v = in ? *(const float4*)(q + c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            top = fmaxf(top, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
        }
        sh.top[0][half][row] = top;
        ti_soft_sync();
        top = fmaxf(top, sh.top[0][half ^ 1][row]);
        int ex = 14;
        if (top > 0.0f && top < INFINITY) frexpf(top, &ex);
        ex = max(ex, -100);
        const float f = copysignf(ldexpf(1.0f, 14 - ex), a.scale);      // (so that a larger sum is a larger score)
        inv = ldexpf(1.0f, ex - 14);
        for (int j = half; j < a.dk / 8; j += 2) {
            float v[8];
#pragma unroll
            for (int i = 0; i < 8; i += 4) {
                const float4 u = in ? *(const float4*)(q + j * 8 + i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                v[i] = u.x * f; v[i + 1] = u.y * f; v[i + 2] = u.z * f; v[i + 3] = u.w * f;
            }
            uint4 h, l;
            pt_cut(v[0], v[1], h.x, l.x); pt_cut(v[2], v[3], h.y, l.y); pt_cut(v[4], v[5], h.z, l.z); pt_cut(v[6], v[7], h.w, l.w);
            *(uint4*)(qs + ti_at(row, j)) = h;
            *(uint4*)(qs + TI_OPERAND + ti_at(row, j)) = l;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    pg_fence_before();
    __syncthreads();
    pg_fence_after();
    const unsigned tmem = sh.tmem_base;

    if (warp >= TI_SOFT / 32) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TI_REGS_REST));
    else asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TI_REGS_SOFT));
    if (warp == 15) {
        // ===== products: one thread =====
        if (lane == 0) {
            const unsigned idesc_s = pg_instr_desc(128, TI_KEYS), idesc_o = pg_instr_desc(128, a.dv) | 1u << 16;
            const unsigned qa = pg_smem(qs);
            bool ok = true;
            auto scores = [&](int k) {
                const unsigned slot = k & 1, at = pg_smem(ks + (size_t)slot * TI_OPERAND);
                if (!(ok = ti_wait(pg_smem(&sh.k_full[slot]), (k >> 1) & 1u, &sh.fail))) return;
                pg_fence_after();
                for (int x = 0; x < 2; x++)
                    for (int kk = 0; kk < a.dk / 16; kk++) {
                        const unsigned off = (unsigned)((kk >> 2) * (TI_OPERAND / 2) + (kk & 3) * 32);
                        pg_umma_f16(tmem + slot * 128, pg_smem_desc(qa + x * TI_OPERAND + off), pg_smem_desc(at + off), idesc_s, x > 0 || kk > 0);
                    }
                pg_umma_commit(pg_smem(&sh.s_full[slot]));
                pg_umma_commit(pg_smem(&sh.k_empty[slot]));
            };
            if (steps > 0) scores(0);
            for (int k = 0; k < steps && ok; k++) {
                const unsigned slot = k & 1, ph = (k >> 1) & 1u;
                if (k + 1 < steps) scores(k + 1);
                if (!ok || !(ok = ti_wait(pg_smem(&sh.p_full[slot]), ph, &sh.fail) && ti_wait(pg_smem(&sh.v_full[slot]), ph, &sh.fail) &&
                                  ti_wait(pg_smem(&sh.o_empty[slot]), ph ^ 1u, &sh.fail))) break;
                pg_fence_after();
                const unsigned at = pg_smem(vs + (size_t)slot * TI_OPERAND);
                for (int x = 0; x < 2; x++)
                    for (int kk = 0; kk < TI_KEYS / 16; kk++)
                        ti_umma_ts(tmem + 256 + slot * 128, tmem + slot * 128 + x * 64 + kk * 8, ti_desc_mn(at + kk * 2048), idesc_o, x > 0 || kk > 0);
                pg_umma_commit(pg_smem(&sh.o_full[slot]));
                pg_umma_commit(pg_smem(&sh.v_empty[slot]));
            }
            int never = 0;                                            // nothing of this CTA is in flight when its TMEM is given back
            pg_umma_commit(pg_smem(&sh.drained));
            ti_wait(pg_smem(&sh.drained), 0, &never);
        }
        __syncwarp();
    } else if (warp >= 8) {
        // ===== keys and values: a warp takes 2 KB of an operand at a time (a group: 16 rows of codes or 8 of 16-bit numbers, in one page), its next one is under way to
        // shared memory meanwhile; every lane reads there what it copied itself =====
        constexpr int N = TI_GROUP / 512, E = I8 ? 16 : 8, GR = I8 ? 16 : 8, PER = TI_KEYS / GR;      // pieces of 16 bytes of a lane, numbers of a piece, rows of a group, groups of an operand
        const int groups = warp < TI_SOFT / 32 + TI_LOADERS ? steps * 2 * PER : 0, per_k = a.dk / E, per_v = a.dv / E;
        uint8_t* mine = vs + 2 * TI_OPERAND + (size_t)(warp - TI_SOFT / 32) * 2 * TI_GROUP + lane * 16;
        const unsigned mine_at = pg_smem(mine);
        // where the lane's pieces lie in an operand's rows; 8-bit: the chunk that is stored first, bit 0 set where that is the piece's second one
        unsigned off_k[N], off_v[N];
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int v = 0; v < 2; v++) {
                const int per = v ? per_v : per_k, e = i * 32 + lane, row = e / per, piece = e - row * per, second = piece >> 2 & 1;
                (v ? off_v : off_k)[i] = row >= GR ? ~0u : I8 ? ti_at(row, 2 * piece + second) | second : ti_at(row, piece);
            }
        auto fetch = [&](int u, unsigned to_smem) {
            if (u < groups) {
                const int step = u / (2 * PER), g = u & (PER - 1), key = lo + step * TI_KEYS + g * GR, page = sh.page[(step * TI_KEYS + g * GR) >> 4];
                const bool val = u & PER;
                const int d = val ? a.dv : a.dk, there = min(GR, to - key) * (d / E);
                if (!I8 || page >= 0) {                                // (the open block's rows come when they are stored)
                    const size_t at = (((size_t)page * a.G + kvh) * a.page + (key & (a.page - 1))) * d;
                    const uint8_t* p = (val ? a.v : a.k) + (I8 ? at : at * 2);
#pragma unroll
                    for (int i = 0; i < N; i++) pt_copy16(to_smem + i * 512, i * 32 + lane < there ? p + (i * 32 + lane) * 16 : p, i * 32 + lane < there);      // zeros behind the end
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        bool ok = true;
        const int first = warp - TI_SOFT / 32;
        unsigned turn = 0;
        fetch(first, mine_at);
#pragma unroll 1
        for (int u = first; u < groups; u += TI_LOADERS, turn ^= TI_GROUP) {
            const int step = u / (2 * PER), g = u & (PER - 1);
            const bool val = u & PER;
            fetch(u + TI_LOADERS, mine_at + (turn ^ TI_GROUP));
            if (!(ok = ti_wait_warp(pg_smem(val ? &sh.v_empty[step & 1] : &sh.k_empty[step & 1]), ((step >> 1) & 1u) ^ 1u, &sh.fail))) break;
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            uint8_t* base = (val ? vs : ks) + (size_t)(step & 1) * TI_OPERAND + g * GR * 128;
            const int page = sh.page[(step * TI_KEYS + g * GR) >> 4];
            bool wild = false;
            if (I8 && page < 0) {
                const int key = lo + step * TI_KEYS + g * GR, d = val ? a.dv : a.dk;
                wild = ti_open_rows(base, (val ? a.vo : a.ko) + (((size_t)(-1 - page) * a.G + kvh) * a.page + (key & (a.page - 1))) * d, d, to - key, val);
            } else {
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const unsigned off = val ? off_v[i] : off_k[i];
                    if (off == ~0u) continue;
                    const uint4 r = *(const uint4*)(mine + turn + i * 512);
                    if (I8) {
                        // the lanes of a row fill all banks at once: those of its second half store their second 8 numbers first (chunk 2 p + 1 is chunk 2 p with 16 flipped)
                        const bool odd = off & 1u;
                        const unsigned a0 = (odd ? r.z : r.x) ^ 0x80808080u, a1 = (odd ? r.w : r.y) ^ 0x80808080u;
                        const unsigned b0 = (odd ? r.x : r.z) ^ 0x80808080u, b1 = (odd ? r.y : r.w) ^ 0x80808080u;
                        const unsigned at = off & ~1u;
                        *(uint4*)(base + at) = make_uint4(pt_half2(a0, 0x4140), pt_half2(a0, 0x4342), pt_half2(a1, 0x4140), pt_half2(a1, 0x4342));
                        *(uint4*)(base + (at ^ 16u)) = make_uint4(pt_half2(b0, 0x4140), pt_half2(b0, 0x4342), pt_half2(b1, 0x4140), pt_half2(b1, 0x4342));
                    } else {
                        uint4 x = r;
                        if (val) {
                            const unsigned w0 = pt_wild(x.x), w1 = pt_wild(x.y), w2 = pt_wild(x.z), w3 = pt_wild(x.w);
                            wild |= (w0 | w1 | w2 | w3) != 0u;
                            x.x &= ~w0; x.y &= ~w1; x.z &= ~w2; x.w &= ~w3;
                        }
                        *(uint4*)(base + off) = x;
                    }
                }
            }
            if (wild) atomicExch(&sh.wild[step & 3], step + 1);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            sg_arrive(pg_smem(val ? &sh.v_full[step & 1] : &sh.k_full[step & 1]));
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else {
        // ===== weights and sums =====
        const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
        const int c_first = half ? ((a.dv / 2 + 15) & ~15) : 0, cols = half ? a.dv - c_first : (a.dv / 2 + 15) & ~15;      // this thread's columns of O
        const int pos = in ? s.pos0 + tok : -1, key_lo = a.window > 0 ? pos - a.window + 1 : 0, key_hi = min(pos, k1 - 1);      // the last step may reach into the next slice
        const float f0 = inv * fabsf(a.scale) * (CAP ? 1.0f : PT_LOG2E);
        ti_f2 acc[TI_D / 4];
        float m = -INFINITY, l = 0.0f, alpha_prev = 0.0f, vref_prev = 0.0f;
        unsigned long long lost = 0;                                  // columns of this thread that have met a value that is not finite
#pragma unroll
        for (int i = 0; i < TI_D / 4; i++) acc[i] = 0ull;
        bool ok = true;
        auto add = [&](int k) {                                       // the sums of step k
            const unsigned slot = k & 1;
            if (!(ok = ok && ti_wait_warp(pg_smem(&sh.o_full[slot]), (k >> 1) & 1u, &sh.fail))) return;
            pg_fence_after();
            const ti_f2 alpha2 = ti_two(alpha_prev, alpha_prev), vref2 = ti_two(vref_prev, vref_prev);
#pragma unroll
            for (int c = 0; c < TI_D / 2; c += 32) {
                if (c >= cols) break;
                unsigned v[32];
                sg_tmem16(tmem + 256 + slot * 128 + lanes + c_first + c, *(unsigned(*)[16])v);
                if (c + 16 < cols) sg_tmem16(tmem + 256 + slot * 128 + lanes + c_first + c + 16, *(unsigned(*)[16])(v + 16));
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    if (i == 16 && c + 16 >= cols) break;
                    asm volatile("" : "+r"(v[i]), "+r"(v[i + 1]));
                    const ti_f2 o = ti_two(__uint_as_float(v[i]), __uint_as_float(v[i + 1]));
                    ti_f2& to = acc[(c + i) / 2];
                    to = I8 ? ti_fma2(o, vref2, ti_mul2(to, alpha2)) : ti_fma2(to, alpha2, o);
                }
            }
            pg_fence_before();
            sg_arrive(pg_smem(&sh.o_empty[slot]));
            if (*(volatile int*)&sh.wild[k & 3] == k + 1 || sh.lost)
                lost |= ti_lost<I8>(a, sh.page + k * (TI_KEYS / 16), sh.nan + k * (TI_KEYS / 16), kvh, lo + k * TI_KEYS, key_lo, key_hi, c_first, cols);
        };
#pragma unroll 1
        for (int k = 0; k < steps; k++) {
            const unsigned slot = k & 1;
            const int key0 = lo + k * TI_KEYS + half * 64;
            float f[4];                                               // factor of 16 keys' sums; 0 (a block of zeros) must not meet the -inf of a hidden key
#pragma unroll
            for (int g = 0; g < 4; g++) {
                f[g] = f0 * sh.kf[k * (TI_KEYS / 16) + half * 4 + g];
                f[g] = f[g] == 0.0f ? 1e-37f : f[g];
            }
            ok = ok && ti_wait_warp(pg_smem(&sh.s_full[slot]), (k >> 1) & 1u, &sh.fail);
            unsigned x[64];
            if (ok) {
                pg_fence_after();
#pragma unroll
                for (int c = 0; c < 64; c += 16) sg_tmem16(tmem + slot * 128 + lanes + half * 64 + c, *(unsigned(*)[16])(x + c));
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int c = 0; c < 64; c++) asm volatile("" : "+r"(x[c]));
            }
            if (CAP) {
#pragma unroll
                for (int c = 0; c < 64; c++) x[c] = __float_as_uint(a.softcap * tanhf(__uint_as_float(x[c]) * f[c / 16] / a.softcap) * PT_LOG2E);
#pragma unroll
                for (int g = 0; g < 4; g++) f[g] = 1.0f;
            }
            if (lo + k * TI_KEYS + TI_KEYS - 1 > min(pos_first, k1 - 1) || (a.window > 0 && lo + k * TI_KEYS < pos_last - a.window + 1)) {
                const int c_lo = key_lo - key0, c_hi = key_hi - key0;
#pragma unroll
                for (int c = 0; c < 64; c++)
                    if (c > c_hi || c < c_lo) x[c] = 0xff800000u;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int g = 0; g < 4; g++) {
                float y = fmaxf(__uint_as_float(x[g * 16]), __uint_as_float(x[g * 16 + 1]));
#pragma unroll
                for (int c = 2; c < 16; c += 2) y = ti_max3(y, __uint_as_float(x[g * 16 + c]), __uint_as_float(x[g * 16 + c + 1]));
                mx = fmaxf(mx, y * f[g]);
            }
            sh.top[slot][half][row] = mx;
            ti_soft_sync();                                           // .. and both halves have read S
            mx = fmaxf(mx, sh.top[slot][half ^ 1][row]);
            const float* vfs = sh.vf + k * (TI_KEYS / 16);
            const float m_new = fmaxf(m, mx), base = m_new == -INFINITY ? 0.0f : PT_SHIFT - m_new;
            const float alpha = m == m_new ? 1.0f : ti_exp2(m - m_new);
            m = m_new;
            ti_f2 sum = 0ull;
            if (ok) {
                const ti_f2 base2 = ti_two(base, base);
#pragma unroll
                for (int g = 0; g < 4; g++) {                         // 16 keys at a time: 8 words of h, 8 of l
                    unsigned h[8], w[8];
                    const float vr = I8 ? vfs[half * 4 + g] : 1.0f;
                    const ti_f2 f2 = ti_two(f[g], f[g]), vr2 = ti_two(vr, vr), minus = ti_two(-1.0f, -1.0f);
#pragma unroll
                    for (int c = 0; c < 16; c += 2) {
                        const float2 y = ti_one(ti_fma2(ti_two(__uint_as_float(x[g * 16 + c]), __uint_as_float(x[g * 16 + c + 1])), f2, base2));
                        ti_f2 p = ti_two(ti_exp2(y.x), ti_exp2(y.y));
                        sum = ti_add2(sum, p);
                        if (I8) p = ti_mul2(p, vr2);
                        const float2 q = ti_one(p);
                        const __half2 a2 = __floats2half2_rn(q.x, q.y);
                        const float2 b2 = __half22float2(a2), rest2 = ti_one(ti_fma2(ti_two(b2.x, b2.y), minus, p));
                        h[c / 2] = *(const unsigned*)&a2;
                        w[c / 2] = pt_pack(rest2.x, rest2.y);
                    }
                    ti_store8(tmem + slot * 128 + lanes + half * 32 + g * 8, h);
                    ti_store8(tmem + slot * 128 + lanes + 64 + half * 32 + g * 8, w);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                pg_fence_before();
                sg_arrive(pg_smem(&sh.p_full[slot]));
            }
            const float2 sums = ti_one(sum);
            l = fmaf(l, alpha, sums.x + sums.y);
            if (k > 0) add(k - 1);
            alpha_prev = alpha; vref_prev = I8 ? sh.vref[k] : 1.0f;
        }
        if (steps > 0) add(steps - 1);
        float o4[TI_D / 2];
#pragma unroll
        for (int c = 0; c < TI_D / 2; c += 2) {
            const float2 u = ti_one(acc[c / 2]);
            o4[c] = lost >> c & 1u ? NAN : u.x;
            o4[c + 1] = lost >> (c + 1) & 1u ? NAN : u.y;
        }
        sh.sum[half][row] = l;
        ti_soft_sync();
        l = sh.sum[0][row] + sh.sum[1][row];
        if (in && ok) {
            if (n_split > 1) {
                const size_t at = ((size_t)blockIdx.x * a.G + kvh) * TI_ROWS + row;
                float* o = a.part + at * a.dv + c_first;
#pragma unroll
                for (int c = 0; c < TI_D / 2; c += 4)
                    if (c < cols) *(float4*)(o + c) = make_float4(o4[c], o4[c + 1], o4[c + 2], o4[c + 3]);
                if (half == 0) a.ml[at] = make_float2(m, l);
            } else {
                float f = 1.0f;
                if (a.sink) {
                    const float sk = a.sink[head] * PT_LOG2E, m2 = fmaxf(m, sk);
                    f = m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : exp2f(m - m2);
                    l = f * l + (sk == -INFINITY ? 0.0f : exp2f(sk - m2 + PT_SHIFT));
                }
                float* o = a.out + ((int64_t)(s.first + tok) * a.H + head) * a.dv + c_first;
                f = f / l;
#pragma unroll
                for (int c = 0; c < TI_D / 2; c += 4)
                    if (c < cols) *(float4*)(o + c) = make_float4(o4[c] * f, o4[c + 1] * f, o4[c + 2] * f, o4[c + 3] * f);
            }
        }
    }
    pg_fence_before();
    __syncthreads();
    if (warp == 15) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
    if (tid == 0 && sh.fail) {
        if (err_dev) atomicExch(err_dev, 5u);
        if (err_host) { *(volatile unsigned*)err_host = 5u; __threadfence_system(); }
    }
}
