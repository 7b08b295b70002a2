// paged_tile.cuh -- attention of many rows over pages (prompts, drafts of many heads), on tcgen05.mma.  Included by paged_attn.cu behind its few-row kernel.
//
// A tile is 128 rows (a row: a query of one head; the heads of a key head side by side) x the keys they see, 128 at a time:
//   S = Q_h K^T + Q_l K^T     (K as f16 in shared memory: codes and 16-bit numbers are exact)     2 x 128 x 128 x dk products
//   P = exp2(S f - largest) as f16 h and l, written over S in TMEM, the first operand of
//   O = P_h V + P_l V         in an accumulator of its own, added to 32-bit registers afterwards: the tensor core cuts its sums off at 24 bits, a chain over
//                             thousands of keys would drift (1e-5 of a result after 2000 keys of one sign)
// S and O have two buffers each (512 TMEM columns), K and V two stages of f16 (128 KB beside the 64 KB of Q): while warps 0-7 make the weights of one step, the
// tensor core computes the scores of the next and the sums of the one before, and warps 8-10 read, convert and store the keys and values behind.
// A row's 128 scores lie with two threads, lane and half; they exchange their largest score once a step.
// Warps 0-7 weights and sums, 8-10 keys and values, 11 issues the products.  Every wait is bounded (sg_wait); where one ran out all roles run to their ends without
// waiting (the barrier of warps 0-7 included) and the host reports it.
#pragma once
#include "split_gemm.cuh"

#define TI_ROWS 128
#define TI_KEYS 128
#define TI_THREADS 384                        // three warps a scheduler: 168 registers a thread (a thirteenth warp would leave 128)
#define TI_SOFT 256
#define TI_LOAD 96
#define TI_EACH 11                            // pieces of 16 bytes of a unit of 16 KB, a thread of TI_LOAD
#define TI_MOST 4096                          // keys of a slice
#define TI_D 128                              // largest dk and dv

struct TiShared {
    unsigned long long k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], o_full[2], o_empty[2], drained;
    unsigned tmem_base;
    int fail, wild[4];                        // wild[step % 4] == step + 1: values that are not finite were left out of the step's sums
    int page[TI_MOST / 16 + 8];              // of every 16 keys: -1 - block for the open one
    float kf[TI_MOST / 16 + 8], vf[TI_MOST / 16 + 8];
    float top[2][2][TI_ROWS], sum[2][TI_ROWS];
};
#define TI_OPERAND (TI_KEYS * TI_D * 2)       // bytes of a tile of f16: two blocks of 64 columns, rows of 128 bytes under the 128-byte swizzle
#define TI_SMEM (6 * TI_OPERAND + 1024)

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
__device__ __forceinline__ float ti_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void ti_soft_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <bool I8>
__global__ void __launch_bounds__(TI_THREADS, 1) paged_tile_kernel(const PtArgs a, unsigned* err_dev, unsigned* err_host) {
    extern __shared__ __align__(1024) uint8_t ti_raw[];
    __shared__ TiShared sh;
    uint8_t* qs = (uint8_t*)(((uintptr_t)ti_raw + 1023) & ~(uintptr_t)1023);      // Q_h, Q_l
    uint8_t *ks = qs + 2 * TI_OPERAND, *vs = ks + 2 * TI_OPERAND;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kvh = blockIdx.y;
    if (tid == 0) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            pg_mbar_init(pg_smem(&sh.k_full[i]), TI_LOAD / 32); pg_mbar_init(pg_smem(&sh.v_full[i]), TI_LOAD / 32); pg_mbar_init(pg_smem(&sh.k_empty[i]), 1); pg_mbar_init(pg_smem(&sh.v_empty[i]), 1);
            pg_mbar_init(pg_smem(&sh.s_full[i]), 1); pg_mbar_init(pg_smem(&sh.p_full[i]), 8); pg_mbar_init(pg_smem(&sh.o_full[i]), 1); pg_mbar_init(pg_smem(&sh.o_empty[i]), 8);
            sh.wild[i] = sh.wild[i + 2] = 0;
        }
        pg_mbar_init(pg_smem(&sh.drained), 1);
        sh.fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_enter();
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
        sh.page[i] = page; sh.kf[i] = kf; sh.vf[i] = vf;
    }
    if (warp == 11) {
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
        const float f = ldexpf(1.0f, 14 - ex);
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

    if (warp == 11) {
        // ===== products: one thread =====
        if (lane == 0) {
            const unsigned idesc_s = pg_instr_desc(128, TI_KEYS), idesc_o = pg_instr_desc(128, a.dv) | 1u << 16;
            const unsigned qa = pg_smem(qs);
            bool ok = true;
            auto scores = [&](int k) {
                const unsigned slot = k & 1, at = pg_smem(ks + (size_t)slot * TI_OPERAND);
                if (!(ok = sg_wait(pg_smem(&sh.k_full[slot]), (k >> 1) & 1u, &sh.fail))) return;
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
                if (!ok || !(ok = sg_wait(pg_smem(&sh.p_full[slot]), ph, &sh.fail) && sg_wait(pg_smem(&sh.v_full[slot]), ph, &sh.fail) &&
                                  sg_wait(pg_smem(&sh.o_empty[slot]), ph ^ 1u, &sh.fail))) break;
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
            sg_wait(pg_smem(&sh.drained), 0, &never);
        }
        __syncwarp();
    } else if (warp >= 8) {
        // ===== keys and values: pieces of 16 bytes, TI_EACH of a thread at a time (a unit); the next unit's are under way while these are converted =====
        const int t = tid - TI_SOFT, E = I8 ? 16 : 8;
        constexpr int PER = I8 ? 1 : 2;                               // units of an operand
        const int units = steps * 2 * PER;
        int4 raw[2][TI_EACH];
        // pieces i * TI_LOAD + t of a unit, rows of `per` pieces: the first one's row and piece, and what TI_LOAD pieces further on are, for keys and for values
        const int per_k = a.dk / E, per_v = a.dv / E, row_k = t / per_k, row_v = t / per_v;
        auto pieces = [&](int unit, auto each) {
            const int op = unit / PER, n = TI_KEYS / PER, first = (unit - op * PER) * n;
            const bool val = op & 1;
            const int per = val ? per_v : per_k, row_by = TI_LOAD / per, piece_by = TI_LOAD - row_by * per;
            int key = val ? row_v : row_k, piece = t - key * per;
#pragma unroll
            for (int i = 0; i < TI_EACH; i++) {
                if (key < n) each(i, op >> 1, val, first + key, piece);
                key += row_by; piece += piece_by;
                if (piece >= per) { piece -= per; key++; }
            }
        };
        auto fetch = [&](int unit, int4 (&r)[TI_EACH]) {
            if (unit >= units) return;
            pieces(unit, [&](int i, int step, bool val, int key, int piece) {
                const int abs_key = lo + step * TI_KEYS + key, page = sh.page[step * (TI_KEYS / 16) + (key >> 4)], d = val ? a.dv : a.dk;
                r[i] = make_int4(0, 0, 0, 0);
                if (abs_key >= to || (I8 && page < 0)) return;        // zeros behind the end; the open block's rows come when they are stored
                const size_t at = (((size_t)page * a.G + kvh) * a.page + (abs_key & (a.page - 1))) * d;
                r[i] = __ldg((const int4*)((val ? a.v : a.k) + (I8 ? at : at * 2)) + piece);
            });
        };
        auto store = [&](int unit, const int4 (&r)[TI_EACH]) {
            bool wild = false;
            int at_step = 0;
            pieces(unit, [&](int i, int step, bool val, int key, int piece) {
                uint8_t* to_smem = (val ? vs : ks) + (size_t)(step & 1) * TI_OPERAND;
                at_step = step;
                if (I8) {
                    const int page = sh.page[step * (TI_KEYS / 16) + (key >> 4)], abs_key = lo + step * TI_KEYS + key, d = val ? a.dv : a.dk;
                    uint4 x, y;
                    if (page < 0) {
                        const __half* p = (val ? a.vo : a.ko) + (((size_t)(-1 - page) * a.G + kvh) * a.page + (abs_key & (a.page - 1))) * d + piece * 16;
                        x = y = make_uint4(0, 0, 0, 0);
                        if (abs_key < to) { x = *(const uint4*)p; y = *(const uint4*)(p + 8); }
                        if (val) {
                            wild |= (pt_wild(x.x) | pt_wild(x.y) | pt_wild(x.z) | pt_wild(x.w) | pt_wild(y.x) | pt_wild(y.y) | pt_wild(y.z) | pt_wild(y.w)) != 0u;
                            x.x &= ~pt_wild(x.x); x.y &= ~pt_wild(x.y); x.z &= ~pt_wild(x.z); x.w &= ~pt_wild(x.w);
                            y.x &= ~pt_wild(y.x); y.y &= ~pt_wild(y.y); y.z &= ~pt_wild(y.z); y.w &= ~pt_wild(y.w);
                        }
                    } else {
                        const unsigned u0 = (unsigned)r[i].x ^ 0x80808080u, u1 = (unsigned)r[i].y ^ 0x80808080u, u2 = (unsigned)r[i].z ^ 0x80808080u, u3 = (unsigned)r[i].w ^ 0x80808080u;
                        x = make_uint4(pt_half2(u0, 0x4140), pt_half2(u0, 0x4342), pt_half2(u1, 0x4140), pt_half2(u1, 0x4342));
                        y = make_uint4(pt_half2(u2, 0x4140), pt_half2(u2, 0x4342), pt_half2(u3, 0x4140), pt_half2(u3, 0x4342));
                        if (abs_key >= to) x = y = make_uint4(0, 0, 0, 0);
                    }
                    const bool odd = piece & 4;                       // the lanes of a row fill all banks at once
                    *(uint4*)(to_smem + ti_at(key, 2 * piece + odd)) = odd ? y : x;
                    *(uint4*)(to_smem + ti_at(key, 2 * piece + !odd)) = odd ? x : y;
                } else {
                    uint4 x = make_uint4((unsigned)r[i].x, (unsigned)r[i].y, (unsigned)r[i].z, (unsigned)r[i].w);
                    if (val) {
                        const unsigned w0 = pt_wild(x.x), w1 = pt_wild(x.y), w2 = pt_wild(x.z), w3 = pt_wild(x.w);
                        wild |= (w0 | w1 | w2 | w3) != 0u;
                        x.x &= ~w0; x.y &= ~w1; x.z &= ~w2; x.w &= ~w3;
                    }
                    *(uint4*)(to_smem + ti_at(key, piece)) = x;
                }
            });
            if (wild) atomicExch(&sh.wild[at_step & 3], at_step + 1);
        };
        bool ok = true;
        fetch(0, raw[0]);
        for (int u0 = 0; u0 < units && ok; u0 += 2) {
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int unit = u0 + x, op = unit / PER, step = op >> 1;
                const unsigned slot = step & 1, ph = (step >> 1) & 1u;
                if (unit >= units || !ok) break;
                fetch(unit + 1, raw[x ^ 1]);
                if (unit % PER == 0 && !(ok = sg_wait_warp(pg_smem(op & 1 ? &sh.v_empty[slot] : &sh.k_empty[slot]), ph ^ 1u, &sh.fail))) break;
                store(unit, raw[x]);
                if (unit % PER == PER - 1) {
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    sg_arrive(pg_smem(op & 1 ? &sh.v_full[slot] : &sh.k_full[slot]));
                }
            }
        }
    } else {
        // ===== weights and sums =====
        const unsigned lanes = (unsigned)((warp & 3) * 32) << 16;
        const int c_first = half ? ((a.dv / 2 + 15) & ~15) : 0, cols = half ? a.dv - c_first : (a.dv / 2 + 15) & ~15;      // this thread's columns of O
        const int pos = in ? s.pos0 + tok : -1, key_lo = a.window > 0 ? pos - a.window + 1 : 0, key_hi = min(pos, k1 - 1);      // the last step may reach into the next slice
        const float f0 = a.softcap > 0.0f ? inv * a.scale : inv * (a.scale * PT_LOG2E);
        float acc[TI_D / 2], m = -INFINITY, l = 0.0f, alpha_prev = 0.0f, vref_prev = 0.0f;
#pragma unroll
        for (int i = 0; i < TI_D / 2; i++) acc[i] = 0.0f;
        bool ok = true;
        auto add = [&](int k) {                                       // the sums of step k
            const unsigned slot = k & 1;
            if (!(ok = ok && sg_wait_warp(pg_smem(&sh.o_full[slot]), (k >> 1) & 1u, &sh.fail))) return;
            pg_fence_after();
#pragma unroll
            for (int c = 0; c < TI_D / 2; c += 16) {
                if (c >= cols) break;
                unsigned v[16];
                sg_tmem16(tmem + 256 + slot * 128 + lanes + c_first + c, v);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    asm volatile("" : "+r"(v[i]));
                    acc[c + i] = fmaf(__uint_as_float(v[i]), vref_prev, acc[c + i] * alpha_prev);
                }
            }
            pg_fence_before();
            if (*(volatile int*)&sh.wild[k & 3] == k + 1) {            // NaN for the rows that see them
                for (int j = 0; j < TI_KEYS; j++) {
                    const int key = lo + k * TI_KEYS + j;
                    if (key > key_hi || key < key_lo) continue;
                    const int page = sh.page[k * (TI_KEYS / 16) + (j >> 4)];
                    if (I8 && page >= 0) continue;
                    const __half* p = (I8 ? a.vo : (const __half*)a.v) + (((size_t)(I8 ? -1 - page : page) * a.G + kvh) * a.page + (key & (a.page - 1))) * a.dv + c_first;
#pragma unroll
                    for (int c = 0; c < TI_D / 2; c++)
                        if (c < cols && ((unsigned)__half_as_ushort(p[c]) & 0x7c00u) == 0x7c00u) acc[c] = NAN;
                }
            }
            sg_arrive(pg_smem(&sh.o_empty[slot]));
        };
        for (int k = 0; k < steps; k++) {
            const unsigned slot = k & 1;
            const int key0 = lo + k * TI_KEYS + half * 64;
            ok = ok && sg_wait_warp(pg_smem(&sh.s_full[slot]), (k >> 1) & 1u, &sh.fail);
            unsigned x[64];
            float vmax = 0.0f;
            if (ok) {
                pg_fence_after();
#pragma unroll
                for (int c = 0; c < 64; c += 16) sg_tmem16(tmem + slot * 128 + lanes + half * 64 + c, *(unsigned(*)[16])(x + c));
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int c = 0; c < 64; c++) asm volatile("" : "+r"(x[c]));
            }
            const float* kf = sh.kf + k * (TI_KEYS / 16) + half * 4;
            const float* vfs = sh.vf + k * (TI_KEYS / 16);
            float mx = -INFINITY;
#pragma unroll
            for (int c = 0; c < 64; c++) {
                float y = __uint_as_float(x[c]) * (f0 * kf[c / 16]);
                if (a.softcap > 0.0f) y = a.softcap * tanhf(y / a.softcap) * PT_LOG2E;
                x[c] = __float_as_uint(y);
            }
            if (lo + k * TI_KEYS + TI_KEYS - 1 > min(pos_first, k1 - 1) || (a.window > 0 && lo + k * TI_KEYS < pos_last - a.window + 1)) {
#pragma unroll
                for (int c = 0; c < 64; c++)
                    if (key0 + c > key_hi || key0 + c < key_lo) x[c] = 0xff800000u;
            }
#pragma unroll
            for (int c = 0; c < 64; c++) mx = fmaxf(mx, __uint_as_float(x[c]));
            sh.top[slot][half][row] = mx;
            ti_soft_sync();                                           // .. and both halves have read S
            mx = fmaxf(mx, sh.top[slot][half ^ 1][row]);
            if (I8) {
#pragma unroll
                for (int g = 0; g < TI_KEYS / 16; g++) vmax = fmaxf(vmax, vfs[g]);
            } else vmax = 1.0f;
            // the step's value factors relative to a power of two
            const float vref = fminf(fmaxf(__uint_as_float(__float_as_uint(vmax) & 0x7f800000u), 0x1p-100f), 0x1p100f), ivref = 1.0f / vref;
            const float m_new = fmaxf(m, mx), base = m_new == -INFINITY ? 0.0f : m_new - PT_SHIFT;
            const float alpha = m == m_new ? 1.0f : ti_exp2(m - m_new);
            m = m_new;
            float sum = 0.0f;
            if (ok) {
#pragma unroll
                for (int g = 0; g < 4; g++) {                         // 16 keys at a time: 8 words of h, 8 of l
                    unsigned h[8], w[8];
                    const float vr = I8 ? vfs[half * 4 + g] * ivref : 1.0f;
#pragma unroll
                    for (int c = 0; c < 16; c += 2) {
                        float p0 = ti_exp2(__uint_as_float(x[g * 16 + c]) - base), p1 = ti_exp2(__uint_as_float(x[g * 16 + c + 1]) - base);
                        sum += p0 + p1;
                        if (I8) {                                     // a weight of zero stays one beside a factor that is NaN
                            p0 = p0 == 0.0f ? 0.0f : p0 * vr;
                            p1 = p1 == 0.0f ? 0.0f : p1 * vr;
                        }
                        pt_cut(p0, p1, h[c / 2], w[c / 2]);
                    }
                    ti_store8(tmem + slot * 128 + lanes + half * 32 + g * 8, h);
                    ti_store8(tmem + slot * 128 + lanes + 64 + half * 32 + g * 8, w);
                }
                asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                pg_fence_before();
                sg_arrive(pg_smem(&sh.p_full[slot]));
            }
            l = fmaf(l, alpha, sum);
            if (k > 0) add(k - 1);
            alpha_prev = alpha; vref_prev = vref;
        }
        if (steps > 0) add(steps - 1);
        sh.sum[half][row] = l;
        ti_soft_sync();
        l = sh.sum[0][row] + sh.sum[1][row];
        if (in && ok) {
            if (n_split > 1) {
                const size_t at = ((size_t)blockIdx.x * a.G + kvh) * TI_ROWS + row;
                float* o = a.part + at * a.dv + c_first;
#pragma unroll
                for (int c = 0; c < TI_D / 2; c += 4)
                    if (c < cols) *(float4*)(o + c) = make_float4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]);
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
                    if (c < cols) *(float4*)(o + c) = make_float4(acc[c] * f, acc[c + 1] * f, acc[c + 2] * f, acc[c + 3] * f);
            }
        }
    }
    pg_fence_before();
    __syncthreads();
    if (warp == 11) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
    if (tid == 0 && sh.fail) {
        if (err_dev) atomicExch(err_dev, 5u);
        if (err_host) { *(volatile unsigned*)err_host = 5u; __threadfence_system(); }
    }
}
