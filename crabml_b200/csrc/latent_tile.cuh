// latent_tile.cuh -- attention over pages of latent rows, expanded: many new tokens of a sequence.  Included by latent_attn.cu behind the absorbed form.
//
// latent_expand_kernel makes the keys U_h c and values V_h c of 256 cached rows and a run of heads: one product of 256 x (dim + vdim) x rank for each head on tcgen05.mma, the rows staying in
// shared memory for all heads.  The results go to images, f16 in the order of the 128-byte swizzle, which bulk copies bring back as they are.  r, which all heads share, is read from the pages.
// 4000 rows, 16 heads of 128 and 128, rank 512: 25 us on 128 SMs (16.8 GFLOP, 0.67 PFLOP/s with the rows' way in and the last block's way out), 8000 37.
//
// latent_tile_kernel: a CTA takes 256 tokens of a head, as two tiles of 128 rows, over the keys that they see, 128 at a time:
//   S = Q K^T (128 x 128 x (dim + rest)), P = exp2(S f - base) as f16 written over S in TMEM, O += P V in TMEM
// The two tiles alternate: while the 256 threads of one make its weights, two a row, the tensor core multiplies for the other.  (With a thread a row a step's 128 scores were a chain of
// 4500 cycles for the one warp a scheduler that a tile had: 4000 tokens of 16 heads took 147 us.)  TMEM holds both S and both O (512 columns), shared memory
// Q (96 KB) and a ring of 16 KB blocks of keys and values (128 KB).
// Now that prompt's call takes 131 us (98.7 GFLOP with its keys and values, 0.75 PFLOP/s); 8000 tokens about 370 (0.93 PFLOP/s).  A step takes 2.7 us, 5100 cycles, whether both tiles have it or one: what
// bounds it is a tile's chain (scores, their way to registers, the largest, the barrier behind it, exponentials, the way back, values, and only then the next scores, since P lies over S).  The step's
// products, fed by shared memory as fast as it can (S reads 8 KB for each 64 cycles of the tensor core), would take 2560 cycles.  Then 7 us of start and end for each item.  base lags: a row's sums are scaled only when a score is TL_LAG above it (sums in TMEM would have to be read and written
// back), and then it goes TL_SHIFT below that score.  So weights reach 2^TL_LAG, which f16 holds, and the largest one is 2^TL_SHIFT at least: those beside it keep f16's 11 bits down to 2^-21 of it.  (With the
// largest at 1 the tail of 32000 equal keys, each 2^-22 of one that stands out, came out in steps of 2^-24: off by 4e-4 of the result.)
// Warps 0-7 and 8-15 the rows of the two tiles, 16 the copies, 17 the products, 18 says what has come.  Every wait is bounded; where one ran out all roles run to their ends and the host reports it.
#pragma once
#include <cuda.h>

#define TL_ROWS 128
#define TL_KEYS 128
#define TL_HALF (TL_KEYS / 2)
#define TL_SOFT 16                            // warps that make weights
#define TL_THREADS (TL_SOFT * 32 + 128)
// 640 threads of 96 registers at launch are 512 of 104 and 128 of 64 afterwards: 64 scores stay in registers
#define TL_REGS 96
#define TL_REGS_SOFT 104
#define TL_REGS_REST 64
static_assert(TL_SOFT * 32 * TL_REGS_SOFT + 128 * TL_REGS_REST <= TL_THREADS * TL_REGS, "more registers than the block was launched with");
#define TL_BLOCK 16384                        // 128 rows of 64 f16 under the 128-byte swizzle
#define TL_SLOTS 8
#define TL_GROUPS 8                           // barriers of the ring: a step's keys, or its values (a wait costs the warp that issues the products 150 to 200 cycles, one for each block 1000 a step)
#define TL_QBLOCKS 3                          // of a row of Q: dim in two, rest in one
#define TL_SMEM ((2 * TL_QBLOCKS + TL_SLOTS) * TL_BLOCK + 1024)
#define TL_LAG 15.0f
#define TL_SHIFT 7.0f
#define TL_O 256                              // TMEM columns: S (and P) of the tiles at 0 and 128, O behind
#define TL_DIM 128                            // largest dim and vdim

struct TlArgs {
    LrArgs a;
    uint8_t *k_image, *v_image;               // [key tile][head of this launch][block]
    int head0, heads, key_tiles, piece;       // piece: steps, about, of what an item is cut into; 0: none is cut
    float* part;                              // sums of pieces [piece][head][2 TL_ROWS][vdim]
    float2* ml;                               // [piece][head][2 TL_ROWS]: base, sum of weights
};
// keys count from a multiple of 128, so that a tile is whole pages
__host__ __device__ __forceinline__ void tl_range(const PgSeq& s, const LrArgs& a, int* from, int* to) {
    lr_range(s, a, from, to);
    *from &= ~(TL_KEYS - 1);
}
__host__ __device__ __forceinline__ int tl_key_tiles(const PgSeq& s, const LrArgs& a) {
    if (s.count <= a.most) return 0;
    int from, to;
    tl_range(s, a, &from, &to);
    return (to - from + TL_KEYS - 1) / TL_KEYS;
}
__host__ __device__ __forceinline__ int tl_items(const PgSeq& s, const LrArgs& a) { return s.count <= a.most ? 0 : (s.count + 2 * TL_ROWS - 1) / (2 * TL_ROWS); }
// steps of an item's two tiles: keys that one of its rows sees, from `lo` for both
__host__ __device__ __forceinline__ void tl_steps(const PgSeq& s, const LrArgs& a, int row0, int* lo, int steps[2]) {
    int from, to;
    tl_range(s, a, &from, &to);
    const int first = a.window > 0 ? (s.pos0 + row0 - a.window + 1) & ~(TL_KEYS - 1) : from;
    *lo = first > from ? first : from;
    for (int i = 0; i < 2; i++) {
        const int end = s.count < row0 + (i + 1) * TL_ROWS ? s.count : row0 + (i + 1) * TL_ROWS;
        steps[i] = row0 + i * TL_ROWS < s.count ? (s.pos0 + end - *lo + TL_KEYS - 1) / TL_KEYS : 0;
    }
}
// pieces of each item of a sequence: as its last one, which sees most
__host__ __device__ __forceinline__ int tl_pieces(const PgSeq& s, const TlArgs& t) {
    if (!t.piece || s.count <= t.a.most) return 1;
    int lo, steps[2];
    tl_steps(s, t.a, (tl_items(s, t.a) - 1) * 2 * TL_ROWS, &lo, steps);
    const int most = steps[0] > steps[1] ? steps[0] : steps[1], n = most / t.piece;
    return n > 1 ? n : 1;
}
// the place of number n in the sequences' counts: every lane gets the sequence and what is left of n
template <class Count>
__device__ __forceinline__ int tl_find(const LrArgs& a, int n, Count count, int* rest) {
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
__device__ __forceinline__ unsigned tl_at(int row, int chunk) { return (unsigned)(row * 128 + ((chunk ^ (row & 7)) << 4)); }      // chunk of 8 numbers of a row of a block
// waits that end after some seconds, or when another one has: they look whether it has every time (asked to hold the thread for up to 2 us a look, it came back later: 136 us instead of 131)
__device__ __forceinline__ bool tl_wait(unsigned bar, unsigned parity, int* fail) { return sg_wait<1>(bar, parity, fail); }
__device__ __forceinline__ bool tl_wait_warp(unsigned bar, unsigned parity, int* fail) { return __all_sync(0xffffffffu, tl_wait(bar, parity, fail)); }
__device__ __forceinline__ void tl_report(int fail, unsigned* err_dev, unsigned* err_host) {
    if (threadIdx.x == 0 && fail) {
        if (err_dev) atomicExch(err_dev, 5u);
        if (err_host) { *(volatile unsigned*)err_host = 5u; __threadfence_system(); }
    }
}
// The pages that hold keys key0 .. key0 + 127 of a sequence, those behind its last token left out: lane i has the i-th one's number (a look-up by each copy's thread took 700 cycles of it), a
// copy brings 64 columns of one
__device__ __forceinline__ int tl_look_up(const LrArgs& a, int seq, int key0, int to) {
    const int key = key0 + (int)(threadIdx.x & 31) * a.page;
    return (int)(threadIdx.x & 31) < TL_KEYS / a.page && key < to ? a.table[(int64_t)seq * a.table_cols + (key >> a.shift)] : 0;
}

// ---- keys and values of 128 rows ------------------------------------------------------------------------------------------------------------------------
// A pair of SMs takes two tiles of 128 keys, which stay in shared memory for all heads of its run, and each of them half of a step's weights: 64 columns of U_h the even one, of V_h the other.  (A
// tile by one SM needs all of them from L2, 32 KB for 512 cycles of products, two under way: 32 us for 4000 keys of 16 heads.)
#define TE_THREADS 384
#define TE_ABLOCKS (LT_RANK / 64)
#define TE_STAGES 4
#define TE_STAGE (TL_DIM * 128)               // 64 columns of U_h or V_h
#define TE_SMEM (TE_ABLOCKS * TL_BLOCK + TE_STAGES * TE_STAGE + 2 * TL_BLOCK + 1024)      // the rows, weights, two blocks of results
struct TeShared {
    unsigned long long a_full[TE_ABLOCKS], full[TE_STAGES], empty[TE_STAGES], acc_full[2], acc_empty[2], drained;
    unsigned tmem_base;
    int fail;
};
// (relaxed: nothing that this thread has written is read behind the barrier, and a release to the cluster waits 1300 cycles for what it has under way)
__device__ __forceinline__ void te_expect(unsigned bar, unsigned bytes) { asm volatile("mbarrier.arrive.expect_tx.relaxed.cluster.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory"); }
__device__ __forceinline__ void te_tma_page(unsigned dst, const void* tmap, unsigned bar, int x, int page) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(tmap), "r"(bar), "r"(x), "r"(0), "r"(page) : "memory");
}
__device__ __forceinline__ void te_sync(int which) { asm volatile("bar.sync %0, 128;" ::"r"(1 + which) : "memory"); }      // the four warps of a block
// grid (key tiles, up to a whole pair, runs of heads)
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(TE_THREADS, 1) latent_expand_kernel(const __grid_constant__ CUtensorMap map_rows, const __grid_constant__ CUtensorMap map_uk,
                                                                                               const __grid_constant__ CUtensorMap map_uv, const __grid_constant__ TlArgs t, unsigned* err_dev, unsigned* err_host) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(1024) uint8_t tl_raw[];
    __shared__ TeShared sh;
    const LrArgs& a = t.a;
    uint8_t *as = (uint8_t*)(((uintptr_t)tl_raw + 1023) & ~(uintptr_t)1023), *bs = as + TE_ABLOCKS * TL_BLOCK;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, rank = (int)cg::this_cluster().block_rank(), wide = max(a.dim, a.vdim), blocks = (a.rank + 63) >> 6;
    const int h0 = (int)((int64_t)t.heads * blockIdx.y / gridDim.y), h1 = (int)((int64_t)t.heads * (blockIdx.y + 1) / gridDim.y);
    if (tid == 0) {
        for (int i = 0; i < TE_ABLOCKS; i++) pg_mbar_init(pg_smem(&sh.a_full[i]), 2);
        for (int i = 0; i < TE_STAGES; i++) { pg_mbar_init(pg_smem(&sh.full[i]), 1); pg_mbar_init(pg_smem(&sh.empty[i]), 1); }
        for (int i = 0; i < 2; i++) { pg_mbar_init(pg_smem(&sh.acc_full[i]), 1); pg_mbar_init(pg_smem(&sh.acc_empty[i]), 16); }
        pg_mbar_init(pg_smem(&sh.drained), 1);
        sh.fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 2) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(pg_smem(&sh.tmem_base)), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    pg_fence_before();
    __syncthreads();
    cg::this_cluster().sync();
    pg_fence_after();
    const unsigned tmem = sh.tmem_base;
    pdl_enter();
    int kt = 0, from, to;
    const int found = (int)blockIdx.x < t.key_tiles ? tl_find(a, blockIdx.x, [&](const PgSeq& s) { return tl_key_tiles(s, a); }, &kt) : -1, seq = max(0, found);
    tl_range(a.seqs[seq], a, &from, &to);
    const int key0 = from + kt * TL_KEYS;
    if (found < 0) to = key0;                                         // the second CTA of the last pair may have no keys
    if (warp == 0) {
        const int pages = found < 0 ? 0 : (min(TL_KEYS, to - key0) + a.page - 1) >> a.shift, mine = tl_look_up(a, seq, key0, to);
        for (int b = 0; b < blocks; b++) {
            const unsigned bar = pg_even(pg_smem(&sh.a_full[b]));
            if (lane == 0) te_expect(bar, (unsigned)(pages * a.page * 128));
            __syncwarp();
            for (int i = 0; i < pages; i++) {
                const int page = __shfl_sync(0xffffffffu, mine, i);
                if (pg_elect()) te_tma_page(pg_smem(as + b * TL_BLOCK) + i * a.page * 128, &map_rows, bar, b * 64, page);
            }
        }
        __syncwarp();
        if (lane == 0) {
            unsigned g = 0;
            bool ok = true;
            for (int h = h0; h < h1 && ok; h++)
                for (int b = 0; b < blocks; b++, g++) {
                    const unsigned slot = g % TE_STAGES, own = pg_smem(&sh.full[slot]);
                    if (!(ok = tl_wait(pg_smem(&sh.empty[slot]), ((g / TE_STAGES) & 1u) ^ 1u, &sh.fail))) break;
                    if (rank == 0) pg_mbar_expect_tx(own, (unsigned)wide * 256);
                    pg_tma_load_2d_pair(pg_smem(bs + slot * TE_STAGE), rank ? &map_uv : &map_uk, pg_even(own), b * 64, (t.head0 + h) * (rank ? a.vdim : a.dim));
                }
            int never = 0;                                            // no copy is under way when the CTAs end (the even one sees those of both), and no arrival
            if (rank == 0)
                for (int b = 0; b < blocks; b++) tl_wait(pg_smem(&sh.a_full[b]), 0, &never);
            for (unsigned i = g > TE_STAGES ? g - TE_STAGES : 0; i < g; i++) {
                if (rank == 0) tl_wait(pg_smem(&sh.full[i % TE_STAGES]), (i / TE_STAGES) & 1u, &never);
                tl_wait(pg_smem(&sh.empty[i % TE_STAGES]), (i / TE_STAGES) & 1u, &never);
            }
            if (!ok || never)                                         // something did not come in time: a while for whatever is still to
                for (int i = 0; i < 1000; i++) __nanosleep(1000);
        }
        __syncwarp();
    } else if (warp == 1) {
        int never = 0;                                                // nothing is in flight when the TMEM is given back
        if (rank == 0) {
            const unsigned idesc = pg_instr_desc(256, 2 * wide);
            const uint64_t a_desc = pg_smem_desc(pg_smem(as)), b_desc = pg_smem_desc(pg_smem(bs));
            unsigned slot = 0, phase = 0;
            bool ok = true;
            for (int h = h0; h < h1 && ok; h++) {
                const unsigned n = (unsigned)(h - h0), acc = tmem + (n & 1u) * 256;
                if (!(ok = tl_wait_warp(pg_smem(&sh.acc_empty[n & 1u]), ((n >> 1) & 1u) ^ 1u, &sh.fail))) break;
                for (int b = 0; b < blocks; b++) {
                    if (!(ok = (h > h0 || tl_wait_warp(pg_smem(&sh.a_full[b]), 0, &sh.fail)) && tl_wait_warp(pg_smem(&sh.full[slot]), phase, &sh.fail))) break;
                    pg_fence_after();
                    const uint64_t x = a_desc + b * (TL_BLOCK >> 4), y = b_desc + slot * (TE_STAGE >> 4);
                    const int steps = min(4, (a.rank - b * 64) >> 4);
                    if (pg_elect()) {
#pragma unroll
                        for (int kk = 0; kk < 4; kk++)
                            if (kk < steps) pg_umma_f16_pair(acc, x + 2 * kk, y + 2 * kk, idesc, b > 0 || kk > 0);
                        pg_umma_commit_pair(pg_smem(&sh.empty[slot]));
                        if (b == blocks - 1) pg_umma_commit_pair(pg_smem(&sh.acc_full[n & 1u]));
                    }
                    __syncwarp();
                    if (++slot == TE_STAGES) { slot = 0; phase ^= 1u; }
                }
            }
            if (pg_elect()) pg_umma_commit_pair(pg_smem(&sh.drained));
            __syncwarp();
        }
        tl_wait_warp(pg_smem(&sh.drained), 0, &never);
    } else if (warp >= 4) {
        // a lane a key; four warps the keys' blocks of 64 columns, the others the values': by way of shared memory, from where a block goes to its image as a whole.  (Stored by each lane 16 bytes
        // at a time, 128 apart, a head took 5500 cycles, its products 4100)
        const int q = warp & 3, row = q * 32 + lane, is_v = (warp - 4) >> 2, d = is_v ? a.vdim : a.dim;
        const bool in = key0 + row < to;
        uint8_t* stage = bs + TE_STAGES * TE_STAGE + is_v * TL_BLOCK;
        lt_rounds(h0, h1, [&](int h) { return tl_wait_warp(pg_smem(&sh.acc_full[(h - h0) & 1]), (unsigned)(h - h0) >> 1 & 1u, &sh.fail); }, [&](int h, bool ok) {
            const unsigned n = (unsigned)(h - h0);
            pg_fence_after();
            uint8_t* image = (is_v ? t.v_image : t.k_image) + ((size_t)blockIdx.x * t.heads + h) * ((d + 63) >> 6) * TL_BLOCK;
#pragma unroll 1
            for (int c = 0; c < d; c += 64) {
                unsigned v[4][16];
#pragma unroll
                for (int x = 0; x < 4; x++)
                    if (ok && c + x * 16 < d) sg_tmem16(tmem + (n & 1u) * 256 + ((unsigned)(q * 32) << 16) + is_v * wide + c + x * 16, v[x]);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                if (row == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // the block before has left
                te_sync(is_v);
#pragma unroll
                for (int x = 0; x < 4; x++) {
#pragma unroll
                    for (int j = 0; j < 16; j++) asm volatile("" : "+r"(v[x][j]));
                    if (!ok || c + x * 16 >= d) continue;
                    unsigned w[8], wild = 0;
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        w[j] = lt_pack(__uint_as_float(v[x][2 * j]), __uint_as_float(v[x][2 * j + 1]));
                        wild |= (w[j] & 0x7c007c00u) + 0x04000400u;   // the exponent of an infinity or a NaN carries into the sign's place
                    }
                    if (wild & 0x80008000u) {
                        // beyond f16; or a cached row that is not finite, which makes all of its keys and values so: a NaN in a key reaches the queries that see it, a zero in its value no one
#pragma unroll
                        for (int j = 0; j < 16; j++)
                            if (!(fabsf(__uint_as_float(v[x][j])) < INFINITY)) v[x][j] = is_v ? 0u : 0x7fc00000u;
#pragma unroll
                        for (int j = 0; j < 8; j++) w[j] = ht_pack_f16(__uint_as_float(v[x][2 * j]), __uint_as_float(v[x][2 * j + 1]));
                    }
                    if (is_v && !in) {
#pragma unroll
                        for (int j = 0; j < 8; j++) w[j] = 0u;
                    }
                    *(uint4*)(stage + tl_at(row, 2 * x)) = make_uint4(w[0], w[1], w[2], w[3]);
                    *(uint4*)(stage + tl_at(row, 2 * x + 1)) = make_uint4(w[4], w[5], w[6], w[7]);
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                te_sync(is_v);
                if (row == 0 && ok && (int)blockIdx.x < t.key_tiles) {
                    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(image + (c >> 6) * TL_BLOCK), "r"(pg_smem(stage)), "r"(TL_BLOCK) : "memory");
                    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
                }
            }
            pg_fence_before();
            __syncwarp();
            if (lane == 0) pg_arrive_relaxed(pg_even(pg_smem(&sh.acc_empty[n & 1u])));
        });
        if (row == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    pg_fence_before();
    __syncthreads();
    cg::this_cluster().sync();
    if (warp == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
    tl_report(sh.fail, err_dev, err_host);
}

// ---- attention -----------------------------------------------------------------------------------------------------------------------------------------------
struct TlShared {
    unsigned long long q_full, full[TL_GROUPS], empty[TL_GROUPS], s_full[2], p_full[2], o_full[2], drained;
    unsigned tmem_base;
    int fail;
    float top[2][TL_ROWS];                    // what the two threads of a row tell each other
};
// the 256 threads of a tile
__device__ __forceinline__ void tl_sync(int bar) { asm volatile("bar.sync %0, %1;" ::"r"(bar), "n"(TL_SOFT * 16) : "memory"); }
__device__ __forceinline__ bool tl_sync_or(int bar, bool x) {
    unsigned r;
    asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbar.red.or.pred q, %2, %3, p;\nselp.u32 %0, 1, 0, q;\n}\n" : "=r"(r) : "r"((unsigned)x), "r"(bar), "n"(TL_SOFT * 16) : "memory");
    return r;
}
__device__ __forceinline__ void tl_tma_page(unsigned dst, const void* tmap, unsigned bar, int x, int page) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst), "l"(tmap), "r"(bar), "r"(x), "r"(0), "r"(page) : "memory");
}
// B whose rows are the sum's index and whose columns (64 of them in 128 bytes) are the result's: blocks of 64 columns `block` bytes apart, groups of 8 rows 1024 bytes
__device__ __forceinline__ uint64_t tl_desc_mn(unsigned addr, unsigned block) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)(block >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ void tl_umma_ts(unsigned d, unsigned a, uint64_t b, unsigned idesc, unsigned accumulate) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tl_store8(unsigned addr, const unsigned* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]),
                 "r"(v[7]) : "memory");
}
typedef unsigned long long tl_f2;             // pairs of 32-bit numbers in one instruction
__device__ __forceinline__ tl_f2 tl_two(float x, float y) {
    tl_f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 tl_one(tl_f2 v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ tl_f2 tl_fma2(tl_f2 a, tl_f2 b, tl_f2 c) {
    tl_f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ tl_f2 tl_add2(tl_f2 a, tl_f2 b) {
    tl_f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ tl_f2 tl_mul2(tl_f2 a, tl_f2 b) {
    tl_f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// the largest of three, NaN if one of them is: a row that sees a score which is none has no result
__device__ __forceinline__ float tl_max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// whether 8 numbers of a query at a time, from the `from`-th on, every `step`-th, hold one that is not finite.  A row all of whose scores are -infinity has sums of 0, which a sink makes a result of 0:
// right where its keys make them so, but a query that is not finite has the result NaN
__device__ __forceinline__ bool tl_wild(const LrArgs& a, int64_t token, int head, int from, int step) {
    const int n = (a.dim + a.rest) / 8;
    const uint4* q = (const uint4*)(a.q + (token * a.H + head) * (a.dim + a.rest));
    unsigned wild = 0;
#pragma unroll 1
    for (int i = from; i < n; i += step) {
        const uint4 v = q[i];
        wild |= ((v.x & 0x7c007c00u) + 0x04000400u) | ((v.y & 0x7c007c00u) + 0x04000400u) | ((v.z & 0x7c007c00u) + 0x04000400u) | ((v.w & 0x7c007c00u) + 0x04000400u);
    }
    return wild & 0x80008000u;
}
// grid: pieces of items x heads, heads fastest
__global__ void __launch_bounds__(TL_THREADS, 1) latent_tile_kernel(const __grid_constant__ CUtensorMap map_rows, const __grid_constant__ CUtensorMap map_q, const __grid_constant__ TlArgs t, unsigned* err_dev,
                                                                    unsigned* err_host) {
    extern __shared__ __align__(1024) uint8_t tl_raw[];
    __shared__ TlShared sh;
    const LrArgs& a = t.a;
    uint8_t *qs = (uint8_t*)(((uintptr_t)tl_raw + 1023) & ~(uintptr_t)1023), *ring = qs + 2 * TL_QBLOCKS * TL_BLOCK;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, item = (int)(blockIdx.x / (unsigned)t.heads), head_at = (int)(blockIdx.x - (unsigned)item * t.heads), head = t.head0 + head_at;
    const int nb = (a.dim + 63) >> 6, rb = a.rest ? 1 : 0, vb = (a.vdim + 63) >> 6;      // blocks of keys, of r, of values
    if (tid == 0) {
        pg_mbar_init(pg_smem(&sh.q_full), 1);
        for (int i = 0; i < TL_GROUPS; i++) { pg_mbar_init(pg_smem(&sh.full[i]), 1); pg_mbar_init(pg_smem(&sh.empty[i]), 1); }
        for (int i = 0; i < 2; i++) { pg_mbar_init(pg_smem(&sh.s_full[i]), 1); pg_mbar_init(pg_smem(&sh.p_full[i]), TL_SOFT / 2 + 1); pg_mbar_init(pg_smem(&sh.o_full[i]), 1); }
        pg_mbar_init(pg_smem(&sh.drained), 1);
        sh.fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == TL_SOFT + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(pg_smem(&sh.tmem_base)), "n"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    pg_fence_before();
    __syncthreads();
    pg_fence_after();
    const unsigned tmem = sh.tmem_base;
    pdl_enter();
    int rest;
    const int seq = max(0, tl_find(a, item, [&](const PgSeq& s) { return tl_items(s, a) * tl_pieces(s, t); }, &rest));
    const PgSeq s = a.seqs[seq];
    const int pieces = tl_pieces(s, t), piece = rest % pieces, row0 = (tl_items(s, a) - 1 - rest / pieces) * 2 * TL_ROWS;      // late rows, which see most, first
    int from, to, before = 0, slot = 0, lo, steps_of[2];
    tl_range(s, a, &from, &to);
    for (int x = lane; x < seq; x += 32) {
        const PgSeq o = a.seqs[x];
        before += tl_key_tiles(o, a);
        if (t.piece) { const int n = tl_pieces(o, t); slot += n > 1 ? n * tl_items(o, a) : 0; }
    }
    before = warp_sum_i(before);
    slot = warp_sum_i(slot) + rest;
    tl_steps(s, a, row0, &lo, steps_of);
    // this piece's steps of them
    const int each = (max(steps_of[0], steps_of[1]) + pieces - 1) / pieces, off = piece * each, steps0 = max(0, min(steps_of[0] - off, each)), steps1 = max(0, min(steps_of[1] - off, each));
    const int steps = max(steps0, steps1), kt0 = before + (lo - from) / TL_KEYS + off, per = nb + rb + vb;
    lo += off * TL_KEYS;
    if (warp >= TL_SOFT) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(TL_REGS_REST));
        if (warp == TL_SOFT) {
            // ===== copies: Q, then the blocks of each step =====
            const int width = a.dim + a.rest;
            if (pg_elect()) {
                pg_mbar_expect_tx(pg_smem(&sh.q_full), (unsigned)(2 * (nb + rb) * TL_BLOCK));
                for (int i = 0; i < 2; i++)
                    for (int b = 0; b < nb + rb; b++)
                        pg_tma_load_2d(pg_smem(qs + (i * TL_QBLOCKS + b) * TL_BLOCK), &map_q, pg_smem(&sh.q_full), head * width + (b < nb ? b * 64 : a.dim), s.first + row0 + i * TL_ROWS);
            }
            __syncwarp();
            unsigned g = 0, groups = 0;
            bool ok = true;
            int mine = tl_look_up(a, seq, lo, to);
            for (int k = 0; k < steps && ok; k++) {
                const size_t image = (size_t)(kt0 + k) * t.heads + head_at;
                const int key0 = lo + k * TL_KEYS, pages = (min(TL_KEYS, to - key0) + a.page - 1) >> a.shift, those = mine;
                if (k + 1 < steps) mine = tl_look_up(a, seq, key0 + TL_KEYS, to);
                for (int b = 0; b < per; b++, g++) {
                    const unsigned at = pg_smem(ring + g % TL_SLOTS * TL_BLOCK), full = pg_smem(&sh.full[(2 * k + (b >= nb + rb)) % TL_GROUPS]);
                    if (g >= TL_SLOTS) {                              // the group of the block that was here is through
                        const unsigned was = g - TL_SLOTS, of = 2 * (was / per) + (was % per >= (unsigned)(nb + rb));
                        if (!(ok = tl_wait_warp(pg_smem(&sh.empty[of % TL_GROUPS]), (of / TL_GROUPS) & 1u, &sh.fail))) break;
                    }
                    if (b == 0 || b == nb + rb) {
                        if (pg_elect()) pg_mbar_expect_tx(full, b ? (unsigned)(vb * TL_BLOCK) : (unsigned)(nb * TL_BLOCK + rb * pages * a.page * 128));
                        __syncwarp();
                        groups++;
                    }
                    if (b >= nb && b < nb + rb)
                        for (int i = 0; i < pages; i++) {
                            const int page = __shfl_sync(0xffffffffu, those, i);
                            if (pg_elect()) tl_tma_page(at + i * a.page * 128, &map_rows, full, a.rank, page);
                        }
                    else if (pg_elect()) {
                        const uint8_t* src = b < nb ? t.k_image + (image * nb + b) * TL_BLOCK : t.v_image + (image * vb + b - nb - rb) * TL_BLOCK;
                        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(at), "l"(src), "r"(TL_BLOCK), "r"(full) : "memory");
                    }
                    __syncwarp();
                }
            }
            // no copy is under way when the CTA ends.  Where a wait ran out in the midst of a group, what it lacks never comes: a while for what does
            int never = 0;
            if (ok) for (unsigned i = groups > TL_GROUPS ? groups - TL_GROUPS : 0; i < groups; i++) tl_wait_warp(pg_smem(&sh.full[i % TL_GROUPS]), (i / TL_GROUPS) & 1u, &never);
            else for (int i = 0; i < 1000; i++) __nanosleep(1000);
            tl_wait_warp(pg_smem(&sh.q_full), 0, &never);
        } else if (warp == TL_SOFT + 1) {
            // ===== products =====
            const unsigned idesc_s = pg_instr_desc(128, TL_KEYS), idesc_o = pg_instr_desc(128, a.vdim) | 1u << 16, idesc_lo = pg_instr_desc(128, 64) | 1u << 16, idesc_hi = pg_instr_desc(128, a.vdim - 64) | 1u << 16;
            const uint64_t q_desc = pg_smem_desc(pg_smem(qs)), ring_desc = pg_smem_desc(pg_smem(ring)), v_desc = tl_desc_mn(pg_smem(ring), TL_BLOCK);
            bool ok = tl_wait_warp(pg_smem(&sh.q_full), 0, &sh.fail);
            auto free_group = [&](int g) {
                if (pg_elect()) pg_umma_commit(pg_smem(&sh.empty[g % TL_GROUPS]));
                __syncwarp();
            };
            auto scores = [&](int i, unsigned g) {                   // of tile i against the keys in blocks g ..
                const unsigned to_s = tmem + i * 128;
                for (int b = 0; b < nb + rb; b++, g++) {
                    const uint64_t x = q_desc + (unsigned)(i * TL_QBLOCKS + b) * (TL_BLOCK >> 4), y = ring_desc + (g % TL_SLOTS) * (TL_BLOCK >> 4);
                    const int n = min(4, (b < nb ? a.dim - b * 64 : a.rest) >> 4);
                    if (pg_elect()) {
#pragma unroll
                        for (int kk = 0; kk < 4; kk++)
                            if (kk < n) pg_umma_f16(to_s, x + 2 * kk, y + 2 * kk, idesc_s, b > 0 || kk > 0);
                        if (b == nb + rb - 1) pg_umma_commit(pg_smem(&sh.s_full[i]));
                    }
                    __syncwarp();
                }
            };
            auto values = [&](int i, unsigned g, int k) {
                const unsigned to_o = tmem + TL_O + i * 128, p = tmem + i * 128;
                const uint64_t v0 = v_desc + (g % TL_SLOTS) * (TL_BLOCK >> 4), v1 = v_desc + ((g + 1) % TL_SLOTS) * (TL_BLOCK >> 4);
                const bool apart = vb == 2 && (g + 1) % TL_SLOTS == 0;       // the ring's blocks lie side by side, but for the last and the first
                if (pg_elect()) {
                    if (!apart) {
#pragma unroll
                        for (int kk = 0; kk < TL_KEYS / 16; kk++) tl_umma_ts(to_o, p + kk * 8, v0 + kk * (2048 >> 4), idesc_o, k > 0 || kk > 0);
                    } else {
#pragma unroll
                        for (int kk = 0; kk < TL_KEYS / 16; kk++) {
                            tl_umma_ts(to_o, p + kk * 8, v0 + kk * (2048 >> 4), idesc_lo, k > 0 || kk > 0);
                            tl_umma_ts(to_o + 64, p + kk * 8, v1 + kk * (2048 >> 4), idesc_hi, k > 0 || kk > 0);
                        }
                    }
                    pg_umma_commit(pg_smem(&sh.o_full[i]));
                }
                __syncwarp();
            };
            if (ok && steps > 0) {
                ok = tl_wait_warp(pg_smem(&sh.full[0]), 0, &sh.fail);
                pg_fence_after();
                if (ok && steps0 > 0) scores(0, 0);
                if (ok && steps1 > 0) scores(1, 0);
                free_group(0);
            }
            for (int k = 0; k < steps && ok; k++) {
                const unsigned gv = (unsigned)(k * per + nb + rb), gk = (unsigned)((k + 1) * per);
#pragma unroll 1
                for (int i = 0; i < 2 && ok; i++) {
                    const int mine = i ? steps1 : steps0;
                    if (k < mine) {
                        if (!(ok = tl_wait_warp(pg_smem(&sh.p_full[i]), k & 1, &sh.fail))) break;      // weights, values and the next keys
                        pg_fence_after();
                        values(i, gv, k);
                    }
                    if (i == 1) free_group(2 * k + 1);
                    if (k + 1 < mine) scores(i, gk);
                }
                if (ok && k + 1 < steps) free_group(2 * k + 2);
            }
            int never = 0;                                            // nothing of this CTA is in flight when its TMEM is given back
            if (pg_elect()) pg_umma_commit(pg_smem(&sh.drained));
            __syncwarp();
            tl_wait_warp(pg_smem(&sh.drained), 0, &never);
        } else if (warp == TL_SOFT + 2) {
            // ===== a step's values and the next one's keys are there: said where the products wait for the weights, so that they wait once (200 to 350 cycles each, among 16 busy warps) =====
            bool ok = true;
            for (int k = 0; k < steps && ok; k++) {
                ok = tl_wait_warp(pg_smem(&sh.full[(2 * k + 1) % TL_GROUPS]), ((2 * k + 1) / TL_GROUPS) & 1, &sh.fail);
                if (ok && k + 1 < steps) ok = tl_wait_warp(pg_smem(&sh.full[(2 * k + 2) % TL_GROUPS]), ((2 * k + 2) / TL_GROUPS) & 1, &sh.fail);
                // (narrow heads leave the ring room for two steps: once a step, when the one before is through)
                if (k < steps0) { if (ok && k > 0) ok = tl_wait_warp(pg_smem(&sh.p_full[0]), (k - 1) & 1, &sh.fail); sg_arrive(pg_smem(&sh.p_full[0])); }
                if (k < steps1) { if (ok && k > 0) ok = tl_wait_warp(pg_smem(&sh.p_full[1]), (k - 1) & 1, &sh.fail); sg_arrive(pg_smem(&sh.p_full[1])); }
            }
        }
    } else {
        // ===== weights: two threads a row, 64 keys of a step each =====
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(TL_REGS_SOFT));
        const int i = warp >> 3, half = (warp >> 2) & 1, in_tile = (warp & 3) * 32 + lane, row = row0 + i * TL_ROWS + in_tile, mine = i ? steps1 : steps0;
        const int pos = s.pos0 + row, key_lo = a.window > 0 ? pos - a.window + 1 : 0, pos_first = s.pos0 + row0 + i * TL_ROWS, pos_last = s.pos0 + min(s.count, row0 + (i + 1) * TL_ROWS) - 1;
        const unsigned lanes = (unsigned)((warp & 3) * 32) << 16, st = tmem + lanes + i * 128, ot = tmem + lanes + TL_O + i * 128;
        const float f = a.scale * LR_LOG2E;
        float base = -INFINITY, l = 0.0f;
        bool ok = true;
#pragma unroll 1
        for (int k = 0; k < mine; k++) {
            const int key0 = lo + k * TL_KEYS + half * TL_HALF;
            ok = ok && tl_wait_warp(pg_smem(&sh.s_full[i]), k & 1, &sh.fail);
            unsigned x[TL_HALF];
            if (ok) {
                pg_fence_after();
#pragma unroll
                for (int c = 0; c < TL_HALF; c += 16) sg_tmem16(st + half * TL_HALF + c, *(unsigned(*)[16])(x + c));
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int c = 0; c < TL_HALF; c++) asm volatile("" : "+r"(x[c]));
            }
            // x ff are the scores in powers of 2
            float ff = f;
            auto scaled = [&]() {
#pragma unroll
                for (int c = 0; c < TL_HALF; c += 2) {
                    const float2 y = tl_one(tl_mul2(tl_two(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), tl_two(f, f)));
                    x[c] = __float_as_uint(y.x); x[c + 1] = __float_as_uint(y.y);
                }
                ff = 1.0f;
            };
            if (!(f > 0.0f)) scaled();
            if (lo + k * TL_KEYS + TL_KEYS - 1 > pos_first || (a.window > 0 && lo + k * TL_KEYS < pos_last - a.window + 1)) {
                const int c_lo = key_lo - key0, c_hi = pos - key0;
#pragma unroll
                for (int c = 0; c < TL_HALF; c++)
                    if (c > c_hi || c < c_lo) x[c] = 0xff800000u;
            }
            float m0 = __uint_as_float(x[0]), m1 = __uint_as_float(x[1]);
#pragma unroll
            for (int c = 2; c + 3 < TL_HALF; c += 4) { m0 = tl_max3(m0, __uint_as_float(x[c]), __uint_as_float(x[c + 1])); m1 = tl_max3(m1, __uint_as_float(x[c + 2]), __uint_as_float(x[c + 3])); }
            m0 = tl_max3(m0, __uint_as_float(x[TL_HALF - 2]), __uint_as_float(x[TL_HALF - 1]));
            const float mx = tl_max3(m0, m1, m1) * ff;
            // The sums are scaled where a row's base has to follow its largest score; else the halves need not meet.  (Behind this all have read S, too)
            if (tl_sync_or(1 + i, !(mx <= __fadd_rd(base, TL_LAG)))) {      // (rounded down: no weight is above 2^TL_LAG)
                if (half) sh.top[i][in_tile] = mx;
                tl_sync(1 + i);
                if (!half) sh.top[i][in_tile] = tl_max3(mx, sh.top[i][in_tile], mx);
                tl_sync(1 + i);
                const float both = sh.top[i][in_tile];
                float alpha = 1.0f;
                if (base == base && !(both <= __fadd_rd(base, TL_LAG))) {      // (a base that is none stays so: keys behind it that are not seen would hide it)
                    const float was = base;
                    base = __fadd_ru(both, -TL_SHIFT);
                    if (was != -INFINITY) alpha = lt_exp2(was - base);
                }
                if (__any_sync(0xffffffffu, alpha != 1.0f)) {
                    if (k > 0 && ok) {
                        ok = tl_wait_warp(pg_smem(&sh.o_full[i]), (k - 1) & 1, &sh.fail);
                        pg_fence_after();
#pragma unroll 1
                        for (int c = half * 16; c < a.vdim && ok; c += 32) {
                            unsigned v[16];
                            sg_tmem16(ot + c, v);
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                            for (int j = 0; j < 16; j++) {
                                asm volatile("" : "+r"(v[j]));
                                v[j] = __float_as_uint(__uint_as_float(v[j]) * alpha);
                            }
                            tl_store8(ot + c, v); tl_store8(ot + c + 8, v + 8);
                        }
                    }
                    l *= alpha;
                }
            }
            const float minus = base == -INFINITY ? 0.0f : -base;
            // score - base in one multiply-add, whose rest of the largest score's rounding is the same for the whole row; scores from 2^24 on, whose rests of 1 and more could lift a weight out of f16, are
            // rounded first
            if (__any_sync(0xffffffffu, fabsf(minus) >= 16777200.0f) && ff == f) scaled();
            const tl_f2 ff2 = tl_two(ff, ff), minus2 = tl_two(minus, minus);
            tl_f2 sum = 0ull, more = 0ull;
#pragma unroll
            for (int g = 0; g < TL_HALF; g += 16) {
                unsigned w[8];
#pragma unroll
                for (int c = 0; c < 16; c += 2) {
                    const float2 y = tl_one(tl_fma2(tl_two(__uint_as_float(x[g + c]), __uint_as_float(x[g + c + 1])), ff2, minus2));
                    const tl_f2 p = tl_two(lt_exp2(y.x), lt_exp2(y.y));
                    if (c & 2) more = tl_add2(more, p);
                    else sum = tl_add2(sum, p);
                    const float2 z = tl_one(p);
                    w[c / 2] = lt_pack(z.x, z.y);
                }
                if (ok) tl_store8(st + half * (TL_HALF / 2) + g / 2, w);
            }
            asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
            pg_fence_before();
            sg_arrive(pg_smem(&sh.p_full[i]));
            const float2 sums = tl_one(tl_add2(sum, more));
            l += sums.x + sums.y;
        }
        if (mine > 0) {
            tl_sync(1 + i);                                           // the last step's largest scores are read
            if (half) sh.top[i][in_tile] = l;
            tl_sync(1 + i);
            if (!half) sh.top[i][in_tile] += l;
            tl_sync(1 + i);
            l = sh.top[i][in_tile];
        }
        const int64_t at = ((int64_t)slot * t.heads + head_at) * (2 * TL_ROWS) + i * TL_ROWS + in_tile;
        if (pieces > 1 && !half) t.ml[at] = make_float2(base, l);
        if (mine > 0 && ok && (ok = tl_wait_warp(pg_smem(&sh.o_full[i]), (mine - 1) & 1, &sh.fail))) {
            pg_fence_after();
            float g = 1.0f, total = l;
            if (a.sink) {
                const float sk = a.sink[head] * LR_LOG2E, m2 = fmaxf(base, sk);
                g = exp2f(base - m2);
                total = g * l + (sk == -INFINITY ? 0.0f : exp2f(sk - m2));
            }
            const bool none = base != base || (base == -INFINITY && row < s.count && tl_wild(a, s.first + row, head, 0, 1));
            const float by = none ? NAN : g / total;
            uint16_t* out = (uint16_t*)a.out + ((int64_t)(s.first + row) * a.H + head) * a.vdim;
#pragma unroll 1
            for (int c = half * 16; c < a.vdim; c += 32) {
                unsigned v[16], w[8];
                sg_tmem16(ot + c, v);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                for (int j = 0; j < 16; j++) asm volatile("" : "+r"(v[j]));
                if (pieces > 1) {
#pragma unroll
                    for (int j = 0; j < 16; j += 4) *(uint4*)(t.part + at * a.vdim + c + j) = make_uint4(v[j], v[j + 1], v[j + 2], v[j + 3]);
                    continue;
                }
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float u = __uint_as_float(v[2 * j]) * by, z = __uint_as_float(v[2 * j + 1]) * by;
                    w[j] = a.out_bf16 ? ht_pack_bf16(u, z) : ht_pack_f16(u, z);
                }
                if (row < s.count) {
                    *(uint4*)(out + c) = make_uint4(w[0], w[1], w[2], w[3]);
                    *(uint4*)(out + c + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                }
            }
        }
    }
    pg_fence_before();
    __syncthreads();
    if (warp == TL_SOFT + 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
    tl_report(sh.fail, err_dev, err_host);
}

// the pieces of an item's rows: a warp a row and head.  grid (tokens' rows by 8, heads of the launch)
__global__ void __launch_bounds__(256) latent_tile_join_kernel(const __grid_constant__ TlArgs t) {
    const LrArgs& a = t.a;
    const int lane = threadIdx.x & 31, head_at = blockIdx.y;
    pdl_enter();
    int rest, slot = 0;                                              // blocks: those of each cut sequence's tokens, by 8
    const int seq = tl_find(a, blockIdx.x, [&](const PgSeq& s) { return tl_pieces(s, t) > 1 ? (s.count + 7) / 8 : 0; }, &rest);
    if (seq < 0) return;
    const PgSeq s = a.seqs[seq];
    for (int x = lane; x < seq; x += 32) { const int n = tl_pieces(a.seqs[x], t); slot += n > 1 ? n * tl_items(a.seqs[x], a) : 0; }
    slot = warp_sum_i(slot);
    const int row = rest * 8 + (threadIdx.x >> 5), pieces = tl_pieces(s, t), item = row / (2 * TL_ROWS);
    if (row >= s.count) return;
    const int64_t at = ((int64_t)(slot + (tl_items(s, a) - 1 - item) * pieces) * t.heads + head_at) * (2 * TL_ROWS) + row % (2 * TL_ROWS), stride = (int64_t)t.heads * 2 * TL_ROWS;
    const float sk = a.sink ? a.sink[t.head0 + head_at] * LR_LOG2E : -INFINITY;
    float m = sk;
    bool none = false, seen = false;                                 // a score that is none, one that is not -infinity
    for (int p = 0; p < pieces; p++) { const float b = t.ml[at + p * stride].x; none |= b != b; seen |= b != -INFINITY; m = fmaxf(m, b); }
    if (!seen) none = __any_sync(0xffffffffu, tl_wild(a, s.first + row, t.head0 + head_at, lane, 32));
    float total = sk == -INFINITY ? 0.0f : exp2f(sk - m);
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
    for (int p = 0; p < pieces; p++) {
        const float2 ml = t.ml[at + p * stride];
        if (ml.x == -INFINITY) continue;                              // nothing of its keys is seen: it may have left no sums
        const float w = exp2f(ml.x - m);
        total = fmaf(w, ml.y, total);
        if (lane * 4 < a.vdim) {
            const float4 v = *(const float4*)(t.part + (at + p * stride) * a.vdim + lane * 4);
            o.x = fmaf(w, v.x, o.x); o.y = fmaf(w, v.y, o.y); o.z = fmaf(w, v.z, o.z); o.w = fmaf(w, v.w, o.w);
        }
    }
    if (lane * 4 >= a.vdim) return;
    const float by = none ? NAN : 1.0f / total;
    uint16_t* out = (uint16_t*)a.out + ((int64_t)(s.first + row) * a.H + t.head0 + head_at) * a.vdim + lane * 4;
    *(uint2*)out = a.out_bf16 ? make_uint2(ht_pack_bf16(o.x * by, o.y * by), ht_pack_bf16(o.z * by, o.w * by)) : make_uint2(ht_pack_f16(o.x * by, o.y * by), ht_pack_f16(o.z * by, o.w * by));
}

// Items over many keys are cut into pieces of about a CTA's share of all steps where that saves TL_GAIN steps, and their sums joined: 16 heads, whole / cut, us: 64 tokens behind 8000 rows 184 / 77, 512 225 / 110,
// 128 behind 32000 681 / 230.  Asked to save 4 steps only: 1500 tokens alone 53 / 70, three prompts 83 / 85 (the sums are 128 KB a piece); 8 steps: 64 behind 8000 87, 16: 77.  Pieces of 4, 6, 8, 12, 16 steps
// and more (64 behind 8000): 91, 77, 97, 105, 120
#define TL_PIECE 6                            // steps of a piece, at least
#define TL_GAIN 16                            // steps that cutting has to save
#define TL_WORKSPACE ((int64_t)256 << 20)     // bytes of images that a call has at a time, as long as those of one sequence and head are no more
static int tl_run(cc_device* dev, const cc_page_plan* plan, const LrArgs& all) {
    const int64_t per = (int64_t)((all.dim + 63) / 64 + (all.vdim + 63) / 64) * TL_BLOCK, width = all.dim + all.rest;
    CUtensorMap rows, q, uk, uv;
    int rc = cc_make_tmap_pages(dev, &rows, all.rows, plan->n_pages, plan->page, all.cols, plan->page, 0);
    if (!rc) rc = cc_make_tmap_rows(dev, &q, all.q, plan->tokens, all.H * width, all.H * width * 2, TL_ROWS, false);
    const int wide = std::max(all.dim, all.vdim);
    if (!rc) rc = cc_make_tmap_rows(dev, &uk, all.uk, (int64_t)all.H * all.dim, all.rank, (int64_t)all.rank * 2, wide, false);
    if (!rc) rc = cc_make_tmap_rows(dev, &uv, all.uv, (int64_t)all.H * all.vdim, all.rank, (int64_t)all.rank * 2, wide, false);
    if (rc) return rc;
    CC_CUDA(dev, cc_smem_limit(dev, CC_LIMIT_LATENT + 3, latent_expand_kernel, TE_SMEM));
    CC_CUDA(dev, cc_smem_limit(dev, CC_LIMIT_LATENT + 4, latent_tile_kernel, TL_SMEM));
    // as many sequences at a time as have their images of one head in TL_WORKSPACE, and as many heads
    for (int first = 0, end; first < plan->n_seqs; first = end) {
        TlArgs t{};
        t.a = all;
        int64_t tiles = 0, steps = 0, longest = 0;
        for (end = first; end < plan->n_seqs; end++) {
            const PgSeq& s = plan->seqs[end];
            const int n = tl_key_tiles(s, all);
            if (tiles && (tiles + n) * per > TL_WORKSPACE) break;
            tiles += n;
            for (int i = tl_items(s, all) - 1; i >= 0; i--) {
                int lo, each[2];
                tl_steps(s, all, i * 2 * TL_ROWS, &lo, each);
                steps += std::max(each[0], each[1]); longest = std::max<int64_t>(longest, std::max(each[0], each[1]));
            }
        }
        if (!tiles) continue;
        t.a.seqs = plan->d_seqs + first; t.a.n_seqs = end - first; t.a.table = plan->d_table + (int64_t)first * all.table_cols;
        const int heads = (int)std::max<int64_t>(1, std::min<int64_t>(all.H, TL_WORKSPACE / (tiles * per)));
        const int64_t share = std::max<int64_t>(TL_PIECE, (steps * heads + dev->sm_count - 1) / dev->sm_count);
        if (longest >= share + TL_GAIN) t.piece = (int)share;
        int64_t items = 0, cut = 0, rows8 = 0;
        for (int i = first; i < end; i++) {
            const PgSeq& s = plan->seqs[i];
            const int64_t n = tl_pieces(s, t), mine = n * tl_items(s, all);
            items += mine;
            if (n > 1) { cut += mine; rows8 += (s.count + 7) / 8; }
        }
        CC_REQUIRE(dev, items * heads < ((int64_t)1 << 31) && tiles < ((int64_t)1 << 31), "paged_latent_attention: too many rows");
        const int64_t images = tiles * heads * per, sums = cut * heads * 2 * TL_ROWS;
        void* ws = nullptr; size_t cls = 0;
        rc = cc_pool_alloc(dev, (size_t)(images + sums * (all.vdim * 4 + 8)), &ws, &cls);
        if (rc) return rc;
        t.part = (float*)((uint8_t*)ws + images); t.ml = (float2*)(t.part + sums * all.vdim);
        t.k_image = (uint8_t*)ws; t.v_image = t.k_image + tiles * heads * ((all.dim + 63) / 64) * TL_BLOCK;
        t.key_tiles = (int)tiles;
        cudaError_t e = cudaSuccess;
        for (t.head0 = 0; t.head0 < all.H && e == cudaSuccess; t.head0 += heads) {
            t.heads = std::min(heads, all.H - t.head0);
            const int runs = (int)std::max<int64_t>(1, std::min<int64_t>(t.heads, dev->sm_count / (tiles + 1)));
            e = cc_launch_pdl(dev, latent_expand_kernel, dim3((unsigned)(tiles + 1) / 2 * 2, (unsigned)runs), TE_THREADS, TE_SMEM, rows, uk, uv, t, dev->err_dev, dev->err_host);
            if (e == cudaSuccess) e = cc_launch_pdl(dev, latent_tile_kernel, (unsigned)(items * t.heads), TL_THREADS, TL_SMEM, rows, q, t, dev->err_dev, dev->err_host);
            if (cut && e == cudaSuccess) { e = cc_launch_pdl(dev, latent_tile_join_kernel, dim3((unsigned)rows8, (unsigned)t.heads), 256, 0, t); dev->launches++; }
            dev->launches += 2;
        }
        cc_pool_free(dev, ws, cls);
        if (e != cudaSuccess) return cc_fail(dev, CC_ERR_CUDA, "paged_latent_attention: %s", cudaGetErrorString(e));
    }
    return CC_OK;
}
