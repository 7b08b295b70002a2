// latent.cu -- from projections to pages of latent rows (include/crabml_paged.h): norm, rotation and rounding of a token's row, and of its queries on the way.
//
// Bound by bytes: a token of 16 heads of 128 + 64 over rows of 512 + 64 is 3648 numbers of 2 or 4 bytes in and as many of 2 out.  The unit of work is a segment of
// the plan (new tokens of one sequence in one page), so that a CTA knows its page without a search; a CTA takes 8 of its rows, 8 neighbouring numbers a thread.
// The angles are made once a row and CTA: position x frequency in 64 bits and brought to a turn there (position 100000: 0.008 of a radian would be lost in 32), sine
// and cosine of the remainder in 32.  Alone and cold: 1 token and 64 7.8 us (latencies: look up, load, sum, store), 1700 tokens of three prompts, 16-bit rows, 18.5 (28.6 MB; 13 in a run of calls).
#include <algorithm>

#include "latent.cuh"

#define LA_THREADS 256
#define LA_ROWS (LA_THREADS / 32)             // of a segment that a CTA takes
#define LA_RUNS 3                             // runs of 8 columns of a cached row that a lane holds
#define LA_AHEAD 4                            // .. of the queries that a thread has under way
static_assert(LA_RUNS * 256 >= LT_RANK + LT_REST, "a warp holds a row");

int lt_check_pages(cc_device* dev, const cc_page_plan* plan, const cc_view* pages, int32_t rank, const char* what, LtPages* o) {
    if (!view_ok(pages)) return cc_fail(dev, CC_ERR_ARG, "%s: bad view of pages", what);
    HT_WHOLE(dev, pages, CC_F16, what);
    CC_REQUIRE(dev, pages->ndim == 3 && pages->shape[1] == plan->page && pages->shape[0] >= plan->n_pages, "%s: pages are not [%lld or more, %d, columns]", what,
               (long long)plan->n_pages, plan->page);
    const int64_t cols = pages->shape[2], rest = cols - rank;
    CC_REQUIRE(dev, rank >= 16 && rank <= LT_RANK && rank % 16 == 0 && rest >= 0 && rest <= LT_REST && rest % 16 == 0,
               "%s: rows of %d + %lld columns (multiples of 16 up to %d and %d)", what, rank, (long long)rest, LT_RANK, LT_REST);
    CC_REQUIRE(dev, ((uintptr_t)pages->buf->plane[0] & 15) == 0, "%s: pages do not start at a multiple of 16 bytes", what);
    o->rows = (__half*)pages->buf->plane[0]; o->rank = rank; o->rest = (int)rest; o->cols = (int)cols;
    return CC_OK;
}

struct LaArgs {
    const PgSegment* segments;
    const void *kv, *q;
    const float *norm, *freq;
    __half *rows, *qo;
    int64_t kv_stride, q_stride;
    int kv_type, q_type, kv_vec, q_vec, rank, rest, cols, page, H, dim, pairs, halves;
    float eps, mag;
};
// 8 numbers at column c of a head's or row's turned part; `at` their index in the source
__device__ __forceinline__ void la_turn(const LaArgs& a, const void* src, int type, int64_t at, int c, const float2* cs, float (&v)[8]) {
    if (!a.halves) {
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            const int i = (c + j) >> 1;
            if (i >= a.pairs) break;
            const float x = v[j], y = v[j + 1];
            v[j] = a.mag * fmaf(x, cs[i].x, -(y * cs[i].y));
            v[j + 1] = a.mag * fmaf(y, cs[i].x, x * cs[i].y);
        }
        return;
    }
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const int i = c + j;
        if (i >= 2 * a.pairs) break;
        const bool first = i < a.pairs;
        const float other = ht_read(src, at + j + (first ? a.pairs : -a.pairs), type);
        const float2 z = cs[first ? i : i - a.pairs];
        v[j] = a.mag * (first ? fmaf(v[j], z.x, -(other * z.y)) : fmaf(v[j], z.x, other * z.y));
    }
}
__device__ __forceinline__ uint4 la_pack(const float (&v)[8]) { return make_uint4(ht_pack_f16(v[0], v[1]), ht_pack_f16(v[2], v[3]), ht_pack_f16(v[4], v[5]), ht_pack_f16(v[6], v[7])); }

// grid (segments, groups of LA_ROWS of their rows, 1 + parts of the heads): the first CTAs the rows of the cache, a warp each, the others queries, 8 columns a thread
__global__ void __launch_bounds__(LA_THREADS) latent_append_kernel(const LaArgs a) {
    __shared__ float2 cs[LA_ROWS][LT_REST / 2];
    const int tid = threadIdx.x, lane = tid & 31;
    pdl_enter();
    const PgSegment g = a.segments[blockIdx.x];
    const int r0 = blockIdx.y * LA_ROWS, n = min(LA_ROWS, g.rows - r0);
    if (n <= 0) return;
    for (int e = tid; e < n * a.pairs; e += LA_THREADS) {
        // a whole number of turns leaves the fraction exactly; what is left of the angle, in turns, has 2^-53 of the position's turns as its error
        const int r = e / a.pairs, i = e - r * a.pairs;
        const double turns = (double)(g.pos0 + r0 + r) * (double)a.freq[i] * 0.15915494309189533577;
        const float part = (float)(turns - rint(turns));
        float s, c;
        sincospif(2.0f * part, &s, &c);
        cs[r][i] = make_float2(c, s);
    }
    __syncthreads();
    if (blockIdx.z == 0) {
        const int r = tid >> 5;
        if (r >= n) return;
        const int64_t from = (int64_t)(g.token0 + r0 + r) * a.kv_stride;
        __half* to = a.rows + ((int64_t)g.page * a.page + g.row0 + r0 + r) * a.cols;
        float v[LA_RUNS][8], s = 0.0f;
#pragma unroll
        for (int i = 0; i < LA_RUNS; i++) {
            const int c = (i * 32 + lane) * 8;
            if (c < a.cols) ht_read8(a.kv, from + c, a.kv_type, a.kv_vec, v[i]);
        }
#pragma unroll
        for (int i = 0; i < LA_RUNS; i++)
            if ((i * 32 + lane) * 8 < a.rank) {
#pragma unroll
                for (int j = 0; j < 8; j++) s = fmaf(v[i][j], v[i][j], s);
            }
        const float size = sqrtf(warp_sum(s) / (float)a.rank + a.eps);
#pragma unroll
        for (int i = 0; i < LA_RUNS; i++) {
            const int c = (i * 32 + lane) * 8;
            if (c >= a.cols) continue;
            if (c < a.rank) {
#pragma unroll
                for (int j = 0; j < 8; j++) v[i][j] = v[i][j] / size * (a.norm ? a.norm[c + j] : 1.0f);
            } else la_turn(a, a.kv, a.kv_type, from + c, c - a.rank, cs[r], v[i]);
            *(uint4*)(to + c) = la_pack(v[i]);
        }
        return;
    }
    const int runs = (a.dim + a.rest) / 8, all = a.H * runs, parts = gridDim.z - 1;
    const int lo = (int)((int64_t)all * (blockIdx.z - 1) / parts), each = (int)((int64_t)all * blockIdx.z / parts) - lo;
    for (int e0 = tid; e0 < n * each; e0 += LA_THREADS * LA_AHEAD) {
        float v[LA_AHEAD][8];
        int at[LA_AHEAD], row[LA_AHEAD];
#pragma unroll
        for (int i = 0; i < LA_AHEAD; i++) {
            const int e = e0 + i * LA_THREADS;
            if (e >= n * each) continue;
            row[i] = e / each; at[i] = lo + e - row[i] * each;
            ht_read8(a.q, (int64_t)(g.token0 + r0 + row[i]) * a.q_stride + (int64_t)at[i] * 8, a.q_type, a.q_vec, v[i]);
        }
#pragma unroll
        for (int i = 0; i < LA_AHEAD; i++) {
            if (e0 + i * LA_THREADS >= n * each) continue;
            const int c = at[i] % runs * 8 - a.dim;
            const int64_t token = g.token0 + r0 + row[i];
            if (c >= 0) la_turn(a, a.q, a.q_type, token * a.q_stride + (int64_t)at[i] * 8, c, cs[row[i]], v[i]);
            ((uint4*)a.qo)[token * all + at[i]] = la_pack(v[i]);
        }
    }
}

extern "C" CC_API int cc_paged_latent_append(cc_device* dev, const cc_page_plan* plan, const cc_view* pages, int32_t rank, const cc_view* kv_src, int32_t kv_col0, const cc_view* norm_w,
                                             float eps, const cc_view* q_src, int32_t q_col0, int32_t H, int32_t dim, const cc_view* freq, int32_t pairing, float mag, cc_buf** out) {
    PG_ENTER(dev, plan, "paged_latent_append");
    if (!out) return cc_fail(dev, CC_ERR_ARG, "paged_latent_append: out is NULL");
    *out = nullptr;
    LtPages c;
    int rc = lt_check_pages(dev, plan, pages, rank, "paged_latent_append", &c);
    if (rc) return rc;
    HT_ROWS(dev, kv_src, "paged_latent_append rows");
    if (q_src) HT_ROWS(dev, q_src, "paged_latent_append queries");
    const int64_t T = plan->tokens;
    CC_REQUIRE(dev, kv_src->shape[0] == T && (!q_src || q_src->shape[0] == T), "paged_latent_append: the plan has %lld tokens, not the sources' rows", (long long)T);
    CC_REQUIRE(dev, kv_col0 >= 0 && kv_col0 + (int64_t)c.cols <= kv_src->shape[1], "paged_latent_append: %d columns from %d on are not in the source", c.cols, kv_col0);
    CC_REQUIRE(dev, !q_src || (H > 0 && H <= 8192 && dim >= 16 && dim <= LT_DIM && dim % 16 == 0), "paged_latent_append: %d heads of %d (multiples of 16 up to %d)", H, dim, LT_DIM);
    CC_REQUIRE(dev, !q_src || (q_col0 >= 0 && q_col0 + (int64_t)H * (dim + c.rest) <= q_src->shape[1]), "paged_latent_append: %d heads of %d + %d from column %d on are not in the source",
               H, dim, c.rest, q_col0);
    CC_REQUIRE(dev, pairing == CC_ROPE_NEIGHBOURS || pairing == CC_ROPE_HALVES, "paged_latent_append: pairing %d", pairing);
    if (norm_w) {
        HT_WHOLE(dev, norm_w, CC_F32, "paged_latent_append norm_w");
        CC_REQUIRE(dev, view_len(norm_w) == rank, "paged_latent_append: norm_w is not [%d]", rank);
    }
    int64_t pairs = 0;
    if (freq) {
        HT_WHOLE(dev, freq, CC_F32, "paged_latent_append freq");
        pairs = view_len(freq);
        CC_REQUIRE(dev, 2 * pairs <= c.rest, "paged_latent_append: %lld pairs in %d columns", (long long)pairs, c.rest);
    }
    CC_REQUIRE(dev, kv_src->buf != pages->buf && (!q_src || q_src->buf != pages->buf), "paged_latent_append: a source is the pages");
    cc_buf* o = nullptr;
    if (q_src) {
        rc = cc_new_activation(dev, T * H * (dim + c.rest), CC_F16, false, &o);
        if (rc) return rc;
    }
    if (T > 0) {
        LaArgs a{};
        a.segments = plan->d_segments;
        const int ks = ht_size(kv_src->buf->dtype);
        a.kv = kv_src->buf->plane[0] + (int64_t)kv_col0 * ks; a.kv_type = kv_src->buf->dtype; a.kv_stride = kv_src->strides[0];
        a.kv_vec = ((uintptr_t)a.kv & 15) == 0 && a.kv_stride * ks % 16 == 0;
        if (q_src) {
            const int qs = ht_size(q_src->buf->dtype);
            a.q = q_src->buf->plane[0] + (int64_t)q_col0 * qs; a.q_type = q_src->buf->dtype; a.q_stride = q_src->strides[0];
            a.q_vec = ((uintptr_t)a.q & 15) == 0 && a.q_stride * qs % 16 == 0;
            a.qo = (__half*)o->base; a.H = H; a.dim = dim;
        }
        a.norm = norm_w ? (const float*)norm_w->buf->plane[0] : nullptr; a.freq = freq ? (const float*)freq->buf->plane[0] : nullptr;
        a.rows = c.rows; a.rank = c.rank; a.rest = c.rest; a.cols = c.cols; a.page = plan->page; a.pairs = (int)pairs; a.halves = pairing == CC_ROPE_HALVES; a.eps = eps; a.mag = mag;
        // the queries' columns over as many CTAs as let each thread have LA_AHEAD runs or fewer of one token, or of LA_ROWS of a portion
        const int64_t runs = q_src ? (int64_t)H * (dim + c.rest) / 8 * (T > 4 * (int64_t)plan->n_segments ? LA_ROWS : 1) : 0;
        const unsigned parts = (unsigned)std::min<int64_t>(64, (runs + LA_THREADS * LA_AHEAD - 1) / (LA_THREADS * LA_AHEAD));
        const unsigned groups = T == plan->n_segments ? 1u : (unsigned)(plan->page + LA_ROWS - 1) / LA_ROWS;
        const cudaError_t e = cc_launch_pdl(dev, latent_append_kernel, dim3((unsigned)plan->n_segments, groups, 1 + parts), LA_THREADS, 0, a);
        dev->launches++;
        if (e != cudaSuccess) {
            if (o) cc_tensor_release(o);
            return cc_fail(dev, CC_ERR_CUDA, "paged_latent_append: %s", cudaGetErrorString(e));
        }
    }
    *out = o;
    return CC_OK;
}
