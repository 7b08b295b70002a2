// paged.cu -- pages of a cache that several sequences share (include/crabml_paged.h): the plan of a step, and what lies between the projections and the pages.
//
// The plan is checked on the host as a whole, so that no kernel meets a page or slot number that it would have to doubt, and copied to the device once a step.
// The append's unit is a segment, the new tokens of one sequence in one block, times a job: one key head, one value head or some query heads.  A segment that
// completes a block of an 8-bit cache has the whole block of a head in shared memory (old rows from the open block, new ones turned and rounded), so the largest
// magnitude is known before a code is written and every number is rounded once.
//
// The turn is computed in 64 bits: a far position times a frequency loses its fraction in 32 (position 100000: 0.008 of a radian), and a key next to a rounding
// border would get another code from another order of the same 32-bit operations.
#include <math.h>
#include <string.h>

#include <algorithm>
#include <new>

#include "paged.cuh"

// ---- the plan ---------------------------------------------------------------------------------------------------------------------------
// Pinned staging of plans on their way to the device, by turns: a host that works ahead of the device takes another buffer, up to CC_PLAN_BUFFERS, and then waits for the oldest copy
static int pg_upload(cc_device* dev, void* dst, const std::vector<uint8_t>& bytes) {
    std::lock_guard<std::mutex> g(dev->plan_mu);
    if (dev->plans.empty() || (dev->plans.size() < CC_PLAN_BUFFERS && cudaEventQuery(dev->plans[dev->plan_turn].through) == cudaErrorNotReady)) {
        dev->plans.insert(dev->plans.begin() + dev->plan_turn, CcPlanBuffer());
        cudaGetLastError();                                 // (the query's answer is no error of a later call)
    }
    CcPlanBuffer& b = dev->plans[dev->plan_turn];
    if (!b.through) CC_CUDA(dev, cudaEventCreateWithFlags(&b.through, cudaEventDisableTiming));
    CC_CUDA(dev, cudaEventSynchronize(b.through));
    if (b.bytes < bytes.size()) {
        if (b.pinned) dev->plan_small.push_back(b.pinned);  // (to free it would wait for the device)
        b.pinned = nullptr; b.bytes = 0;
        size_t n = 64 << 10;
        while (n < bytes.size()) n *= 2;
        CC_CUDA(dev, cudaMallocHost(&b.pinned, n));
        b.bytes = n;
    }
    memcpy(b.pinned, bytes.data(), bytes.size());
    CC_CUDA(dev, cudaMemcpyAsync(dst, b.pinned, bytes.size(), cudaMemcpyHostToDevice, dev->stream));
    CC_CUDA(dev, cudaEventRecord(b.through, dev->stream));
    dev->plan_turn = (dev->plan_turn + 1) % dev->plans.size();
    return CC_OK;
}

static int pg_plan(cc_device* dev, const cc_page_plan_desc* d, cc_page_plan* p) {
    if (d->n_seqs > 0 && (!d->pos0 || !d->counts || (d->table_cols > 0 && !d->table))) return cc_fail(dev, CC_ERR_ARG, "page_plan: a NULL array");
    PgParts parts;
    const std::string wrong = pg_build(*d, parts);
    CC_REQUIRE(dev, wrong.empty(), "page_plan: %s", wrong.c_str());
    p->dev = dev; p->n_seqs = d->n_seqs; p->page = d->page_size; p->table_cols = d->table_cols; p->n_pages = d->n_pages; p->n_slots = d->n_slots;
    p->n_items = parts.n_items; p->n_segments = (int)parts.segments.size(); p->tokens = parts.tokens;
    while ((1 << p->shift) < p->page) p->shift++;
    const size_t seg = parts.segments.size() * sizeof(PgSegment), sq = parts.seqs.size() * sizeof(PgSeq), tab = parts.table.size() * sizeof(int);
    std::vector<uint8_t> bytes(seg + sq + tab + 16);
    if (seg) memcpy(bytes.data(), parts.segments.data(), seg);
    if (sq) memcpy(bytes.data() + seg, parts.seqs.data(), sq);
    if (tab) memcpy(bytes.data() + seg + sq, parts.table.data(), tab);
    p->seqs = std::move(parts.seqs);
    int rc = cc_pool_alloc(dev, bytes.size(), &p->base, &p->cls);
    if (!rc) rc = pg_upload(dev, p->base, bytes);
    if (rc) return rc;
    p->d_segments = (const PgSegment*)p->base;
    p->d_seqs = (const PgSeq*)((uint8_t*)p->base + seg);
    p->d_table = (const int*)((uint8_t*)p->base + seg + sq);
    return CC_OK;
}
extern "C" CC_API int cc_page_plan_create(cc_device* dev, const cc_page_plan_desc* desc, cc_page_plan** out) {
    if (!dev) return CC_ERR_ARG;
    CC_ENTER(dev);
    if (!desc || !out) return cc_fail(dev, CC_ERR_ARG, "page_plan: a NULL argument");
    *out = nullptr;
    if (LAZY(dev)) return cc_fail(dev, CC_ERR_UNSUPPORTED, "page_plan: not available on a lazy (graph / megakernel) device");
    cc_page_plan* p = new (std::nothrow) cc_page_plan();
    if (!p) return cc_fail(dev, CC_ERR_ARG, "page_plan: out of memory");
    int rc;
    try {
        rc = pg_plan(dev, desc, p);
    } catch (const std::bad_alloc&) {
        rc = cc_fail(dev, CC_ERR_ARG, "page_plan: out of memory");
    }
    if (rc) { cc_page_plan_release(p); return rc; }
    *out = p;
    return CC_OK;
}
extern "C" CC_API void cc_page_plan_release(cc_page_plan* plan) {
    if (!plan) return;
    if (plan->base) cc_pool_free(plan->dev, plan->base, plan->cls);
    delete plan;
}
extern "C" CC_API int64_t cc_page_plan_tokens(const cc_page_plan* plan) { return plan ? plan->tokens : 0; }

// ---- a cache's views ----------------------------------------------------------------------------------------------------------------------
static int pg_check_pages(cc_device* dev, const cc_view* v, int dtype, int ndim, const char* what, const char* name) {
    if (!view_ok(v)) return cc_fail(dev, CC_ERR_ARG, "%s: bad view of %s", what, name);
    CC_REQUIRE(dev, view_in_bounds(v) && view_contiguous(v) && v->ndim == ndim, "%s: %s is not a contiguous tensor of %d dimensions inside its buffer", what, name, ndim);
    CC_REQUIRE(dev, v->buf->dev == dev, "%s: %s is another device's", what, name);
    CC_REQUIRE(dev, v->buf->dtype == dtype, "%s: %s has type %d, not %d", what, name, v->buf->dtype, dtype);
    CC_REQUIRE(dev, ((uintptr_t)v->buf->plane[0] & 15) == 0, "%s: %s does not start at a multiple of 16 bytes", what, name);
    return CC_OK;
}
int pg_check_cache(cc_device* dev, const cc_page_plan* plan, const cc_paged_cache* c, const char* what, PgCache* o) {
    if (!c || !view_ok(&c->k) || !view_ok(&c->v)) return cc_fail(dev, CC_ERR_ARG, "%s: bad cache", what);
    const int type = c->k.buf->dtype;
    CC_REQUIRE(dev, type == CC_F16 || type == CC_I8, "%s: pages of type %d (F16 or I8)", what, type);
    int rc = pg_check_pages(dev, &c->k, type, 4, what, "k");
    if (!rc) rc = pg_check_pages(dev, &c->v, type, 4, what, "v");
    if (rc) return rc;
    const int64_t G = c->k.shape[1], dk = c->k.shape[3], dv = c->v.shape[3];
    CC_REQUIRE(dev, c->k.shape[0] == c->v.shape[0] && c->v.shape[1] == G && c->k.shape[2] == plan->page && c->v.shape[2] == plan->page,
               "%s: k and v are not [pages, heads, %d, size] alike", what, plan->page);
    CC_REQUIRE(dev, c->k.shape[0] >= plan->n_pages, "%s: %lld pages, the plan has %lld", what, (long long)c->k.shape[0], (long long)plan->n_pages);
    CC_REQUIRE(dev, G >= 1 && G <= 1024 && dk >= 16 && dk <= 256 && dk % 16 == 0 && dv >= 16 && dv <= 256 && dv % 16 == 0,
               "%s: %lld heads of %lld and %lld (multiples of 16 up to 256)", what, (long long)G, (long long)dk, (long long)dv);
    *o = PgCache{};
    o->k = c->k.buf->plane[0]; o->v = c->v.buf->plane[0]; o->G = (int)G; o->dk = (int)dk; o->dv = (int)dv; o->i8 = type == CC_I8;
    if (!o->i8) return CC_OK;
    const cc_view* more[4] = {&c->k_scale, &c->v_scale, &c->k_open, &c->v_open};
    const char* names[4] = {"k_scale", "v_scale", "k_open", "v_open"};
    for (int i = 0; i < 4 && !rc; i++) rc = pg_check_pages(dev, more[i], i < 2 ? CC_F32 : CC_F16, i < 2 ? 2 : 4, what, names[i]);
    if (rc) return rc;
    for (int i = 0; i < 2; i++) {
        const cc_view *s = more[i], *w = more[2 + i];
        CC_REQUIRE(dev, s->shape[0] >= plan->n_pages && s->shape[1] == G, "%s: %s is not [pages, heads]", what, names[i]);
        CC_REQUIRE(dev, plan->n_slots > 0 || plan->n_seqs == 0, "%s: 8-bit pages need a plan with slots", what);
        CC_REQUIRE(dev, w->shape[0] >= 2 * plan->n_slots && w->shape[1] == G && w->shape[2] == plan->page && w->shape[3] == (i ? dv : dk),
                   "%s: %s is not [2 * %lld, %lld, %d, size]", what, names[2 + i], (long long)plan->n_slots, (long long)G, plan->page);
    }
    o->ks = (float*)c->k_scale.buf->plane[0]; o->vs = (float*)c->v_scale.buf->plane[0];
    o->ko = (__half*)c->k_open.buf->plane[0]; o->vo = (__half*)c->v_open.buf->plane[0];
    return CC_OK;
}

// ---- append --------------------------------------------------------------------------------------------------------------------------------
#define PA_THREADS 256
#define PA_WARPS (PA_THREADS / 32)
#define PA_ROWS 4                            // rows of angles that a CTA makes for itself at a time
#define PA_SMEM ((int)(PA_ROWS * 128 * sizeof(double2)) + 128 * 256 * 2)      // .. of 128 pairs, and a block of 128 rows of 256
struct PaArgs {
    const PgSegment* segments;
    const float *q, *k, *v, *freq;
    double2* angles;                         // [T][pairs] cos and sin times mag, or NULL: every CTA makes its own
    float* qo;
    uint8_t *kp, *vp;
    float *ks, *vs;
    __half *ko, *vo;
    int64_t qrs, krs, vrs;                   // row strides
    int H, G, dk, dv, page, pairs, offset, step, gap, hq, q_parts, vec;      // pair i: columns offset + step * i and + gap behind it; hq: query heads of a job, which takes PA_Q_ROWS rows where q_parts > 1; vec: neighbours that can be read as one
    double mag;
};
// F16 of a 32-bit number; what is finite stays finite
__device__ __forceinline__ __half pa_half(float x) {
    __half h = __float2half_rn(x);
    if (__hisinf(h) && !isinf(x)) h = __ushort_as_half((unsigned short)(x > 0.0f ? 0x7bff : 0xfbff));
    return h;
}
__device__ __forceinline__ __half2 pa_half2(float2 v) {
    if (fmaxf(fabsf(v.x), fabsf(v.y)) >= 65520.0f) return __halves2half2(pa_half(v.x), pa_half(v.y));
    return __floats2half2_rn(v.x, v.y);
}
__device__ __forceinline__ double2 pa_angle(const PaArgs& a, int pos, int i) {
    double s, c;
    sincos((double)pos * (double)a.freq[i], &s, &c);
    return make_double2(c * a.mag, s * a.mag);
}
// the angles of all tokens, once for all heads: a thread a pair of a token, CTAs of a segment
__global__ void __launch_bounds__(PA_THREADS) paged_angles_kernel(const PaArgs a, int n_segments) {
    pdl_enter();
    for (int at = blockIdx.x; at < n_segments; at += gridDim.x) {
        const PgSegment g = a.segments[at];
        for (int e = blockIdx.y * PA_THREADS + threadIdx.x; e < g.rows * a.pairs; e += gridDim.y * PA_THREADS) {
            const int r = e / a.pairs, i = e - r * a.pairs;
            a.angles[(int64_t)(g.token0 + r) * a.pairs + i] = pa_angle(a, g.pos0 + r, i);
        }
    }
}
// Units of a head's row: pairs, which are turned, and behind them the columns that stay.  Where unit u lies
__device__ __forceinline__ int pa_column(const PaArgs& a, int u) {
    if (u < a.pairs) return a.offset + a.step * u;
    const int c = u - a.pairs;
    return c >= a.offset ? c + 2 * a.pairs : c;
}
// what a unit reads and writes at its first column: a pair (its second number `gap` further on), or one number
__device__ __forceinline__ float2 pa_read(const PaArgs& a, const float* p, bool pair) {
    if (!pair) return make_float2(__ldg(p), 0.0f);
    if (a.vec) return __ldg((const float2*)p);
    return make_float2(__ldg(p), __ldg(p + a.gap));
}
__device__ __forceinline__ float2 pa_turn(float2 v, const double2& t) {
    const double x = (double)v.x, y = (double)v.y;
    return make_float2((float)fma(x, t.x, -(y * t.y)), (float)fma(x, t.y, y * t.x));
}
__device__ __forceinline__ void pa_write(const PaArgs& a, float* p, float2 v, bool pair) {
    if (pair && a.step == 2 && ((uintptr_t)p & 7) == 0) { *(float2*)p = v; return; }
    p[0] = v.x;
    if (pair) p[a.gap] = v.y;
}
__device__ __forceinline__ void pa_write(const PaArgs& a, __half* p, float2 v, bool pair) {
    if (!pair) { p[0] = pa_half(v.x); return; }
    const __half2 h = pa_half2(v);
    if (a.step == 2 && ((uintptr_t)p & 3) == 0) { *(__half2*)p = h; return; }
    p[0] = __low2half(h); p[a.gap] = __high2half(h);
}
// round(127 x / most) of four of a block's numbers, ties to even, as the exact quotient rounds.  x and most have 11 bits, so 127 x is exact and a quotient that is not a tie is further from one than
// a 32-bit division errs; 127 / most and the product err by less than 2e-5, and where that leaves it open the quotient is taken
__device__ __forceinline__ unsigned pa_code4(uint2 u, float most, float r) {
    constexpr float M = 12582912.0f;
    const float2 lo = __half22float2(*(const __half2*)&u.x), hi = __half22float2(*(const __half2*)&u.y);
    const float x[4] = {lo.x, lo.y, hi.x, hi.y};
    float n[4], far = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float y = x[i] * r;
        n[i] = y + M;
        far = fmaxf(far, fabsf(y - (n[i] - M)));
    }
    if (far < 0.49998f)
        return __byte_perm(__byte_perm(__float_as_uint(n[0]), __float_as_uint(n[1]), 0x0040), __byte_perm(__float_as_uint(n[2]), __float_as_uint(n[3]), 0x0040), 0x5410);
    unsigned c = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) c |= ((unsigned)(int)rintf(x[i] * 127.0f / most) & 255u) << (8 * i);
    return c;
}
#define PA_Q_ROWS 16
#define PA_AHEAD 4                           // rows of a head, or heads of a row, that a warp reads before it turns the first
// f(row r0, so many rows, their angles): all rows of a job, or portions whose angles the CTA makes first
template <bool TABLE, class F>
__device__ __forceinline__ void pa_portions(const PaArgs& a, const PgSegment& g, int row_from, int row_to, bool turned, double2* made, F f) {
    if constexpr (!TABLE) {
        if (turned && a.pairs > 0) {
            for (int r0 = 0; r0 < g.rows; r0 += PA_ROWS) {
                const int rows = min(PA_ROWS, g.rows - r0);
                __syncthreads();
                for (int e = threadIdx.x; e < rows * a.pairs; e += PA_THREADS) { const int r = e / a.pairs; made[e] = pa_angle(a, g.pos0 + r0 + r, e - r * a.pairs); }
                __syncthreads();
                f(r0, rows, made);
            }
            return;
        }
    }
    f(row_from, row_to - row_from, a.angles + (int64_t)(g.token0 + row_from) * a.pairs);
}
// grid (segments, jobs): jobs 0 .. G - 1 key heads, then G value heads (of the first n_items segments, and those behind them in their chains), then query heads by hq (and their rows by PA_Q_ROWS).
// A warp takes 32 units of a head, in rows so many further on as warps share them
template <bool I8, bool TABLE>
__global__ void __launch_bounds__(PA_THREADS, 4) paged_append_kernel(const PaArgs a, int n_items) {
    extern __shared__ __align__(16) uint8_t pa_sm[];
    double2* made = (double2*)pa_sm;                            // [PA_ROWS][pairs], where the angles are not there already
    __half* block = (__half*)(pa_sm + (TABLE ? 0 : (size_t)PA_ROWS * a.pairs * sizeof(double2)));      // [page][d]
    __shared__ unsigned tops[PA_WARPS];
    const int job = blockIdx.y, tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
    const bool is_k = job < a.G, is_v = !is_k && job < 2 * a.G, is_q = !is_k && !is_v;
    pdl_enter();
    if (!is_q && blockIdx.x >= n_items) return;
    for (int at = blockIdx.x; at >= 0;) {
        const PgSegment g = a.segments[at];
        at = is_q ? -1 : g.next;
        const int part = is_q ? (job - 2 * a.G) % a.q_parts : 0, row_from = part * PA_Q_ROWS, row_to = is_q && a.q_parts > 1 ? min(g.rows, row_from + PA_Q_ROWS) : g.rows;
        auto portions = [&](bool turned, auto f) { pa_portions<TABLE>(a, g, row_from, row_to, turned, made, f); };
        // the CTA's warps over `kinds` kinds of work and rows: f(kind, first row, rows from one to the next)
        auto share = [&](int kinds, auto f) {
            const int at_once = min(kinds, PA_WARPS), by = PA_WARPS / at_once, first = w / at_once;
            if (first < by)
                for (int k = w - first * at_once; k < kinds; k += at_once) f(k, first, by);
        };
        if (is_q) {
            const int h0 = (job - 2 * a.G) / a.q_parts * a.hq, nh = min(a.hq, a.H - h0), units = a.dk - a.pairs, runs = (units + 31) >> 5, batches = (nh + PA_AHEAD - 1) / PA_AHEAD;
            portions(true, [&](int r0, int rows, const double2* cs) {
                share(runs * batches, [&](int kind, int first, int by) {
                    const int b = kind / runs, u = (kind - b * runs) * 32 + lane, n = min(PA_AHEAD, nh - b * PA_AHEAD), c = pa_column(a, u);
                    if (u >= units) return;
                    const bool pair = u < a.pairs;
                    const int64_t t = g.token0 + r0 + first, at_head = (int64_t)(h0 + b * PA_AHEAD) * a.dk + c, out_step = (int64_t)by * a.H * a.dk;
                    const float* src = a.q + t * a.qrs + at_head;
                    float* dst = a.qo + t * a.H * a.dk + at_head;
                    const double2* angle = cs + first * a.pairs + u;
                    for (int r = first; r < rows; r += by, src += by * a.qrs, dst += out_step, angle += by * a.pairs) {
                        float2 v[PA_AHEAD];
                        double2 z = make_double2(0.0, 0.0);
#pragma unroll
                        for (int i = 0; i < PA_AHEAD; i++)
                            if (i < n) v[i] = pa_read(a, src + i * a.dk, pair);
                        if (pair) z = *angle;
#pragma unroll
                        for (int i = 0; i < PA_AHEAD; i++)
                            if (i < n) pa_write(a, dst + i * a.dk, pair ? pa_turn(v[i], z) : v[i], pair);
                    }
                });
            });
            continue;
        }
        const int head = is_k ? job : job - a.G, d = is_k ? a.dk : a.dv;
        const size_t page_at = ((size_t)g.page * a.G + head) * a.page * d;
        __half* open = I8 ? (is_k ? a.ko : a.vo) + ((size_t)g.half * a.G + head) * a.page * d : nullptr;
        __half* to = (I8 ? block : (__half*)(is_k ? a.kp : a.vp) + page_at) + g.row0 * d;      // 16-bit pages: straight to their place
        if (I8 && (g.flags & PG_FULL))                          // the block's older rows
            for (int e = tid; e < g.row0 * d / 8; e += PA_THREADS) ((uint4*)block)[e] = ((const uint4*)open)[e];
        const float* src = (is_k ? a.k : a.v) + (int64_t)head * d;
        const int64_t rs = is_k ? a.krs : a.vrs;
        const int units = is_k ? d - a.pairs : d;
        portions(is_k, [&](int r0, int rows, const double2* cs) {
            share((units + 31) >> 5, [&](int kind, int first, int by) {
                constexpr int AHEAD = TABLE ? PA_AHEAD : 1;
                const int u = kind * 32 + lane, c = is_k ? pa_column(a, u) : u;
                if (u >= units) return;
                const bool pair = is_k && u < a.pairs;
                const float* from = src + (g.token0 + r0 + first) * rs + c;
                __half* dst = to + (r0 + first) * d + c;
                const double2* angle = cs + first * a.pairs + u;
                for (int r = first; r < rows; r += by * AHEAD, from += by * AHEAD * rs, dst += by * AHEAD * d, angle += by * AHEAD * a.pairs) {
                    float2 v[AHEAD];
                    double2 z[AHEAD];
#pragma unroll
                    for (int i = 0; i < AHEAD; i++) {
                        if (r + i * by >= rows) continue;
                        v[i] = pa_read(a, from + i * by * rs, pair);
                        if (pair) z[i] = angle[i * by * a.pairs];
                    }
#pragma unroll
                    for (int i = 0; i < AHEAD; i++)
                        if (r + i * by < rows) pa_write(a, dst + i * by * d, pair ? pa_turn(v[i], z[i]) : v[i], pair);
                }
            });
        });
        if (!I8) continue;
        __syncthreads();
        if (g.flags & PG_KEPT)
            for (int e = tid; e < g.rows * d / 8; e += PA_THREADS) ((uint4*)(open + g.row0 * d))[e] = ((const uint4*)(block + g.row0 * d))[e];
        if (g.flags & PG_FULL) {
            unsigned m = 0;
            for (int e = tid; e < a.page * d / 2; e += PA_THREADS) m = __vmaxu2(m, ((const unsigned*)block)[e] & 0x7fff7fffu);
            m = __reduce_max_sync(0xffffffffu, max(m & 0xffffu, m >> 16));
            if (lane == 0) tops[w] = m;
            __syncthreads();
            unsigned top = 0;
#pragma unroll
            for (int i = 0; i < PA_WARPS; i++) top = max(top, tops[i]);
            const bool finite = top < 0x7c00u;
            const float most = __half2float(__ushort_as_half((unsigned short)top));
            uint2* codes = (uint2*)((is_k ? a.kp : a.vp) + page_at);
            const bool some = finite && top;
            const float r = 127.0f / most;
            for (int e = tid; e < a.page * d / 8; e += PA_THREADS) {
                const uint4 x = ((const uint4*)block)[e];
                codes[e] = some ? make_uint2(pa_code4(make_uint2(x.x, x.y), most, r), pa_code4(make_uint2(x.z, x.w), most, r)) : make_uint2(0u, 0u);
            }
            if (tid == 0) (is_k ? a.ks : a.vs)[(size_t)g.page * a.G + head] = finite ? most / 127.0f : NAN;
        }
        __syncthreads();                                        // the block and `tops`, before the next segment
    }
}
extern "C" CC_API int cc_paged_append(cc_device* dev, const cc_page_plan* plan, const cc_paged_cache* cache, const cc_view* q_src, int32_t q_col0, const cc_view* k_src,
                                      int32_t k_col0, const cc_view* v_src, int32_t v_col0, int32_t H, const cc_view* freq, int32_t pairing, int32_t offset, float mag,
                                      cc_buf** out) {
    PG_ENTER(dev, plan, "paged_append");
    if (!out) return cc_fail(dev, CC_ERR_ARG, "paged_append: out is NULL");
    *out = nullptr;
    PgCache c;
    int rc = pg_check_cache(dev, plan, cache, "paged_append", &c);
    if (rc) return rc;
    CC_REQUIRE(dev, c.k != c.v && (!c.i8 || (c.ks != c.vs && c.ko != c.vo)), "paged_append: keys and values go to one tensor");      // different CTAs write them
    PG_ROWS(dev, k_src, "paged_append keys"); PG_ROWS(dev, v_src, "paged_append values");
    if (q_src) PG_ROWS(dev, q_src, "paged_append queries");
    const int64_t T = plan->tokens;
    CC_REQUIRE(dev, k_src->shape[0] == T && v_src->shape[0] == T && (!q_src || q_src->shape[0] == T), "paged_append: the plan has %lld tokens, not the sources' rows", (long long)T);
    CC_REQUIRE(dev, !q_src || (H > 0 && H <= 8192 && H % c.G == 0), "paged_append: %d query heads over %d", H, c.G);
    CC_REQUIRE(dev, k_col0 >= 0 && v_col0 >= 0 && k_col0 + (int64_t)c.G * c.dk <= k_src->shape[1] && v_col0 + (int64_t)c.G * c.dv <= v_src->shape[1] &&
               (!q_src || (q_col0 >= 0 && q_col0 + (int64_t)H * c.dk <= q_src->shape[1])), "paged_append: columns %d / %d / %d do not fit %d and %d heads of %d and %d", q_col0,
               k_col0, v_col0, H, c.G, c.dk, c.dv);
    CC_REQUIRE(dev, pairing == CC_ROPE_NEIGHBOURS || pairing == CC_ROPE_HALVES, "paged_append: pairing %d", pairing);
    int64_t pairs = 0;
    if (freq) {
        if (!view_ok(freq)) return cc_fail(dev, CC_ERR_ARG, "paged_append: bad view of freq");
        CC_REQUIRE(dev, view_in_bounds(freq) && view_contiguous(freq) && freq->buf->dev == dev && freq->buf->dtype == CC_F32, "paged_append: freq is not contiguous F32 of this device");
        pairs = view_len(freq);
        CC_REQUIRE(dev, offset >= 0 && offset + 2 * pairs <= c.dk, "paged_append: %lld pairs from column %d do not fit heads of %d", (long long)pairs, offset, c.dk);
    }
    cc_buf* o = nullptr;
    if (q_src) {
        rc = cc_new_activation(dev, T * H * c.dk, CC_F32, false, &o);
        if (rc) return rc;
    }
    if (T > 0) {
        PaArgs a{};
        a.segments = plan->d_segments;
        if (q_src) { a.q = (const float*)q_src->buf->plane[0] + q_col0; a.qrs = q_src->strides[0]; a.qo = (float*)o->base; }
        a.k = (const float*)k_src->buf->plane[0] + k_col0; a.krs = k_src->strides[0];
        a.v = (const float*)v_src->buf->plane[0] + v_col0; a.vrs = v_src->strides[0];
        a.freq = freq ? (const float*)freq->buf->plane[0] : nullptr;
        a.kp = c.k; a.vp = c.v; a.ks = c.ks; a.vs = c.vs; a.ko = c.ko; a.vo = c.vo;
        a.H = q_src ? H : 0; a.G = c.G; a.dk = c.dk; a.dv = c.dv; a.page = plan->page; a.pairs = (int)pairs; a.offset = offset; a.mag = (double)mag;
        a.step = pairing == CC_ROPE_NEIGHBOURS ? 2 : 1; a.gap = pairing == CC_ROPE_NEIGHBOURS ? 1 : (int)pairs;
        a.vec = pairing == CC_ROPE_NEIGHBOURS && ((offset | c.dk | k_col0 | (int)(a.krs & 1)) & 1) == 0 && (!q_src || ((q_col0 | (int)(a.qrs & 1)) & 1) == 0) &&
                (((uintptr_t)k_src->buf->plane[0] | (q_src ? (uintptr_t)q_src->buf->plane[0] : 0)) & 7) == 0;
        // a portion of many rows a block: the angles once for all heads, in a kernel of their own (64 rows of 64 pairs made by each of 16 CTAs:
        // three prompts of 1957 tokens, 32 heads on 8, 125 us, with the table 4 + 32); single tokens: by every CTA
        const bool table = pairs > 0 && T > 4 * (int64_t)plan->n_segments;
        a.hq = table ? 4 : 8; a.q_parts = table ? plan->page / PA_Q_ROWS : 1;
        void* ws = nullptr; size_t cls = 0;
        if (table) {
            rc = cc_pool_alloc(dev, (size_t)T * pairs * sizeof(double2), &ws, &cls);
            if (rc) { if (o) cc_tensor_release(o); return rc; }
            a.angles = (double2*)ws;
        }
        const size_t smem = (table ? 0 : (size_t)PA_ROWS * a.pairs * sizeof(double2)) + (c.i8 ? (size_t)a.page * std::max(c.dk, c.dv) * 2 : 0);
        const dim3 grid((unsigned)plan->n_segments, (unsigned)(2 * c.G + (a.H + a.hq - 1) / a.hq * a.q_parts));
        cudaError_t e = cudaSuccess;
        if (table) {
            const int64_t per = ((int64_t)plan->page * pairs + PA_THREADS - 1) / PA_THREADS;
            e = cc_launch_pdl(dev, paged_angles_kernel, dim3((unsigned)std::min(plan->n_segments, 65535), (unsigned)std::min<int64_t>(per, 16)), PA_THREADS, 0, a, plan->n_segments);
            dev->launches++;
        }
        auto kernel = c.i8 ? (table ? paged_append_kernel<true, true> : paged_append_kernel<true, false>) : (table ? paged_append_kernel<false, true> : paged_append_kernel<false, false>);
        // the most that any call needs, always: the attribute is the kernel's, not this call's, and another thread's device may be between here and its launch
        if (e == cudaSuccess && smem > 40 * 1024) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PA_SMEM);
        if (e == cudaSuccess) e = cc_launch_pdl(dev, kernel, grid, PA_THREADS, smem, a, plan->n_items);
        dev->launches++;
        if (ws) cc_pool_free(dev, ws, cls);
        if (e != cudaSuccess) {
            if (o) cc_tensor_release(o);
            return cc_fail(dev, CC_ERR_CUDA, "paged_append: %s", cudaGetErrorString(e));
        }
    }
    *out = o;
    return CC_OK;
}
