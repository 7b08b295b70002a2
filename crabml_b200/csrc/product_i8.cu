// product_i8.cu -- products in 8-bit integers (cc_product_i8 of include/crabml_seqops.h): activations coded row by row, exact integer sums, one factor per token
// and one per output channel.
#include <math.h>

#include "../../include/crabml_seqops.h"
#include "capi_checks.cuh"

// ---- activations -> codes ------------------------------------------------------------------------------------------------------------------
// round(127 x / a), ties to even, as the exact quotient rounds.  127 / a and the product err by less than 1e-4 of a step; where that leaves it open (one number
// in 500 is so near to a border) and for rows whose 127 / a is no ordinary number the quotient is taken in 64 bits: two 24-bit numbers' quotient that is not a tie is
// 2^-25 of itself away from one at least.
__device__ __forceinline__ int i8_code(float x, float a, float r) {
    const float y = x * r, n = rintf(y);
    if (fabsf(y - n) < 0.499f && a > 1e-30f) return (int)n;
    return (int)rint((double)x * 127.0 / (double)a);
}
#define I8_THREADS 256
// codes [T][kp], zeros behind a row's k; factors [T].  A CTA a row
__global__ void __launch_bounds__(I8_THREADS) i8_rows_kernel(const float* __restrict__ x, int64_t rs, int k, int kp, int8_t* __restrict__ codes, float* __restrict__ factors) {
    __shared__ unsigned tops[I8_THREADS / 32];
    pdl_enter();
    const int64_t t = blockIdx.x;
    const float* row = x + t * rs;
    unsigned top = 0;
    for (int c = threadIdx.x; c < k; c += I8_THREADS) top = max(top, __float_as_uint(row[c]) & 0x7fffffffu);
    top = __reduce_max_sync(0xffffffffu, top);
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < I8_THREADS / 32; w++) top = max(top, tops[w]);
    const bool finite = top < 0x7f800000u;
    const float a = __uint_as_float(top), r = 127.0f / a;
    for (int c = threadIdx.x; c < kp; c += I8_THREADS) codes[t * kp + c] = c < k && finite && top ? (int8_t)i8_code(row[c], a, r) : (int8_t)0;
    if (threadIdx.x == 0) factors[t] = finite ? a / 127.0f : NAN;
}

// ---- few rows: a warp an output channel ------------------------------------------------------------------------------------------------------
#define I8_ROWS 8
__global__ void __launch_bounds__(I8_THREADS) i8_few_kernel(const int8_t* __restrict__ w, const float* __restrict__ ws, const int8_t* __restrict__ x, const float* __restrict__ xs,
                                                            float* __restrict__ out, int T, int m, int k, int kp) {
    pdl_enter();
    const int lane = threadIdx.x & 31, t0 = blockIdx.y * I8_ROWS, n = min(I8_ROWS, T - t0);
    const int64_t row = (int64_t)blockIdx.x * (I8_THREADS / 32) + (threadIdx.x >> 5);
    if (row >= m) return;
    const int8_t* wr = w + row * k;
    const bool vec = k % 16 == 0;
    int acc[I8_ROWS];
#pragma unroll
    for (int i = 0; i < I8_ROWS; i++) acc[i] = 0;
    for (int c = lane * 16; c < k; c += 512) {
        int4 u;
        if (vec) u = ld_stream_16(wr + c);
        else {
            int z[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 16; j++)
                if (c + j < k) z[j / 4] |= (int)(uint8_t)wr[c + j] << (j % 4 * 8);
            u = make_int4(z[0], z[1], z[2], z[3]);
        }
#pragma unroll
        for (int i = 0; i < I8_ROWS; i++) {
            if (i >= n) break;
            const int4 v = *(const int4*)(x + (int64_t)(t0 + i) * kp + c);
            acc[i] = __dp4a(u.x, v.x, __dp4a(u.y, v.y, __dp4a(u.z, v.z, __dp4a(u.w, v.w, acc[i]))));
        }
    }
#pragma unroll
    for (int i = 0; i < I8_ROWS; i++) acc[i] = warp_sum_i(acc[i]);
    if (lane == 0)
        for (int i = 0; i < n; i++) out[(int64_t)(t0 + i) * m + row] = (float)acc[i] * ws[row] * xs[t0 + i];
}

extern "C" CC_API int cc_product_i8(cc_device* dev, const cc_view* w, const cc_view* w_scale, const cc_view* x, cc_buf** out) {
    if (!dev) return CC_ERR_ARG;
    CC_ENTER(dev);
    if (LAZY(dev)) return cc_fail(dev, CC_ERR_UNSUPPORTED, "product_i8: not available on a lazy (graph / megakernel) device");
    if (!out) return cc_fail(dev, CC_ERR_ARG, "product_i8: out is NULL");
    *out = nullptr;
    if (!view_ok(w) || !view_ok(w_scale) || !view_ok(x)) return cc_fail(dev, CC_ERR_ARG, "product_i8: bad tensor view");
    CC_REQUIRE(dev, view_in_bounds(w) && view_in_bounds(w_scale) && view_in_bounds(x), "product_i8: a view addresses elements behind its buffer");
    CC_REQUIRE(dev, w->buf->dev == dev && w_scale->buf->dev == dev && x->buf->dev == dev, "product_i8: a tensor of another device");
    CC_REQUIRE(dev, w->buf->dtype == CC_I8 && w->ndim == 2 && view_contiguous(w), "product_i8: w is not a contiguous I8 matrix");
    REQUIRE_F32(dev, w_scale, "product_i8 w_scale"); REQUIRE_F32(dev, x, "product_i8 x");
    const int64_t m = w->shape[0], k = w->shape[1], T = x->shape[0];
    CC_REQUIRE(dev, view_contiguous(w_scale) && view_len(w_scale) == m, "product_i8: w_scale is not [%lld]", (long long)m);
    CC_REQUIRE(dev, x->ndim == 2 && x->shape[1] == k && x->strides[1] == 1 && x->strides[0] >= k, "product_i8: x is not rows of %lld", (long long)k);
    CC_REQUIRE(dev, k >= 1 && k <= 131072 && m < ((int64_t)1 << 30) && T < ((int64_t)1 << 24), "product_i8: %lld rows, %lld x %lld", (long long)T, (long long)m, (long long)k);
    cc_buf* o = nullptr;
    int rc = cc_new_activation(dev, T * m, CC_F32, false, &o);
    if (rc) return rc;
    if (T > 0 && m > 0) {
        const int kp = (int)((k + 15) / 16 * 16);
        void* ws = nullptr; size_t cls = 0;
        const size_t codes = ((size_t)T * kp + 255) / 256 * 256;
        rc = cc_pool_alloc(dev, codes + (size_t)T * 4, &ws, &cls);
        if (rc) { cc_tensor_release(o); return rc; }
        int8_t* xq = (int8_t*)ws;
        float* xs = (float*)((uint8_t*)ws + codes);
        cudaError_t e = cc_launch_pdl(dev, i8_rows_kernel, (unsigned)T, I8_THREADS, 0, (const float*)x->buf->plane[0], x->strides[0], (int)k, kp, xq, xs);
        dev->launches++;
        if (e == cudaSuccess) {
            e = cc_launch_pdl(dev, i8_few_kernel, dim3((unsigned)((m + I8_THREADS / 32 - 1) / (I8_THREADS / 32)), (unsigned)((T + I8_ROWS - 1) / I8_ROWS)), I8_THREADS, 0,
                              (const int8_t*)w->buf->plane[0], (const float*)w_scale->buf->plane[0], xq, xs, (float*)o->base, (int)T, (int)m, (int)k, kp);
            dev->launches++;
        }
        cc_pool_free(dev, ws, cls);
        if (e != cudaSuccess) { cc_tensor_release(o); return cc_fail(dev, CC_ERR_CUDA, "product_i8: %s", cudaGetErrorString(e)); }
    }
    *out = o;
    return CC_OK;
}
