// half_types.cuh -- activations of 16 bits beside those of 32 (product.cu, latent.cu): reading and writing runs of 8 numbers of any of the three types, and the checks of their views.
#pragma once
#include <cuda_bf16.h>
#include <math.h>

#include "capi_checks.cuh"

static inline bool ht_plain(int t) { return t == CC_F32 || t == CC_F16 || t == CC_BF16; }
static inline int ht_size(int t) { return t == CC_F32 ? 4 : 2; }

// rows of a matrix of this device, any row stride that holds a row
#define HT_ROWS(dev, v, what)                                                                                                                      \
    do {                                                                                                                                           \
        if (!view_ok(v)) return cc_fail((dev), CC_ERR_ARG, "%s: bad tensor view", what);                                                           \
        if (!view_in_bounds(v)) return cc_fail((dev), CC_ERR_TENSOR, "%s: view addresses element %lld of a buffer of %lld", what,                   \
                                               (long long)view_max_offset(v), (long long)(v)->buf->nelems);                                        \
        CC_REQUIRE(dev, (v)->buf->dev == (dev), "%s: a tensor of another device", what);                                                           \
        CC_REQUIRE(dev, ht_plain((v)->buf->dtype), "%s: not f32, f16 or bf16, but type %d", what, (v)->buf->dtype);                                \
        CC_REQUIRE(dev, (v)->ndim == 2 && (v)->strides[1] == 1 && (v)->strides[0] >= (v)->shape[1], "%s: not rows of a matrix", what);             \
    } while (0)
// a contiguous tensor of this device
#define HT_WHOLE(dev, v, type, what)                                                                                                               \
    do {                                                                                                                                           \
        if (!view_ok(v)) return cc_fail((dev), CC_ERR_ARG, "%s: bad tensor view", what);                                                           \
        CC_REQUIRE(dev, view_in_bounds(v) && view_contiguous(v) && (v)->buf->dev == (dev) && (v)->buf->dtype == (type),                            \
                   "%s: not a contiguous tensor of type %d on this device, inside its buffer", what, (int)(type));                                 \
    } while (0)

#ifdef __CUDACC__
// rounded to 16 bits; finite numbers beyond the range of f16 become its largest, infinities and NaN stay (max and min of the hardware drop NaN)
__device__ __forceinline__ float ht_clamp(float x) { return fabsf(x) < INFINITY ? fminf(fmaxf(x, -65504.0f), 65504.0f) : x; }
__device__ __forceinline__ unsigned ht_pack_f16(float x, float y) {
    const __half2 h = __floats2half2_rn(ht_clamp(x), ht_clamp(y));
    return *(const unsigned*)&h;
}
__device__ __forceinline__ unsigned ht_pack_bf16(float x, float y) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
    return *(const unsigned*)&h;
}
__device__ __forceinline__ float ht_read(const void* p, int64_t i, int type) {
    return type == CC_F32 ? ((const float*)p)[i] : type == CC_F16 ? __half2float(((const __half*)p)[i]) : __bfloat162float(((const __nv_bfloat16*)p)[i]);
}
__device__ __forceinline__ void ht_write(void* p, int64_t i, int type, float x) {
    if (type == CC_F32) ((float*)p)[i] = x;
    else if (type == CC_F16) ((__half*)p)[i] = __float2half_rn(ht_clamp(x));
    else ((__nv_bfloat16*)p)[i] = __float2bfloat16_rn(x);
}
// 8 neighbouring numbers; vec: they start at a multiple of 16 bytes
__device__ __forceinline__ void ht_read8(const void* p, int64_t i, int type, bool vec, float (&v)[8]) {
    if (!vec) {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = ht_read(p, i + j, type);
    } else if (type == CC_F32) {
        const float4 a = *(const float4*)((const float*)p + i), b = *(const float4*)((const float*)p + i + 4);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
        const uint4 u = *(const uint4*)((const uint16_t*)p + i);
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (type == CC_F16) {
                const float2 f = __half22float2(*(const __half2*)&w[j]);
                v[2 * j] = f.x; v[2 * j + 1] = f.y;
            } else {
                v[2 * j] = __uint_as_float(w[j] << 16); v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            }
        }
    }
}
#endif
