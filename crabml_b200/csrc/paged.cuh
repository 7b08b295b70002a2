// paged.cuh -- the plan of a step over several sequences (include/crabml_paged.h): what the host checked once, and its copy on the device that the kernels of
// paged.cu and paged_attn.cu read.
#pragma once
#include "capi_checks.cuh"
#include "paged_plan.hpp"

struct cc_page_plan {
    cc_device* dev = nullptr;
    int n_seqs = 0, page = 0, shift = 0, table_cols = 0, n_items = 0, n_segments = 0;
    int64_t n_pages = 0, n_slots = 0, tokens = 0;
    std::vector<PgSeq> seqs;
    void* base = nullptr; size_t cls = 0;                // the device's copy
    const PgSeq* d_seqs = nullptr;
    const PgSegment* d_segments = nullptr;
    const int* d_table = nullptr;
};

// the views of a cache after its checks
struct PgCache {
    uint8_t *k, *v;
    float *ks, *vs;
    __half *ko, *vo;
    int G, dk, dv;
    bool i8;
};
int pg_check_cache(cc_device* dev, const cc_page_plan* plan, const cc_paged_cache* c, const char* what, PgCache* out);

#define PG_ENTER(dev, plan, what)                                                                                                                  \
    if (!(dev) || !(plan)) return CC_ERR_ARG;                                                                                                      \
    CC_ENTER(dev);                                                                                                                                 \
    if (LAZY(dev)) return cc_fail((dev), CC_ERR_UNSUPPORTED, "%s: not available on a lazy (graph / megakernel) device", what);                    \
    CC_REQUIRE(dev, (plan)->dev == (dev), "%s: the plan is another device's", what)
// rows of a matrix of this device, any row stride that holds a row
#define PG_ROWS(dev, v, what)                                                                                                                      \
    do {                                                                                                                                           \
        if (!view_ok(v)) return cc_fail((dev), CC_ERR_ARG, "%s: bad tensor view", what);                                                           \
        if (!view_in_bounds(v)) return cc_fail((dev), CC_ERR_TENSOR, "%s: view addresses element %lld of a buffer of %lld", what,                   \
                                               (long long)view_max_offset(v), (long long)(v)->buf->nelems);                                        \
        CC_REQUIRE(dev, (v)->buf->dev == (dev), "%s: a tensor of another device", what);                                                           \
        REQUIRE_F32(dev, v, what);                                                                                                                 \
        CC_REQUIRE(dev, (v)->ndim == 2 && (v)->strides[1] == 1 && (v)->strides[0] >= (v)->shape[1], "%s: not rows of a matrix", what);             \
    } while (0)
