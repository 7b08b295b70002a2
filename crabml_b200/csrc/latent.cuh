// latent.cuh -- layers whose keys and values all heads make of one latent row a token, over pages (include/crabml_paged.h): what the append and the attention share.
#pragma once
#include "half_types.cuh"
#include "paged.cuh"

#define LT_RANK 512                           // largest rank,
#define LT_REST 64                            // .. rotated part of a row,
#define LT_DIM 256                            // .. and columns of a head beside it, or of its values

// a layer's pages after their checks
struct LtPages { __half* rows; int rank, rest, cols; };
int lt_check_pages(cc_device* dev, const cc_page_plan* plan, const cc_view* pages, int32_t rank, const char* what, LtPages* out);
