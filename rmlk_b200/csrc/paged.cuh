// The paged 8-bit cache, as its two kernels (paged_append.cu, paged_attention.cu) see it.
#pragma once

#include "common.cuh"

namespace rmlk {
namespace paged {

struct Cache {
    int8_t *k, *v;
    float *ks, *vs;
    int pages, kv_heads, page, page_log, d;
};

// The sequences of a call: new tokens [starts[b], starts[b + 1]) or `each` per sequence; lengths count them.
struct Batch {
    const int32_t *starts, *lens, *table;
    int64_t width;
    int64_t tokens;
    int batch, each;

    // Rows of sequence b.  What `starts` may hold beyond the rows of the call is cut off.
    __device__ __forceinline__ void rows(int b, int64_t& first, int64_t& count) const {
        if (!starts) {
            first = static_cast<int64_t>(b) * each;
            count = each;
        } else {
            first = min(max(static_cast<int64_t>(starts[b]), int64_t(0)), tokens);
            count = max(min(static_cast<int64_t>(starts[b + 1]), tokens) - first, int64_t(0));
        }
    }
};

// Checks that the entry points share; fills `c` and `q`.
int take(const char* what, const rmlk_paged_cache* cache, int64_t tokens, int64_t batch, const int32_t* starts, const int32_t* lens, const int32_t* table, int64_t table_width,
         Cache& c, Batch& q);

}  // namespace paged
}  // namespace rmlk
