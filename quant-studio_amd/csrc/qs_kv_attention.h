// Attention of new tokens over a quantised, paged cache: what its C entry and
// its kernels share.
#pragma once

#include <hip/hip_runtime.h>

#include "qs_kv.h"

namespace qskv {

// checks a cache of the C ABI and fills in `c`; 0, or the error's code
int cache_of(const qs_kv_cache* cache, Cache& c);

constexpr int COLUMNS = 8;          // queries of a workgroup: a matrix product's 16 columns are two for each

struct AttentionArgs {
    Cache c;
    const void* q;
    void* out;                      // contiguous
    const int32_t *tables, *lengths;
    int64_t q_stride, table_stride; // q's between tokens, in values
    int32_t batch, fresh, group;    // fresh: new tokens of a sequence; group: query heads of a key/value head
    int32_t pages_each;             // columns of the tables
    int32_t window;                 // 0: none
    int32_t type;                   // of q and out (QS_SRC_*)
    float scale;
};

// one workgroup's queries: COLUMNS of a key/value head's group * fresh
inline __host__ __device__ int column_tiles(const AttentionArgs& a) {
    return (a.group * a.fresh + COLUMNS - 1) / COLUMNS;
}

template <int K_BITS, int V_BITS>
hipError_t launch_attention(const AttentionArgs& a, hipStream_t st);

}  // namespace qskv
