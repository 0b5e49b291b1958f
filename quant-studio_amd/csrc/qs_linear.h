// Products of 8-bit rows with packed weights: what the C ABI hands to the
// per-format launch units.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qsl {

struct LinearArgs {
    const uint8_t* w;       // n rows of row_bytes
    const int8_t* q;        // t rows of k codes
    const float* s;         // t rows of k / 32 scales
    void* dst;              // t rows of n values of dst_type
    int64_t row_bytes, n, k, t;
    int dst_type;           // QS_SRC_*
    // low-rank adapters: ids is null without them
    const int32_t* ids;     // adapter of each row; outside 0..adapters-1: none
    const int32_t* off;     // adapters + 1 rank offsets, multiples of 8
    const uint16_t* b;      // adapter i: n rows of its rank, from n * off[i]
    const float* v;         // t rows of ldv: scale * A x
    int64_t ldv;
    int32_t adapters;
    int b_type;             // QS_SRC_F16 / QS_SRC_BF16
};

template <int TYPE>
hipError_t launch_linear(const LinearArgs& a, hipStream_t st);

}  // namespace qsl
