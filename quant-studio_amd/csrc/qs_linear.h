// Products of 8-bit rows with packed weights: what the C ABI hands to the
// per-format launch units.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "quant_studio.h"

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

// Many rows: both factors are laid out for the matrix units first, in `work`.
// A weight is taken in slices of at most SLICE values, whose layout the 256 MB
// cache behind the L2s holds.
constexpr int64_t SLICE = INT64_C(1) << 26;
constexpr int STAGE_GROUPS = 2, TILE = 128;

constexpr bool two_planes(int type) { return type == QS_TYPE_Q6_K || type == QS_TYPE_IQ2_XS || type == QS_TYPE_IQ2_S; }
constexpr int minima(int type) {
    return type == QS_TYPE_Q2_K ? 2
           : type == QS_TYPE_Q4_1 || type == QS_TYPE_Q5_1 || type == QS_TYPE_Q4_K || type == QS_TYPE_Q5_K ? 1
                                                                                                          : 0;
}
// bytes of a group of a panel of 32 rows (qs_matrix.h)
constexpr int panel_group_bytes(int planes, int mins) { return planes * 1024 + (1 + mins) * 256; }

struct MatrixPlan {
    int64_t slice;              // weight rows of a slice, a multiple of TILE
    int groups;                 // of a row, rounded up to whole stages
    int64_t x_bytes, w_bytes;   // of the layouts
};
inline MatrixPlan matrix_plan(int type, int64_t n, int64_t k, int64_t t) {
    MatrixPlan p;
    p.groups = (int)((k / 32 + STAGE_GROUPS - 1) / STAGE_GROUPS * STAGE_GROUPS);
    const int64_t rows = SLICE / k / TILE * TILE, all = (n + TILE - 1) / TILE * TILE;
    p.slice = rows < TILE ? TILE : rows < all ? rows : all;
    p.x_bytes = (t + TILE - 1) / TILE * (TILE / 32) * p.groups * panel_group_bytes(1, minima(type));
    p.w_bytes = p.slice / 32 * p.groups * panel_group_bytes(two_planes(type) ? 2 : 1, minima(type));
    return p;
}
// whether a product takes that way
inline bool takes_matrix(int64_t t) { return t > 128; }

template <int TYPE>
hipError_t launch_linear(const LinearArgs& a, void* work, hipStream_t st);

struct MatrixArgs {
    LinearArgs l;
    const uint8_t *xl, *wl;     // laid out: all rows; the weight's rows first .. first + count
    int64_t first, count;
    int groups;                 // as laid out
};
hipError_t launch_matrix(int planes, int mins, const MatrixArgs& a, hipStream_t st);

}  // namespace qsl
