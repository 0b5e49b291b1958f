// Products of 8-bit rows with packed weights: what the C ABI hands to the
// per-format launch units.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "quant_studio.h"

namespace qsl {

// A few rows take dot products (takes_few), more tiles that decode the weight
// themselves, or both factors laid out for the matrix units (takes_matrix).

constexpr int few_record(int t) { return 3 * t + (3 * t + 1) % 2; }     // 16s of a group of x
constexpr int FEW_LDS = 160 * 1024, FEW_GRID = 4096;    // bytes of a CU, and of the largest code book
// Up to 8 rows, 4 where they are long, of which four weight rows and the rows
// themselves fit in LDS. us, and of a tile: 8 rows with q6_k 151,936 x 2,560 133 and
// 161, q4_k 9,728 x 2,560 15.9 and 15.6, q4_0 1,024 x 2,560 7.7 and 8.2, q6_k 2,560 x
// 9,728 28 and 20, 5 of those 22 and 19.
inline bool takes_few(int64_t row_bytes, int64_t t, int64_t k) {
    if (t > (k > 4096 ? 4 : 8)) return false;
    return 4 * row_bytes + 48 + k / 32 * few_record(t <= 6 ? (int)t : 8) * 16 + FEW_GRID <= FEW_LDS;
}

struct LinearArgs {
    const uint8_t* w;       // n rows of row_bytes
    const int8_t* q;        // t rows of k codes
    const float* s;         // t rows of k / 32 scales
    void* dst;              // t rows of n values of dst_type
    int64_t row_bytes, n, k, t;
    int dst_type;           // QS_SRC_*
    bool f16;               // laid-out factors are rounded to f16 (takes_f16)
    // low-rank adapters: ids is null without them
    const int32_t* ids;     // adapter of each row; outside 0..adapters-1: none
    const int32_t* off;     // adapters + 1 rank offsets, multiples of 8
    const uint16_t* b;      // adapter i: n rows of its rank, from n * off[i]
    int64_t ldv;
    int32_t adapters;
    int b_type;             // QS_SRC_F16 / QS_SRC_BF16
    const float* v;         // dot products: scale * A x, t rows of ldv
    const float* delta;     // tiles: B v, t rows of n
    float* parts;           // of a product split over its groups: splits x t rows of n
    int splits;
    // laid-out factors: scale * A x as hi + lo (+ rest: exact codes), t rows of ldv
    const uint16_t *v_hi, *v_lo, *v_rest;
    const float* v_unit;            // and what that is to be multiplied by (F16), t rows of ldv / 32
};

// Many rows: both factors are laid out for the matrix units first, in `work`.
// A weight is taken in slices of at most SLICE values, whose layout the 256 MB
// cache behind the L2s holds.
constexpr int64_t SLICE = INT64_C(1) << 26;
constexpr int STAGE_GROUPS = 8, STAGE_GROUPS16 = 8, TILE = 256;     // a row's groups are laid out in whole eights

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
    int64_t scale_bytes;        // of the factors' row scales (F16)
    int64_t x_bytes, w_bytes;   // of the layouts
    int64_t bytes() const { return scale_bytes + x_bytes + w_bytes; }
};
inline int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
// f16: the layout of qs_matrix16.h, else that of qs_matrix.h
inline MatrixPlan matrix_plan(int type, bool f16, int64_t n, int64_t k, int64_t t) {
    MatrixPlan p;
    p.groups = (int)round_up(k / 32, f16 ? STAGE_GROUPS16 : STAGE_GROUPS);
    const int64_t rows = SLICE / k / TILE * TILE, all = round_up(n, TILE), panels = round_up(t, TILE) / 32;
    p.slice = rows < TILE ? TILE : rows < all ? rows : all;
    p.scale_bytes = f16 ? round_up((t + p.slice) * 4, 256) : 0;
    p.x_bytes = panels * p.groups * (f16 ? 2048 : panel_group_bytes(1, minima(type)));
    p.w_bytes = p.slice / 32 * p.groups * (f16 ? 2048 : panel_group_bytes(two_planes(type) ? 2 : 1, minima(type)));
    return p;
}
inline int64_t tile_count(int64_t t, int64_t n, int bm, int bn) { return ((t + bm - 1) / bm) * ((n + bn - 1) / bn); }
// Tiles that decode the weight for each 64 rows save its layout's way through
// memory, as long as one round of 64 x 64 takes them all, or a split half a round
// where rows are long. us of tiles and of laid-out factors: 128 rows with q4_k
// 9,728 x 2,560 38 and 38; 192 with q6_k 2,560 x 9,728 51 and 90; 256 with q4_0
// 4,096 x 4,096 26 and 36; 512 with 1,024 x 2,560 14 and 23, with 8 adapters of
// rank 64 32 and 40; but 320 with 4,096 x 4,096 46 and 41, 512 with q6_k 2,048 x
// 9,728 90 and 87, 71 with factors of f16. Above 512 rows the adapters' products row by row lose.
inline bool takes_matrix(int64_t t, int64_t n, int64_t k) {
    const int64_t tiles = tile_count(t, n, 64, 64);
    return t > 512 || (t > 128 && tiles > (k <= 4096 ? 256 : 128));
}

// Large products whose result is bf16 (8 bits) take factors of f16 (11 bits) where
// the caller leaves that open (`dst` without QS_EXACT); everything else exact codes.
// F16 factors are laid out in two launches and twice the bytes, and multiplied at up
// to 1.0 PFLOP/s where exact codes reach 0.8, 0.64 with minima. q4_k, us f16 and
// exact: 512 rows, 2,560 x 2,560 40 and 34; 2,048, 1,024 x 2,560 41 and 35; 1,024,
// 2,560 x 2,560 41 and 49; 300, 9,728 x 2,560 52 and 54; 4,096, 9,728 x 2,560 215
// and 336. Rows under 1,024 values do not repay a launch more: 2,000 rows, 3,000 x
// 256 33 and 18.
inline bool takes_f16(int dst, int64_t t, int64_t n, int64_t k) {
    return dst == QS_SRC_BF16 && takes_matrix(t, n, k) && k >= 1024 && t * n >= INT64_C(3) * (INT64_C(1) << 31) / k;
}

// Tiles of a product of laid-out factors, and the time measured for a round of
// as many as the 256 CUs hold, in tenths of a microsecond at rows of 2,560
// values (it grows with the rows).
struct Tiles {
    int bm, bn, held, cost;
};

// F16 factors. Larger tiles do more per LDS byte (256 x 320: 1.02 PFLOP/s where
// they fill the chip, 64 x 64: 0.46). Adapters need registers that 160 columns a
// wave do not leave, and with them a CU has registers for one workgroup of 64 x 64.
constexpr Tiles TILES16[] = {{256, 320, 256, 1000}, {256, 256, 256, 770}, {128, 160, 256, 385}, {128, 96, 256, 258},
                             {64, 64, 512, 227}};
constexpr int MOST_PARTS = 4;
struct Choice16 {
    int tile, splits;
};
// The tile, and the parts of the groups, that cost least: few tiles leave CUs
// idle, each of the rest waiting for its copies; parts cost what writing and
// joining their f32 sums takes, 12 bytes of each at 4 TB/s, and two launches'
// ends. us of a call: 509 rows with q5_k 2,560 x 9,728 71 in four parts of 128 x
// 160, 88 whole in 64 x 64; 2,047 rows with q6_k 160 in three parts of 256 x 256,
// 152 whole in 128 x 160, which the rule takes.
inline Choice16 choose16(bool adapted, int64_t t, int64_t n, int64_t k, int most) {
    Choice16 best{};
    double least = 1e300;
    for (int i = adapted ? 1 : 0; i < 5; i++)
        for (int s = 1; s <= most; s++) {
            const int64_t pairs = (k / 32 + 7) / 8, per = (pairs + s - 1) / s;
            if ((s - 1) * per >= pairs) continue;       // of stages: no part is empty
            const Tiles& c = TILES16[i];
            const int64_t held = adapted && c.held > 256 ? 256 : c.held, rounds = (tile_count(t, n, c.bm, c.bn) * s + held - 1) / held;
            const double cost = (double)rounds * c.cost * (double)k / (2560.0 * s) +
                                (s > 1 ? (adapted ? 100 : 40) + (double)(t * n) * 12 * s / 4e5 : 0);
            if (cost < least) least = cost, best = {i, s};
        }
    return best;
}

// Parts that a product that is not laid out is split into over its groups, so
// that there are two workgroups of 64 x 32 for every CU (where they are 64 x 64,
// one); a part is whole stages of 8 groups. us whole, in up to 4 parts and in up to
// 8: 61 rows with q8_0 1,024 x 2,560 14.3, 10.3 and 9.6; 64 with q6_k 2,560 x 9,728
// 90, 31 and 27. Parts for twice the workgroups: 9.5 and 37.
inline int tile_splits(int64_t t, int64_t n, int64_t k) {
    const int64_t tiles = (t + 63) / 64 * ((n + 31) / 32), stages = (k / 32 + 7) / 8;
    int64_t s = 512 / tiles < 8 ? 512 / tiles : 8;
    s = s < stages ? s : stages;
    if (s < 2) return 1;
    const int64_t per = (stages + s - 1) / s;
    return (int)((stages + per - 1) / per);
}
hipError_t launch_join(const LinearArgs& a, hipStream_t st);

template <int TYPE>
hipError_t launch_linear(const LinearArgs& a, void* work, hipStream_t st);

struct MatrixArgs {
    LinearArgs l;
    const uint8_t *xl, *wl;     // laid out: all rows; the weight's rows first .. first + count
    int64_t first, count;
    int groups;                 // as laid out
};
hipError_t launch_matrix(int planes, int mins, const MatrixArgs& a, hipStream_t st);

struct Matrix16Args {
    LinearArgs l;
    const uint8_t *xl, *wl;
    const float *ws, *xs;       // row scales
    int64_t first, count;       // the weight's rows of this slice
    int groups;                 // as laid out
};
hipError_t launch_matrix16(const Matrix16Args& a, hipStream_t st);

struct AdapterArgs {
    const int8_t* q;
    const float* s;
    const uint16_t *a, *b;      // adapter i: rows off[i] .. off[i + 1] of k; n rows of its rank from n * off[i]
    const int32_t *ids, *off;
    const float* scales;
    float* v;                   // [t][ldv]
    uint16_t *hi, *lo, *rest;   // v as a sum of values of the adapters' type: [t][ldv]; rest is null for factors of f16
    float* unit;                // what that is to be multiplied by (F16): [t][ldv / 32]
    float* delta;               // [t][n]
    float* sums;                // [parts][t][ldv]
    int64_t k, n, t, ldv;
    int32_t adapters;
    int parts;
    bool few;                   // the product takes v itself
};
// Parts that the rows' values are split into: up to 1,024 workgroups, where a
// row has 512 values or more for each. The CUs hold 512 at a time; parts half as
// long leave less to the 32 rows that have two adapters (us of a call, 2,047 rows
// with q6_k 2,560 x 9,728, ranks to 128: 211 for 512 workgroups, 196 for 1,024, 212
// unsplit).
inline int adapter_parts(int64_t t, int64_t k, int64_t ldv) {
    const int64_t blocks = (t + 31) / 32 * ((ldv + 31) / 32), p = 1024 / blocks < k / 512 ? 1024 / blocks : k / 512;
    return p < 1 ? 1 : (int)p;
}
hipError_t launch_adapters(int type, const AdapterArgs& a, hipStream_t st);

}  // namespace qsl
