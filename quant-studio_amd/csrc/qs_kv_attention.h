// Attention of new tokens over a quantised, paged cache: what its C entry and
// its kernels share.
#pragma once

#include <hip/hip_runtime.h>

#include "qs_kv.h"
#include "qs_rows.h"

namespace qskv {

// checks a cache of the C ABI and fills in `c`; 0, or the error's code
int cache_of(const qs_kv_cache* cache, Cache& c);


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

// Queries of a workgroup, of a key/value head's group * fresh: eight, for each of which a
// matrix product has two of its 16 columns, or twice as many, which read and unpack the
// head once and not twice, where there are so many and a wave's registers hold them (8
// sequences of 8,000 slots, 12 queries of each head: 49.7 us, 56.3 in eights).
inline __host__ __device__ int columns_of(const AttentionArgs& a) {
    return a.group * a.fresh > 8 && a.c.blocks <= 4 && a.type != QS_SRC_F32 ? 16 : 8;
}
inline __host__ __device__ int column_tiles(const AttentionArgs& a) {
    return (a.group * a.fresh + columns_of(a) - 1) / columns_of(a);
}

// A code c of the matrix products is c 2^-CODE_POWER, a normal f16; ONCE times a sum of
// products with values' codes is the sum.
constexpr int CODE_POWER = 9;
constexpr float ONCE = 1 << CODE_POWER;

// A running maximum is -infinity where a query sees nothing, else LOWEST or more. What its sums
// are to be multiplied by: nothing seen gives zeros, scores of -infinity alone give no values.
constexpr float LOWEST = -0x1.fffffep127f;
QS_DEV float inverse_of(float top, float total) {
    return total != 0.0f ? ONCE / total : top >= LOWEST ? __builtin_nanf("") : 0.0f;
}

// How a call's work is split, and where its workgroups leave what is joined.
constexpr int TILE = 32;            // slots of a wave's step
// Steps of its waves that a workgroup takes as long to begin with another segment: 61 ragged
// sequences of up to 2,047 slots take 77 us with 0, 32.3 with 2, 35.6 with 8.
constexpr int OPENING = 2;
// Workgroups of four waves that a CU holds, by the registers of a wave. More workgroups than
// these would wait for others to end (8 sequences of 16,000 slots 61.9 us, one more 64.0; of
// 64-value heads 38.9 and 43.8), and fewer registers for more of them would not do: heads of
// 64 65 us, 79 with one more and 66 with one less, sixteen queries of them 55, 102 and 55; of
// 128 63, 89 and 63, sixteen 52, 139 and 59, f32 68, 71 and 71; of 192 42, 64 and 45, f32
// 44.5 and 45.4 with one more. f32 ones of 256 need some 350 registers.
__host__ __device__ constexpr int resident(int blocks, int columns, bool wide) {
    return blocks == 2 ? (columns == 16 ? 3 : 4) : blocks == 4 ? (wide || columns == 16 ? 2 : 3) : wide ? 1 : 2;
}
struct Split {
    int32_t groups, waves;          // workgroups, waves in each: 4, which take steps in turn, or 1
    int32_t share;                  // workgroups of a head's and column tile's steps of a sequence, 1: they take all;
                                    // 0: they take equal runs of all steps of the call
    // of each workgroup, first for a segment that begins before it, then for one that goes on after it
    float* parts;                   // [groups][2][columns][head size], sums relative to the maximum, in units of ONCE
    float2* stats;                  // [groups][2][columns]: maximum, sum of p
    // Of runs: segments that more than one workgroup has, as sequence, head and column tile, first and last
    // workgroup (-1: it is one's alone). One entry for each head and column tile of a sequence where these
    // are no more than workgroups (`listed`), else one for that which goes on after each workgroup.
    int4* segments;
    int32_t listed;
    int64_t bytes;                  // of the workspace
};
Split split_of(const AttentionArgs& a, void* workspace);

// two values of a result's row
QS_DEV void store_two(const AttentionArgs& a, int64_t at, float x, float y) {
    if (a.type == QS_SRC_F32) *reinterpret_cast<float2*>(static_cast<float*>(a.out) + at) = float2{x, y};
    else *reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.out) + at) =
        a.type == QS_SRC_BF16 ? qsr::bits16<qs::SRC_BF16>(x) | qsr::bits16<qs::SRC_BF16>(y) << 16
                              : qsr::bits16<qs::SRC_F16>(x) | qsr::bits16<qs::SRC_F16>(y) << 16;
}
// first value of a query's row of the result; -1: the column has no query
QS_DEV int64_t row_of(const AttentionArgs& a, int seq, int head, int column) {
    if (column >= a.group * a.fresh) return -1;
    const int token = column / a.group;
    return ((((int64_t)seq * a.fresh + token) * a.c.heads + head) * a.group + column - token * a.group) * (32 * a.c.blocks);
}

hipError_t launch_join(const AttentionArgs& a, const Split& split, hipStream_t st);

template <int K_BITS, int V_BITS>
hipError_t launch_attention(const AttentionArgs& a, const Split& split, hipStream_t st);

}  // namespace qskv
