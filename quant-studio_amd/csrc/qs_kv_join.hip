// Joins what workgroups of the attention left of sequences that were split.
#include "qs_kv_attention.h"
#include "qs_launch_kernel.h"

namespace qskv {

typedef float f32x4 __attribute__((ext_vector_type(4)));

// The parts of the segments that began in one workgroup and ended in another:
// grid (workgroups, columns). D / 4 threads take a part's row, the others the next
// parts; every thread keeps a running maximum, and LDS joins them in a fixed order.
template <int BLOCKS>
__global__ __launch_bounds__(256) void k_kv_join(AttentionArgs a, Split split) {
    const int4 s = split.segments[blockIdx.x];
    if (s.z < 0) return;
    constexpr int D = 32 * BLOCKS, LANES = D / 4, ROWS = 256 / LANES;
    __shared__ f32x4 acc[ROWS][LANES];
    __shared__ float2 stats[ROWS];
    const int tiles = column_tiles(a), head = s.y / tiles, column = (int)blockIdx.y;
    const int64_t row = row_of(a, s.x, head, (s.y - head * tiles) * COLUMNS + column);
    if (row < 0) return;
    const int mine = (int)threadIdx.x / LANES, lane = (int)threadIdx.x - mine * LANES;
    const int count = s.z - (int)blockIdx.x + 1;
    f32x4 sum{0, 0, 0, 0};
    float ref = -__builtin_inff(), total = 0.0f;
    if (mine < ROWS) {
#pragma unroll 4
        for (int i = mine; i < count; i += ROWS) {
            const int64_t slot = ((int64_t)(blockIdx.x + i) * 2 + (i == 0)) * COLUMNS + column;
            const float2 part = split.stats[slot];
            const f32x4 v = *reinterpret_cast<const f32x4*>(split.parts + slot * D + 4 * lane);
            const float top = fmaxf(ref, part.x);
            const float was = ref > -__builtin_inff() ? __builtin_amdgcn_exp2f(ref - top) : 0.0f;
            const float is = part.x > -__builtin_inff() ? __builtin_amdgcn_exp2f(part.x - top) : part.y;    // 0, or NaN
#pragma unroll
            for (int j = 0; j < 4; j++) sum[j] = __builtin_fmaf(v[j], is, sum[j] * was);
            total = __builtin_fmaf(part.y, is, total * was);
            ref = top;
        }
        acc[mine][lane] = sum;
        if (lane == 0) stats[mine] = float2{ref, total};
    }
    __syncthreads();
    if ((int)threadIdx.x >= LANES) return;
    ref = -__builtin_inff();
#pragma unroll
    for (int i = 0; i < ROWS; i++) ref = fmaxf(ref, stats[i].x);
    sum = f32x4{0, 0, 0, 0};
    total = 0.0f;
#pragma unroll
    for (int i = 0; i < ROWS; i++) {
        const float2 part = stats[i];
        const float is = part.x > -__builtin_inff() ? __builtin_amdgcn_exp2f(part.x - ref) : part.y;
        total = __builtin_fmaf(part.y, is, total);
#pragma unroll
        for (int j = 0; j < 4; j++) sum[j] = __builtin_fmaf(acc[i][lane][j], is, sum[j]);
    }
    const float inverse = total != 0.0f ? 0x1p24f / total : 0.0f;
    store_two(a, row + 4 * lane, sum[0] * inverse, sum[1] * inverse);
    store_two(a, row + 4 * lane + 2, sum[2] * inverse, sum[3] * inverse);
}

hipError_t launch_join(const AttentionArgs& a, const Split& split, hipStream_t st) {
    const int columns = a.group * a.fresh < COLUMNS ? a.group * a.fresh : COLUMNS;
    const auto kernel = a.c.blocks == 2 ? k_kv_join<2> : a.c.blocks == 4 ? k_kv_join<4> : a.c.blocks == 6 ? k_kv_join<6> : k_kv_join<8>;
    return qs_host::launch_kernel(kernel, dim3((unsigned)split.groups, (unsigned)columns), dim3(256), 0, st, a, split);
}

}  // namespace qskv
