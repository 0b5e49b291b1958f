// Joins what workgroups of the attention left of sequences that were split.
#include "qs_kv_attention.h"
#include "qs_launch_kernel.h"

namespace qskv {

typedef float f32x4 __attribute__((ext_vector_type(4)));

QS_DEV float power(float part, float top, float total) {    // total: of a part that saw nothing 0, or NaN
    return part > -__builtin_inff() ? __builtin_amdgcn_exp2f(part - top) : total;
}

// Grid (segments, columns). D / 4 threads take a part's row, the others the next parts,
// four of them at a time, and LDS joins what they have in a fixed order. Latency is
// all there is to it, 3.7 to 5.5 us of a call. Of more than 128 parts of a segment 1,024
// threads have nearly all on their way at once: one sequence of 100,000 slots takes 21.4 us
// with one head (384 parts or more; 25.8 with 256 threads) and 31.4 with four (192; 31.3),
// but 16.0 and 14.8 of 8,000 slots with eight heads (63), 26.1 and 25.3 of 40,000 (96).
template <int BLOCKS, int THREADS>
__global__ __launch_bounds__(THREADS) void k_kv_join(AttentionArgs a, Split split) {
    constexpr int D = 32 * BLOCKS, LANES = D / 4, ROWS = THREADS / LANES, TIMES = 4;
    __shared__ f32x4 acc[ROWS][LANES];
    __shared__ float2 stats[ROWS];
    const int tiles = column_tiles(a), columns = columns_of(a), column = (int)blockIdx.y;
    int4 s;
    if (split.share) {
        const int heads = a.c.heads * tiles, seq = (int)blockIdx.x / heads, first = (int)blockIdx.x * split.share;
        s = int4{seq, (int)blockIdx.x - seq * heads, first, first + split.share - 1};
    } else {
        // all of them within bounds, unless lengths changed meanwhile
        s = split.segments[blockIdx.x];
        if ((unsigned)s.x >= (unsigned)a.batch || (unsigned)s.y >= (unsigned)(a.c.heads * tiles) || s.z < 0 || s.w < s.z || s.w >= split.groups) return;
    }
    const int head = s.y / tiles;
    const int64_t row = row_of(a, s.x, head, (s.y - head * tiles) * columns + column);
    if (row < 0) return;
    const int mine = (int)threadIdx.x / LANES, lane = (int)threadIdx.x - mine * LANES;
    const int count = s.w - s.z + 1;
    f32x4 sum{0, 0, 0, 0};
    float ref = -__builtin_inff(), total = 0.0f;
    if (mine < ROWS) {
        for (int i = mine; i < count; i += TIMES * ROWS) {
            float2 part[TIMES];
            f32x4 v[TIMES];
#pragma unroll
            for (int j = 0; j < TIMES; j++) {
                const int n = i + j * ROWS;
                part[j] = float2{-__builtin_inff(), 0.0f};
                v[j] = f32x4{0, 0, 0, 0};
                if (n < count) {
                    const int64_t slot = ((int64_t)(s.z + n) * 2 + (n == 0)) * columns + column;
                    part[j] = split.stats[slot];
                    v[j] = *reinterpret_cast<const f32x4*>(split.parts + slot * D + 4 * lane);
                }
            }
            float top = ref;
#pragma unroll
            for (int j = 0; j < TIMES; j++) top = fmaxf(top, part[j].x);
            const float was = power(ref, top, 0.0f);
            total *= was;
#pragma unroll
            for (int e = 0; e < 4; e++) sum[e] *= was;
#pragma unroll
            for (int j = 0; j < TIMES; j++) {
                const float is = power(part[j].x, top, part[j].y);
                total = __builtin_fmaf(part[j].y, is, total);
#pragma unroll
                for (int e = 0; e < 4; e++) sum[e] = __builtin_fmaf(v[j][e], is, sum[e]);
            }
            ref = top;
        }
        acc[mine][lane] = sum;
        if (lane == 0) stats[mine] = float2{ref, total};
    }
    __syncthreads();
    if ((int)threadIdx.x >= LANES) return;
    const int rows = count < ROWS ? count : ROWS;
    ref = -__builtin_inff();
    for (int i = 0; i < rows; i++) ref = fmaxf(ref, stats[i].x);
    sum = f32x4{0, 0, 0, 0};
    total = 0.0f;
#pragma unroll 4
    for (int i = 0; i < rows; i++) {
        const float2 part = stats[i];
        const float is = power(part.x, ref, part.y);
        total = __builtin_fmaf(part.y, is, total);
#pragma unroll
        for (int e = 0; e < 4; e++) sum[e] = __builtin_fmaf(acc[i][threadIdx.x][e], is, sum[e]);
    }
    const float inverse = inverse_of(ref, total);
    store_two(a, row + 4 * threadIdx.x, sum[0] * inverse, sum[1] * inverse);
    store_two(a, row + 4 * threadIdx.x + 2, sum[2] * inverse, sum[3] * inverse);
}

template <int BLOCKS>
hipError_t launch_blocks(const AttentionArgs& a, const Split& split, hipStream_t st) {
    const int columns = a.group * a.fresh < columns_of(a) ? a.group * a.fresh : columns_of(a);
    const int segments = split.share ? split.groups / split.share : split.listed ? split.listed : split.groups;
    const bool many = split.groups > 128 * segments;       // parts of a segment
    return qs_host::launch_kernel(many ? k_kv_join<BLOCKS, 1024> : k_kv_join<BLOCKS, 256>, dim3((unsigned)segments, (unsigned)columns),
                                  dim3(many ? 1024 : 256), 0, st, a, split);
}

hipError_t launch_join(const AttentionArgs& a, const Split& split, hipStream_t st) {
    switch (a.c.blocks) {
        case 2: return launch_blocks<2>(a, split, st);
        case 4: return launch_blocks<4>(a, split, st);
        case 6: return launch_blocks<6>(a, split, st);
        default: return launch_blocks<8>(a, split, st);
    }
}

}  // namespace qskv
