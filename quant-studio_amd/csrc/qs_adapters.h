// Low-rank adapters beside a product with a packed weight (gfx950):
//     y[t] += B[id] (scale * A[id] x[t]),   id = ids[t]
// First v = scale * A x for every row (k_adapter_few; k_adapter_many
// and k_adapter_join), then
// B v: for dot products in the product's own lanes (adapter_sum), for tiles by a
// kernel that writes the sums for the product to add (k_adapter_delta), for
// laid-out factors by matrix instructions on the product's tile (add_adapters).
#pragma once

#include <type_traits>

#include "qs_linear_kernels.h"

namespace qsl {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <int TYPE>
QS_DEV float from16(uint32_t bits) {
    return TYPE == QS_SRC_BF16 ? __uint_as_float(bits << 16) : qsd::half_bits(bits);
}

// A workgroup takes a row and 8 ranks, a wave two of them; a lane 8 values at a
// time. Up to 512 rows, where a row or two use an adapter: bound by the latency
// of ids, offsets and A, one after another (4 us for a row of 2,560 values and
// rank 16, 6 us for 64 rows and ranks to 64).
template <int TYPE>
__global__ __launch_bounds__(256) void k_adapter_few(AdapterArgs a) {
    const int64_t t = blockIdx.x;
    const int id = a.ids[t], lane = threadIdx.x % 64;
    if (id < 0 || id >= a.adapters) return;
    const int o = a.off[id], rank = a.off[id + 1] - o, r0 = blockIdx.y * 8 + threadIdx.x / 64 * 2;
    if (r0 >= rank) return;         // ranks are multiples of 8
    const uint16_t* rows = a.a + (int64_t)(o + r0) * a.k;
    float sum[2] = {};
    for (int64_t c0 = lane * 8; c0 < a.k; c0 += 4 * 512) {
        uint2 x[4];
        float s[4];
        uint4 w[4][2];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int64_t c = c0 + 512 * j < a.k ? c0 + 512 * j : c0;
            x[j] = *reinterpret_cast<const uint2*>(a.q + t * a.k + c);
            s[j] = c0 + 512 * j < a.k ? a.s[t * (a.k / 32) + c / 32] : 0.0f;
#pragma unroll
            for (int r = 0; r < 2; r++) w[j][r] = *reinterpret_cast<const uint4*>(rows + r * a.k + c);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            if (j > 0 && c0 + 512 * j >= a.k) break;
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const uint32_t ww[4] = {w[j][r].x, w[j][r].y, w[j][r].z, w[j][r].w};
                float p = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; i++)
                    p = __builtin_fmaf((float)(int8_t)((i < 4 ? x[j].x : x[j].y) >> (8 * (i & 3))),
                                       from16<TYPE>((ww[i >> 1] >> (16 * (i & 1))) & 0xffffu), p);
                sum[r] = __builtin_fmaf(s[j], p, sum[r]);
            }
        }
    }
#pragma unroll
    for (int r = 0; r < 2; r++) {
        sum[r] = sum16(sum[r]);
        sum[r] += __shfl_xor(sum[r], 16);
        sum[r] += __shfl_xor(sum[r], 32);
    }
    if (lane < 2) a.v[t * a.ldv + r0 + lane] = a.scales[id] * (lane ? sum[1] : sum[0]);
}

// delta[t, n] = sum over r of v[t, r] * B[n, r]; 0 for a row without an adapter.
// A lane takes a column: the wave's rows of B are one run of bytes. Bound by
// reading B for each row: 64 rows, 9,728 columns, ranks 64, 32 and 16, 46 MB: 14 us.
template <int TYPE>
__global__ __launch_bounds__(256) void k_adapter_delta(AdapterArgs a) {
    const int64_t t = blockIdx.y, n = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int id = a.ids[t];
    if (n >= a.n) return;
    float sum = 0.0f;
    if (id >= 0 && id < a.adapters) {
        const int o = a.off[id], rank = a.off[id + 1] - o;
        const uint16_t* b = a.b + a.n * o + n * rank;
        const float* v = a.v + t * a.ldv;
        for (int r0 = 0; r0 < rank; r0 += 32) {
            uint4 w[4];
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (r0 + 8 * j < rank) w[j] = *reinterpret_cast<const uint4*>(b + r0 + 8 * j);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if (r0 + 8 * j >= rank) break;
                const uint32_t ww[4] = {w[j].x, w[j].y, w[j].z, w[j].w};
#pragma unroll
                for (int i = 0; i < 8; i++)
                    sum = __builtin_fmaf(v[r0 + 8 * j + i], from16<TYPE>((ww[i >> 1] >> (16 * (i & 1))) & 0xffffu), sum);
            }
        }
    }
    a.delta[t * a.n + n] = sum;
}

// ---- many rows: matrix instructions ----

template <int TYPE>
QS_DEV f32x16 mfma16(uint4 a, uint4 b, f32x16 c) {
    if constexpr (TYPE == QS_SRC_BF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
// eight codes, exact in both types
template <int TYPE>
QS_DEV uint4 codes16(uint2 c) {
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t w = i < 2 ? c.x : c.y;
        const float lo = (float)(int8_t)(w >> (16 * (i & 1))), hi = (float)(int8_t)(w >> (16 * (i & 1) + 8));
        if constexpr (TYPE == QS_SRC_BF16) o[i] = two(__float_as_uint(lo), __float_as_uint(hi));
        else o[i] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)lo) | ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)hi) << 16);
    }
    return uint4{o[0], o[1], o[2], o[3]};
}
// v to 16 bits, and what that leaves of it (exactly). Two pieces hold 16 (BF16) or
// 22 (F16) bits of v, three all 24. An infinity leaves nothing, and a finite
// v that bf16 would round to one is cut, so that the pieces' sum stays v.
template <int TYPE>
QS_DEV float piece16(float v, uint16_t& piece) {
    using T = std::conditional_t<TYPE == QS_SRC_BF16, __bf16, _Float16>;
    T h = (T)v;
    if constexpr (TYPE == QS_SRC_BF16)
        if (fabsf(v) < __builtin_inff() && !(fabsf((float)h) < __builtin_inff()))
            h = __builtin_bit_cast(__bf16, (uint16_t)(__float_as_uint(v) >> 16));
    piece = __builtin_bit_cast(uint16_t, h);
    return fabsf((float)h) < __builtin_inff() ? v - (float)h : 0.0f;
}

// A workgroup takes 32 rows and 32 ranks. Eight groups of 32 values at a time
// lie in LDS, copied there in whole runs of each row (an operand read from
// memory is 32 runs of 16 bytes), those of the next two turns in flight; a wave
// takes one of the groups. The codes are exact in the adapters' type: only the
// products' sums are scaled, in f32. The rows' adapters are taken one after
// another (packed sequences have one or two to 32 rows). A row's values are
// split over `parts` workgroups, whose sums k_adapter_join adds. 2,047 rows of
// 9,728 values, ranks 128, 64 and 32: 30 to 36 us, bound by the latency of a turn's
// copies, LDS and barrier (vector instructions, which widen the codes and scale the
// products, take 0.22 of the cycles, matrix ones 0.03); the join takes 4 to 5 us.
template <int TYPE>
__global__ __launch_bounds__(512) void k_adapter_many(AdapterArgs a) {
    constexpr int XS = 256 + 16, AS = 512 + 16;     // strides that spread rows over the banks
    __shared__ __attribute__((aligned(16))) uint8_t xl[2][32 * XS], al[2][32 * AS];
    __shared__ float sl[2][8][32];
    static_assert(sizeof(al) >= 8 * 32 * 33 * 4, "the waves' sums, over A's place");
    float(*join)[32][33] = reinterpret_cast<float(*)[32][33]>(al);
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64, col = lane % 32, half = lane / 32;
    const int64_t t0 = (int64_t)blockIdx.x * 32, t = t0 + col < a.t ? t0 + col : a.t - 1;
    const int r0 = blockIdx.y * 32, groups = (int)(a.k / 32), turns = (groups + 7) / 8;
    const int per = (turns + a.parts - 1) / a.parts, begin = blockIdx.z * per, end = begin + per < turns ? begin + per : turns;
    const int raw = a.ids[t], id = t0 + col < a.t && raw >= 0 && raw < a.adapters ? raw : -1;
    uint32_t left = (uint32_t)__ballot(id >= 0);
    // this thread's copies of a turn: 16 bytes of codes, 32 of A, a scale
    const int64_t xt = t0 + tid / 16 < a.t ? t0 + tid / 16 : a.t - 1, st = t0 + tid / 8 < a.t ? t0 + tid / 8 : a.t - 1;
    const int8_t* xrow = a.q + xt * a.k;
    const float* srow = a.s + st * groups;      // of the first 256 threads
    while (left) {
        const int now = __builtin_amdgcn_readlane(id, __builtin_ctz(left));
        const uint32_t mine = (uint32_t)__ballot(id == now);
        left &= ~mine;
        const int o = a.off[now], rank = a.off[now + 1] - o;
        if (r0 >= rank) continue;
        const uint16_t* arow = a.a + (int64_t)(o + (r0 + tid / 16 < rank ? r0 + tid / 16 : rank - 1)) * a.k;
        struct Ahead {
            i32x4 x, a0, a1;
            float s;
        } ahead0, ahead1;
        auto load = [&](Ahead& r, int turn) __attribute__((always_inline)) {
            const int64_t c = (int64_t)turn * 256 + tid % 16 * 16, last = a.k - 16;
            const int g = turn * 8 + tid % 8;
            r.x = *reinterpret_cast<const i32x4*>(xrow + (c < last ? c : last));
            r.a0 = *reinterpret_cast<const i32x4*>(arow + (c < last ? c : last));
            r.a1 = *reinterpret_cast<const i32x4*>(arow + (c < last ? c : last) + 8);
            r.s = srow[g < groups ? g : groups - 1];
        };
        f32x16 acc = {};
        auto turn_of = [&](int b, Ahead& r, int turn) __attribute__((always_inline)) {
            *reinterpret_cast<i32x4*>(xl[b] + tid / 16 * XS + tid % 16 * 16) = r.x;
            *reinterpret_cast<i32x4*>(al[b] + tid / 16 * AS + tid % 16 * 32) = r.a0;
            *reinterpret_cast<i32x4*>(al[b] + tid / 16 * AS + tid % 16 * 32 + 16) = r.a1;
            if (tid < 256) sl[b][tid % 8][tid / 8] = r.s;
            load(r, turn + 2);
            lds_barrier();
            f32x16 p = {};
#pragma unroll
            for (int h = 0; h < 2; h++)
                p = mfma16<TYPE>(*reinterpret_cast<const uint4*>(al[b] + col * AS + 64 * wave + 32 * h + 16 * half),
                                 codes16<TYPE>(*reinterpret_cast<const uint2*>(xl[b] + col * XS + 32 * wave + 16 * h + 8 * half)), p);
            const float s = sl[b][wave][col];
            const bool live = turn < end && turn * 8 + wave < groups;   // past the end lie other values
#pragma unroll
            for (int i = 0; i < 16; i++) acc[i] = live ? __builtin_fmaf(p[i], s, acc[i]) : acc[i];
        };
        load(ahead0, begin);
        load(ahead1, begin + 1);
        lds_barrier();      // the places are free
        for (int turn = begin; turn < end; turn += 2) {     // turns past the end count nothing
            turn_of(0, ahead0, turn);
            turn_of(1, ahead1, turn + 1);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 16; i++) join[wave][col][8 * (i / 4) + 4 * half + i % 4] = acc[i];
        __syncthreads();
        // 16 lanes to a row, two ranks each
        const int row32 = tid / 16, r = tid % 16 * 2;
        float v[2] = {};
#pragma unroll
        for (int w = 0; w < 8; w++) v[0] += join[w][row32][r], v[1] += join[w][row32][r + 1];
        if ((mine >> row32) & 1) {
            float* sum = a.sums + (blockIdx.z * a.t + t0 + row32) * a.ldv + r0 + r;
            if (r0 + r < rank) sum[0] = v[0];
            if (r0 + r + 1 < rank) sum[1] = v[1];
        }
        __syncthreads();
    }
}

// The parts' sums, scaled, as hi + lo (+ rest): 16 lanes to a row's 32 ranks, two each.
template <int TYPE>
__global__ __launch_bounds__(256) void k_adapter_join(AdapterArgs a) {
    const int64_t t = (int64_t)blockIdx.x * 16 + threadIdx.x / 16;
    const int r0 = blockIdx.y * 32, r = r0 + threadIdx.x % 16 * 2;
    const int id = t < a.t ? a.ids[t] : -1;
    const bool has = id >= 0 && id < a.adapters;
    const int rank = has ? a.off[id + 1] - a.off[id] : 0;
    const bool live = r < rank;     // ranks are multiples of 8
    float v[2] = {};
    for (int z = 0; z < a.parts; z++)
#pragma unroll
        for (int i = 0; i < 2; i++) v[i] += live ? a.sums[(z * a.t + t) * a.ldv + r + i] : 0.0f;
    const float scale = has ? a.scales[id] : 0.0f;
    v[0] = live ? v[0] * scale : 0.0f, v[1] = live ? v[1] * scale : 0.0f;
    float unit = 1.0f;
    if constexpr (TYPE == QS_SRC_F16) {
        // a power of two that takes the largest finite one of the 32 to f16's upper range
        const auto finite = [](float f) { return fabsf(f) < __builtin_inff() ? fabsf(f) : 0.0f; };
        float top = fmaxf(finite(v[0]), finite(v[1]));
        top = fmaxf(top, __shfl_xor(top, 1)), top = fmaxf(top, __shfl_xor(top, 2));
        top = fmaxf(top, __shfl_xor(top, 4)), top = fmaxf(top, __shfl_xor(top, 8));
        int e = 0;
        if (top > 0.0f) (void)__builtin_frexpf(top, &e);
        e = e < -80 ? -80 : e;
        unit = __builtin_ldexpf(1.0f, e - 15);
        v[0] = __builtin_ldexpf(v[0], 15 - e), v[1] = __builtin_ldexpf(v[1], 15 - e);
    }
    if (!live) return;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int64_t at = t * a.ldv + r + i;
        const float left = piece16<TYPE>(piece16<TYPE>(v[i], a.hi[at]), a.lo[at]);
        if (a.rest) piece16<TYPE>(left, a.rest[at]);
    }
    if (TYPE == QS_SRC_F16 && r == r0) a.unit[t * ((a.ldv + 31) / 32) + r0 / 32] = unit;
}

// What add_adapters reads.
struct AdapterTile {
    const int32_t *ids, *off;
    const uint16_t *b, *hi, *lo, *rest;
    const float* unit;
    int64_t ldv;
    int32_t adapters;
};

// y += B v on UM x UN units of 32 x 32 (rows t0 .., columns n0 ..) that a wave
// holds. The rows' adapters are taken one after another, 32 ranks a step; a
// unit's products are kept apart and added to the rows that have the adapter,
// so that a NaN in another's B does not reach them. Of WK waves that share the
// sums of these units each takes every WK-th step: a step is bound by the
// latency of what it reads (512 rows with q4_k 2,560 x 2,560, 4 adapters: the
// product took 44 us with the steps in one wave of eight). PIECES of v: with exact
// codes three, which hold it whole, two with factors of f16, whose result is bf16.
template <int TYPE, int PIECES, int WK, int UM, int UN>
QS_DEV void add_adapters(const AdapterTile& a, f32x16 (&y)[UM][UN], int64_t t0, int64_t rows, int64_t n0, int64_t n, int wk) {
    const int lane = threadIdx.x % 64, col = lane % 32, half = lane / 32;
    const int64_t units = (a.ldv + 31) / 32;
    int step = 0;
#pragma unroll
    for (int um = 0; um < UM; um++) {
        const int64_t tb = t0 + 32 * um, t = tb + col < rows ? tb + col : rows - 1;
        const int raw = a.ids[t], id = tb + col < rows && raw >= 0 && raw < a.adapters ? raw : -1;
        uint32_t left = (uint32_t)__ballot(id >= 0);
        while (left) {
            const int now = __builtin_amdgcn_readlane(id, __builtin_ctz(left));
            const uint32_t mine = (uint32_t)__ballot(id == now), elements = mine >> (4 * half);
            left &= ~mine;
            const int o = a.off[now], rank = a.off[now + 1] - o;
            const uint16_t* const from[3] = {a.hi + t * a.ldv, a.lo + t * a.ldv, PIECES > 2 ? a.rest + t * a.ldv : nullptr};
            for (int r0 = 0; r0 < rank; r0 += 32) {
                if (step++ % WK != wk) continue;
                uint4 v[PIECES][2];
#pragma unroll
                for (int s = 0; s < 2; s++) {
                    const int r = r0 + 16 * s + 8 * half;
                    const bool live = id == now && r < rank;
#pragma unroll
                    for (int j = 0; j < PIECES; j++)
                        v[j][s] = live ? *reinterpret_cast<const uint4*>(from[j] + r) : uint4{0, 0, 0, 0};
                }
                float unit[16];
                if constexpr (TYPE == QS_SRC_F16)
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const int64_t ti = tb + 8 * (i / 4) + 4 * half + i % 4;
                        unit[i] = a.unit[(ti < rows ? ti : rows - 1) * units + r0 / 32];
                    }
#pragma unroll
                for (int un = 0; un < UN; un++) {
                    const int64_t c = n0 + 32 * un + col;
                    const uint16_t* b = a.b + n * o + (c < n ? c : n - 1) * rank;
                    __builtin_amdgcn_sched_barrier(0);      // one unit's operands at a time: y fills the registers
                    f32x16 p = {};
#pragma unroll
                    for (int s = 0; s < 2; s++) {
                        const int r = r0 + 16 * s + 8 * half;
                        const uint4 w = r < rank ? *reinterpret_cast<const uint4*>(b + r) : uint4{0, 0, 0, 0};
#pragma unroll
                        for (int j = PIECES - 1; j >= 0; j--) p = mfma16<TYPE>(v[j][s], w, p);
                    }
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const float d = TYPE == QS_SRC_F16 ? p[i] * unit[i] : p[i];
                        y[um][un][i] = (elements >> (8 * (i / 4) + i % 4)) & 1 ? y[um][un][i] + d : y[um][un][i];
                    }
                }
            }
        }
    }
}
}  // namespace qsl
