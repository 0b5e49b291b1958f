// Products of many 8-bit rows with a packed weight whose result is bf16
// (gfx950): both factors laid out in f16 for the matrix units, once per call.
//
// Matrix and vector instructions of a SIMD do not overlap (an 8-bit 32x32x32
// product and the 32 vector instructions that scale its result take the sum of
// their times, 37 and 80 clocks), so products that are scaled group by group
// cost three times those that are not. Here d * c - m and s * q are rounded to
// f16, 2^-11 of each value, an eighth of what rounding the result to bf16 does
// to it: together with that rounding the error of a sum of them is 1.5% larger
// than the rounding's alone, and far larger where its terms cancel. Each row is
// first multiplied by a power of two that takes its largest possible value near
// 2^15, so nothing overflows and what is lost below f16's range is under 2^-39 of
// that value.
#pragma once

#include "qs_matrix.h"

namespace qsl {

// The largest |d c| and |m| of a block by its f16 scales: a bound of its values.
template <int TYPE, typename P>
QS_DEV float block_bound(P b) {
    const auto h = [&](int at) { return fabsf(qsd::half_bits(qsd::load_u16(b + at))); };
    if constexpr (TYPE == QS_TYPE_Q4_0) return 8 * h(0);
    else if constexpr (TYPE == QS_TYPE_Q4_1) return 15 * h(0) + h(2);
    else if constexpr (TYPE == QS_TYPE_Q5_0) return 16 * h(0);
    else if constexpr (TYPE == QS_TYPE_Q5_1) return 31 * h(0) + h(2);
    else if constexpr (TYPE == QS_TYPE_Q8_0) return 128 * h(0);
    else if constexpr (TYPE == QS_TYPE_IQ4_NL) return 127 * h(0);
    else if constexpr (TYPE == QS_TYPE_Q2_K) return 45 * h(80) + 15 * h(82);
    else if constexpr (TYPE == QS_TYPE_Q3_K) return 128 * h(108);
    else if constexpr (TYPE == QS_TYPE_Q4_K) return 63 * 15 * h(0) + 63 * h(2);
    else if constexpr (TYPE == QS_TYPE_Q5_K) return 63 * 31 * h(0) + 63 * h(2);
    else if constexpr (TYPE == QS_TYPE_Q6_K) return 4096 * h(208);
    else if constexpr (TYPE == QS_TYPE_IQ4_XS) return 32 * 127 * h(0);
    else if constexpr (TYPE == QS_TYPE_IQ3_XXS) return 481 * h(0);      // 0.5 * 15.5 * 62
    else if constexpr (TYPE == QS_TYPE_IQ3_S) return 465 * h(0);        // 31 * 15
    else return 167 * h(0);                                             // IQ2: 0.25 * 15.5 * 43
}

// 2^-e for the largest possible |value| of a row, bound * 2^bits (which may pass f32's
// largest number), that takes it to 2^14 .. 2^15
QS_DEV float row_scale(float bound, int bits) {
    if (!(bound > 0.0f && bound < __builtin_inff())) return 1.0f;
    int e;
    (void)__builtin_frexpf(bound, &e);          // 2^(e-1) <= bound < 2^e
    e += bits;
    e = e < -110 ? -110 : e;
    return __builtin_ldexpf(1.0f, 15 - e);
}

QS_DEV float inverse_of_power(float f) { return __uint_as_float((254u << 23) - __float_as_uint(f)); }

struct ScaleArgs {
    const uint8_t* w;
    const float* s;
    float *ws, *xs;             // of the weight's and the rows' rows
    int64_t row_bytes, n, t, k;
    int64_t w_blocks;           // workgroups that take the weight's rows; the rest take x's
};

// Eight lanes to a row, which read the f16 scales of its blocks: 5 us for 9,728
// rows of q4_k, the latency of a few such reads.
template <int TYPE>
__global__ __launch_bounds__(256) void k_row_scales(ScaleArgs a) {
    const bool weight = (int64_t)blockIdx.x < a.w_blocks;
    const int64_t row = (weight ? blockIdx.x : blockIdx.x - a.w_blocks) * (int64_t)32 + threadIdx.x / 8;
    const int lane = threadIdx.x % 8;
    float top = 0.0f;
    const auto take = [&](float v) { top = v > top || v != v ? v : top; };      // keeps a NaN
    if (weight) {
        const int blocks = (int)(a.k / Format<TYPE>::BLK);
        if (row < a.n)
#pragma unroll 4
            for (int b = lane; b < blocks; b += 8) take(block_bound<TYPE>(a.w + row * a.row_bytes + (int64_t)b * Format<TYPE>::BYTES));
    } else {
        const int groups = (int)(a.k / 32);
        if (row < a.t)
#pragma unroll 4
            for (int g = lane; g < groups; g += 8) take(fabsf(a.s[row * groups + g]));
    }
#pragma unroll
    for (int o = 1; o < 8; o *= 2) take(__shfl_xor(top, o));
    if (lane == 0 && row < (weight ? a.n : a.t)) (weight ? a.ws : a.xs)[row] = row_scale(top, weight ? 0 : 7);
}

struct Layout16Args {
    const uint8_t* w;
    const int8_t* q;
    const float *s, *ws, *xs;
    uint8_t *wl, *xl;
    int64_t row_bytes, n, t, k;
    int64_t w_blocks;
    int groups;             // of a row, rounded up to the stages'
};

// Layout: panels of 32 rows; in a panel, for each 16 values, [2][32 rows][8]:
// an operand of the 32x32x16 instructions is 1,024 bytes in a row. A workgroup
// lays out 32 rows by 8 groups, a group to a thread. Bound by memory: 4,096 rows
// and q4_k 9,728 x 2,560, 96 MB read and written, 19 to 22 us, a copy's rate.
template <int TYPE>
__global__ __launch_bounds__(256) void k_lay_out16(Layout16Args a) {
    __shared__ uint16_t grid[Format<TYPE>::GRID ? Format<TYPE>::GRID : 1];
    const bool weight = (int64_t)blockIdx.x < a.w_blocks;
    if (weight) {
        qsd::stage_grid<TYPE>(grid, threadIdx.x, 256);
        if (Format<TYPE>::GRID) __syncthreads();
    }
    const int per = (a.groups + 7) / 8, row = threadIdx.x % 32, live_groups = (int)(a.k / 32);
    const int64_t b = weight ? blockIdx.x : blockIdx.x - a.w_blocks, panel = b / per;
    const int g = (int)(b % per) * 8 + threadIdx.x / 32;
    if (g >= a.groups) return;
    const bool live = g < live_groups;
    uint32_t c[8];
    float d[2], m[2];           // of the two halves: value = d * c - m
    if (weight) {
        const int64_t n = panel * 32 + row, at = n < a.n ? n : a.n - 1;
        Raw<TYPE> raw;
        Group<TYPE> w;
        qsd::load_row_group<TYPE>(a.w + at * a.row_bytes, live ? g : live_groups - 1, raw);
        qsd::decode_group<TYPE>(raw, qsd::group_in_block<TYPE>(live ? g : live_groups - 1), grid, w);
        const float f = live ? a.ws[at] : 0.0f;
#pragma unroll
        for (int h = 0; h < 2; h++) d[h] = w.d[h * (Format<TYPE>::SUB - 1)] * f, m[h] = w.m[h * (Format<TYPE>::SUB - 1)] * f;
#pragma unroll
        for (int i = 0; i < 8; i++) c[i] = w.c[i];
    } else {
        const int64_t t = panel * 32 + row, at = t < a.t ? t : a.t - 1;
        const uint4* x = reinterpret_cast<const uint4*>(a.q + at * a.k + 32 * (live ? g : live_groups - 1));
        const uint4 lo = x[0], hi = x[1];
        c[0] = lo.x, c[1] = lo.y, c[2] = lo.z, c[3] = lo.w, c[4] = hi.x, c[5] = hi.y, c[6] = hi.z, c[7] = hi.w;
        d[0] = d[1] = live ? qsd::scale_of(a.s[at * live_groups + g]) * a.xs[at] : 0.0f;
        m[0] = m[1] = 0.0f;
    }
    uint4* p = reinterpret_cast<uint4*>((weight ? a.wl : a.xl) + (panel * a.groups + g) * 2048) + row;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        f16x8 v;
#pragma unroll
        for (int j = 0; j < 8; j++)
            v[j] = (_Float16)__builtin_fmaf(d[i / 2], (float)(int8_t)(c[2 * i + j / 4] >> (8 * (j % 4))), -m[i / 2]);
        p[32 * i] = __builtin_bit_cast(uint4, v);
    }
}

// A tile of BM rows by BN weight rows. Two stages of S x 16 values lie in LDS;
// while one is multiplied the next one's copies are in flight. WM x WN waves
// split the tile, WK the steps of a stage (their sums are joined in LDS at the
// end, in order): a wave's part of the tile stays large where the tile is not.
// Where tiles are few the stages are split over workgroups too. 4,096 rows with
// q4_k 9,728 x 2,560 in tiles of 256 x 320: 197 us, 1.0 PFLOP/s, what a library's
// product of the same size in bf16 takes; bound there by the power that matrix
// instructions draw (the clock falls from 2.4 GHz to 1.9 to 2.0), in smaller
// products by the latency of a stage's copies, of which one is in flight.
// The stages are two arrays, so that the compiler sees that a read of one does
// not wait for copies to the other.
template <int BM, int BN, int WM, int WN, int WK, int S, int ADAPT>
__global__ __launch_bounds__(64 * WM * WN * WK, 2) void k_matrix16(Matrix16Args a) {
    constexpr int WAVES = WM * WN * WK, UM = BM / WM / 32, UN = BN / WN / 32, STEPS = S / WK;
    constexpr int XS = BM / 32 * S * 1024, STAGE = XS + BN / 32 * S * 1024, COPIES = STAGE / 1024 / WAVES;
    static_assert(STAGE / 1024 % WAVES == 0 && S % WK == 0, "copies");
    __shared__ __attribute__((aligned(1024))) uint8_t even[STAGE], odd[STAGE];
    const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int wn = wave % WN, wm = wave / WN % WM, wk = wave / WN / WM, col = lane % 32, half = lane / 32;
    const LinearArgs& l = a.l;
    // XCDs and strips as in k_matrix
    const int64_t tiles_m = (l.t + BM - 1) / BM, tiles_n = (a.count + BN - 1) / BN, tiles = tiles_m * tiles_n;
    const int64_t place = (int64_t)(blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8, at = place % tiles;
    if (place >= tiles * l.splits) return;
    const int64_t strip = at / (8 * tiles_m), left = tiles_n - 8 * strip, wide = left < 8 ? left : 8;
    const int64_t in = at - strip * 8 * tiles_m;
    const int64_t t0 = in / wide * BM, n0 = (8 * strip + in % wide) * BN;
    // an even number of stages, and this part's of them (no part is empty)
    const int all = a.groups * 2 / S, per = (all / 2 + l.splits - 1) / l.splits * 2, split = (int)(place / tiles);
    const int begin = split * per, end = begin + per < all ? begin + per : all;

    // This wave's copies of a stage: 1,024 bytes each, panel after panel; panels
    // past the last (a tile may reach past the layout) are the last one again.
    const int64_t panel_bytes = (int64_t)a.groups * 2048;
    const int last_x = (int)((l.t - 1) / 32 - t0 / 32), last_w = (int)((a.count - 1) / 32 - n0 / 32);
    const uint8_t* from[COPIES];
#pragma unroll
    for (int i = 0; i < COPIES; i++) {
        const int c = wave * COPIES + i, panel = c / S, p = panel < BM / 32 ? panel : panel - BM / 32;
        from[i] = (panel < BM / 32 ? a.xl + (t0 / 32 + (p < last_x ? p : last_x)) * panel_bytes
                                   : a.wl + (n0 / 32 + (p < last_w ? p : last_w)) * panel_bytes) + c % S * 1024;
    }
    const uint32_t lane16 = (uint32_t)lane * 16;
    auto copy = [&](int stage, uint8_t* to) {
        const int64_t off = (int64_t)stage * (S * 1024);
#pragma unroll
        for (int i = 0; i < COPIES; i++) copy_to_lds(from[i] + off + lane16, to + (wave * COPIES + i) * 1024);
    };
    f32x16 acc[UM][UN] = {};
    f16x8 xa[2][UM], wb[2][UN];
    // places as one sum: the compiler follows which array a read is of through
    // few steps of address arithmetic only
    const int x0 = (wm * UM * S + wk * STEPS) * 1024 + lane * 16, w0 = XS + (wn * UN * S + wk * STEPS) * 1024 + lane * 16;
    auto read = [&](const uint8_t* stage, int step, int to) {
#pragma unroll
        for (int u = 0; u < UM; u++) xa[to][u] = *reinterpret_cast<const f16x8*>(stage + (x0 + (u * S + step) * 1024));
#pragma unroll
        for (int u = 0; u < UN; u++) wb[to][u] = *reinterpret_cast<const f16x8*>(stage + (w0 + (u * S + step) * 1024));
    };
    auto multiply = [&](int from) {
#pragma unroll
        for (int um = 0; um < UM; um++)
#pragma unroll
            for (int un = 0; un < UN; un++)
                acc[um][un] = __builtin_amdgcn_mfma_f32_32x32x16_f16(xa[from][um], wb[from][un], acc[um][un], 0, 0, 0);
    };
    // A stage's steps, from the operands of its first one (in buffer `b`). The
    // last step's are in registers when the stages change: after the barrier
    // every wave has them and every wave's copies of the next stage have landed,
    // so the copies after next go to this stage's place, and the next stage's
    // operands are read under the last step's products.
    auto turn = [&](uint8_t* stage, const uint8_t* next, int after, int b) {
#pragma unroll
        for (int s = 0; s < STEPS - 1; s++) {
            read(stage, s + 1, (b + s + 1) % 2);
            __builtin_amdgcn_sched_barrier(0);      // under the products of this step
            multiply((b + s) % 2);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_waitcnt(0x0070);         // vmcnt(0), lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        copy(after < end ? after : end - 1, stage);     // no branch: the last stage again
        __builtin_amdgcn_sched_barrier(0);                  // they go out first
        read(next, 0, (b + STEPS) % 2);
        __builtin_amdgcn_sched_barrier(0);
        multiply((b + STEPS - 1) % 2);
        __builtin_amdgcn_sched_barrier(0);
    };
    copy(begin, even);
    copy(begin + 1, odd);
    __builtin_amdgcn_s_waitcnt(0x0f70);             // vmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(even, 0, 0);
    for (int s = begin; s < end; s += 2) {
        turn(even, odd, s + 2, 0);
        turn(odd, even, s + 3, STEPS % 2);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);     // no copy to LDS outlives the workgroup
    float unw[UN];
#pragma unroll
    for (int un = 0; un < UN; un++) {
        const int64_t n = n0 + (wn * UN + un) * 32 + col;
        unw[un] = inverse_of_power(a.ws[n < a.count ? n : a.count - 1]);
    }
#pragma unroll
    for (int um = 0; um < UM; um++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int64_t t = t0 + (wm * UM + um) * 32 + 8 * (i / 4) + 4 * half + i % 4;
            const float unx = inverse_of_power(a.xs[t < l.t ? t : l.t - 1]);
#pragma unroll
            for (int un = 0; un < UN; un++) acc[um][un][i] = acc[um][un][i] * unw[un] * unx;
        }
    if constexpr (ADAPT)
        if (split == 0) add_adapters<ADAPT, 2, WK>(adapter_tile(l), acc, t0 + wm * UM * 32, l.t, a.first + n0 + wn * UN * 32, l.n, wk);
    if constexpr (WK > 1) {
        static_assert(STAGE >= BM * BN * 4 / UN, "a column of units");
        join_waves<WK, WM * WN>(acc, reinterpret_cast<float*>(even), wk, wm * WN + wn);
        if (wk > 0) return;
    }
    store_tile(l.splits > 1 ? l.parts + split * l.t * l.n : l.dst, l.splits > 1 ? QS_SRC_F32 : l.dst_type, l, acc,
               t0 + wm * UM * 32, a.first + n0 + wn * UN * 32, a.first + a.count);
}

}  // namespace qsl
