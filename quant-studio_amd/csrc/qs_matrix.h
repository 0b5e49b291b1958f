// Products of many 8-bit rows with a packed weight (gfx950). Both factors are
// first laid out as the matrix instructions read them, once per call, so that
// the product itself decodes nothing: every weight would otherwise be decoded
// again for each tile of rows.
#pragma once

#include <type_traits>

#include "qs_adapters.h"
#include "qs_linear_kernels.h"

namespace qsl {

typedef short s16x4 __attribute__((ext_vector_type(4)));

// A format as the matrix units take it: groups of 32 integers with ONE scale.
// Where a format scales 16 values at a time its integer scale is multiplied
// into the codes (block scale d, code c * sc): within 8 bits for Q2_K and Q3_K,
// else in two planes, c * sc = 128 hi + lo.
//   PLANES: byte planes of the codes; MINS: minima of a group (1, or 2 of 16).
template <int TYPE>
struct MatrixFormat {
    static constexpr int SUB = Format<TYPE>::SUB;
    static constexpr int PLANES = two_planes(TYPE) ? 2 : 1, MINS = minima(TYPE);
    static_assert(MINS == (Format<TYPE>::MIN ? SUB : 0), "minima");
};

// Layout of a laid-out factor: panels of 32 rows; in a panel, for each group,
//   PLANES x [2 halves][32 rows][16 codes]
//   (1 + MINS) x [32 rows][8 bytes: the three bf16 pieces of a scale]
// (panel_group_bytes)

QS_DEV uint2 piece_words(float f) {
    const Pieces p = pieces(f);
    return uint2{two(p.a, p.b), p.c >> 16};
}

// the integer scales of a group's two halves, and what their product with the
// codes is still to be multiplied by
template <int TYPE>
QS_DEV void integer_scales(const Raw<TYPE>& r, int g, int (&sc)[2], float& d) {
    if constexpr (TYPE == QS_TYPE_Q2_K) {
        sc[0] = (int)(r.w[9] & 15u), sc[1] = (int)((r.w[9] >> 8) & 15u);
        d = qsd::half_bits(r.w[8] & 0xffffu);
    } else if constexpr (TYPE == QS_TYPE_Q3_K) {
#pragma unroll
        for (int j = 0; j < 2; j++) sc[j] = -qsd::q3_scale(r, 2 * g + j);   // -4 * -32 is over 127, -(-4 * -32) fits
        d = -qsd::half_bits(r.w[19]);
    } else if constexpr (TYPE == QS_TYPE_Q6_K) {
        sc[0] = (int8_t)(r.w[16] & 0xffu), sc[1] = (int8_t)((r.w[16] >> 8) & 0xffu);
        d = qsd::half_bits(r.w[17]);
    } else {
        const uint32_t s = r.w[TYPE == QS_TYPE_IQ2_XS ? 3 : 4];
        sc[0] = (int)(2u * (s & 15u) + 1u), sc[1] = (int)(2u * ((s >> 4) & 15u) + 1u);
        d = qsd::half_bits(r.w[2]) * 0.125f;
    }
}

// Lays out one group of one weight row at p (its panel's group).
template <int TYPE>
QS_DEV void lay_out_weight(const Raw<TYPE>& raw, int g, const uint16_t* grid, bool live, uint8_t* p, int row) {
    using M = MatrixFormat<TYPE>;
    Group<TYPE> w;
    qsd::decode_group<TYPE>(raw, g, grid, w);
    float d = w.d[0];
    uint32_t c[M::PLANES][8];
    if constexpr (M::SUB == 1) {
#pragma unroll
        for (int i = 0; i < 8; i++) c[0][i] = w.c[i];
    } else {
        int sc[2];
        integer_scales<TYPE>(raw, g, sc, d);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            uint32_t lo = 0, hi = 0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int v = (int)(int8_t)(w.c[i] >> (8 * j)) * sc[i / 4];
                if constexpr (M::PLANES == 1) lo |= (uint32_t)(v & 255) << (8 * j);
                else lo |= (uint32_t)(v & 127) << (8 * j), hi |= (uint32_t)((v >> 7) & 255) << (8 * j);
            }
            c[0][i] = lo;
            if constexpr (M::PLANES == 2) c[1][i] = hi;
        }
    }
#pragma unroll
    for (int j = 0; j < M::PLANES; j++) {
        uint4* q = reinterpret_cast<uint4*>(p + 1024 * j) + row;
        q[0] = uint4{c[j][0], c[j][1], c[j][2], c[j][3]};
        q[32] = uint4{c[j][4], c[j][5], c[j][6], c[j][7]};
    }
    uint2* s = reinterpret_cast<uint2*>(p + 1024 * M::PLANES) + row;
    s[0] = piece_words(live ? d : 0.0f);
#pragma unroll
    for (int h = 0; h < M::MINS; h++) s[32 * (1 + h)] = piece_words(live ? -w.m[h] * MIN_UNIT : 0.0f);
}

struct LayoutArgs {
    const uint8_t* w;
    uint8_t* wl;            // the weight's panels
    const int8_t* q;
    const float* s;
    uint8_t* xl;            // the rows' panels
    int64_t row_bytes, n, t, k;
    int64_t w_blocks;       // workgroups that lay out the weight; the rest take the rows
    int groups;             // of a row, rounded up to the stages' (the last ones hold zeros)
};

// A workgroup lays out 32 rows by 8 groups, a group to a thread: the lanes of
// a half wave write 512 bytes in a row. 333 rows and q4_0 4,099 x 4,096: 13 us.
template <int TYPE>
__global__ __launch_bounds__(256) void k_lay_out(LayoutArgs a) {
    using M = MatrixFormat<TYPE>;
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
    const int from = live ? g : live_groups - 1;
    if (weight) {
        const int64_t n = panel * 32 + row;
        Raw<TYPE> raw;
        qsd::load_row_group<TYPE>(a.w + (n < a.n ? n : a.n - 1) * a.row_bytes, from, raw);
        lay_out_weight<TYPE>(raw, qsd::group_in_block<TYPE>(from), grid, live,
                             a.wl + (panel * a.groups + g) * panel_group_bytes(M::PLANES, M::MINS), row);
        return;
    }
    const int64_t t = panel * 32 + row, at = t < a.t ? t : a.t - 1;
    const uint4* x = reinterpret_cast<const uint4*>(a.q + at * a.k + 32 * from);
    const uint4 lo = x[0], hi = x[1];
    const float s = live ? a.s[at * live_groups + from] : 0.0f;
    uint8_t* p = a.xl + (panel * a.groups + g) * panel_group_bytes(1, M::MINS);
    reinterpret_cast<uint4*>(p)[row] = lo;
    reinterpret_cast<uint4*>(p)[32 + row] = hi;
    uint2* o = reinterpret_cast<uint2*>(p + 1024) + row;
    o[0] = piece_words(s);
    if constexpr (M::MINS > 0) {
        const int o0 = dot4(lo.x, qsd::ONES, dot4(lo.y, qsd::ONES, dot4(lo.z, qsd::ONES, dot4(lo.w, qsd::ONES, 0))));
        const int o1 = dot4(hi.x, qsd::ONES, dot4(hi.y, qsd::ONES, dot4(hi.z, qsd::ONES, dot4(hi.w, qsd::ONES, 0))));
        o[32] = piece_words(s * ((float)(M::MINS == 2 ? o0 : o0 + o1) * CODE_SUM_UNIT));
        if constexpr (M::MINS == 2) o[64] = piece_words(s * ((float)o1 * CODE_SUM_UNIT));
    }
}

// ---- the product ----

QS_DEV AdapterTile adapter_tile(const LinearArgs& l) {
    return {l.ids, l.off, l.b, l.v_hi, l.v_lo, l.v_rest, l.v_unit, l.ldv, l.adapters};
}

// A wave's units to memory of a type: rows from t0, columns from n0 to `end`. Element i
// of a unit: row 8 (i / 4) + 4 half + i % 4, column lane % 32.
template <int UM, int UN>
QS_DEV void store_tile(void* to, int type, const LinearArgs& l, const f32x16 (&y)[UM][UN], int64_t t0, int64_t n0, int64_t end) {
    const int lane = threadIdx.x % 64, col = lane % 32, half = lane / 32;
    const auto store = [&](auto* dst) {
        using T = std::remove_pointer_t<decltype(dst)>;
#pragma unroll
        for (int um = 0; um < UM; um++)
#pragma unroll
            for (int i = 0; i < 16; i++) {
                const int64_t t = t0 + um * 32 + 8 * (i / 4) + 4 * half + i % 4;
                T* row = dst + t * l.n + n0 + col;
#pragma unroll
                for (int un = 0; un < UN; un++)
                    if (t < l.t && n0 + un * 32 + col < end) row[un * 32] = (T)y[um][un][i];
            }
    };
    if (type == QS_SRC_F32) store(static_cast<float*>(to));
    else if (type == QS_SRC_F16) store(static_cast<_Float16*>(to));
    else store(static_cast<__bf16*>(to));
}

// The sums of WK waves that hold the same units, in the first one, one wave's
// after another's; a column of units of all PARTS waves at a time in LDS.
template <int WK, int PARTS, int UM, int UN>
QS_DEV void join_waves(f32x16 (&acc)[UM][UN], float* lds, int wk, int part) {
    const int lane = threadIdx.x % 64;
#pragma unroll
    for (int w = 1; w < WK; w++)
#pragma unroll
        for (int un = 0; un < UN; un++) {
            __syncthreads();
            if (wk == w)
#pragma unroll
                for (int um = 0; um < UM; um++)
#pragma unroll
                    for (int i = 0; i < 16; i++) lds[((part * UM + um) * 16 + i) * 64 + lane] = acc[um][un][i];
            __syncthreads();
            if (wk == 0)
#pragma unroll
                for (int um = 0; um < UM; um++)
#pragma unroll
                    for (int i = 0; i < 16; i++) acc[um][un][i] += lds[((part * UM + um) * 16 + i) * 64 + lane];
        }
}

// 16 bytes a lane from memory to LDS, a wave's 1,024 in a row from `to`
QS_DEV void copy_to_lds(const uint8_t* from, uint8_t* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}

// A tile of BM rows by BN weight rows. Two stages of G groups lie in LDS; while
// one is multiplied the next one's copies are in flight. WM x WN waves split the
// tile, WK the groups of a stage (their sums are joined in LDS at the end, in
// order). The stages are two arrays, and places in them one sum, so that the
// compiler sees that a read of one does not wait for copies to the other.
// Each 32 x 32 x 32 of codes takes three units of matrix time or more: the codes'
// instruction (37 clocks), the scales' outer product (32), a minimum's (32) and 32
// vector instructions that apply it (80), which do not overlap with them. 4,000
// rows with q4_0 4,096 x 2,560, layout included: 121 us, 0.69 PFLOP/s; 333 with
// 4,099 x 4,096: 31 us of product, where one round of 64 x 64 fills the chip once.
template <int PLANES, int MINS, int BM, int BN, int WM, int WN, int WK, int G, int ADAPT>
__global__ __launch_bounds__(64 * WM * WN * WK, 2) void k_matrix(MatrixArgs a) {
    constexpr int WAVES = WM * WN * WK, UM = BM / WM / 32, UN = BN / WN / 32, GW = G / WK;
    constexpr int XB = panel_group_bytes(1, MINS), WB = panel_group_bytes(PLANES, MINS);
    // a panel's G groups lie together in memory and in LDS
    constexpr int XP = G * XB, WP = G * WB, XS = BM / 32 * XP, WS = BN / 32 * WP, STAGE = XS + WS;
    constexpr int COPIES = (STAGE / 1024 + WAVES - 1) / WAVES;
    static_assert(XP % 256 == 0 && WP % 256 == 0 && XS % 1024 == 0 && WS % 1024 == 0 && G % WK == 0, "copies of 1,024 bytes");
    __shared__ __attribute__((aligned(1024))) uint8_t even[STAGE], odd[STAGE];
    const int tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    const int wn = wave % WN, wm = wave / WN % WM, wk = wave / WN / WM, col = lane % 32, half = lane / 32;
    const LinearArgs& l = a.l;
    // Workgroups go round the 8 XCDs in turn; each XCD takes a run of tiles, in
    // strips of 8 columns of tiles, so that what it works on at a time shares
    // rows and weights in its L2.
    const int64_t tiles_m = (l.t + BM - 1) / BM, tiles_n = (a.count + BN - 1) / BN, tiles = tiles_m * tiles_n;
    const int64_t at = (int64_t)(blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8;
    if (at >= tiles) return;
    const int64_t strip = at / (8 * tiles_m), left = tiles_n - 8 * strip, wide = left < 8 ? left : 8;
    const int64_t in = at - strip * 8 * tiles_m;
    const int64_t t0 = in / wide * BM, n0 = (8 * strip + in % wide) * BN;
    const int stages = a.groups / G;

    // This wave's copies of a stage: 1,024 bytes each, over both factors' panels;
    // panels past the last (a tile may reach past the layout) are the last again.
    const int64_t x_step = (int64_t)a.groups * XB, w_step = (int64_t)a.groups * WB;
    const int last_x = (int)((l.t - 1) / 32 - t0 / 32), last_w = (int)((a.count - 1) / 32 - n0 / 32);
    const uint8_t* from[COPIES];
#pragma unroll
    for (int i = 0; i < COPIES; i++) {
        const int c = i * WAVES + wave, byte = c * 1024 + lane * 16;
        const bool x = byte < XS;
        const int in_s = x ? byte : byte - XS, p = in_s / (x ? XP : WP), o = in_s - p * (x ? XP : WP);
        from[i] = x ? a.xl + (t0 / 32 + (p < last_x ? p : last_x)) * x_step + o
                    : a.wl + (n0 / 32 + (p < last_w ? p : last_w)) * w_step + o;
    }
    auto copy = [&](int stage, uint8_t* to) {
#pragma unroll
        for (int i = 0; i < COPIES; i++) {
            const int c = i * WAVES + wave;
            if (STAGE / 1024 % WAVES && c >= STAGE / 1024) break;
            copy_to_lds(from[i] + (int64_t)stage * (c * 1024 < XS ? XP : WP), to + c * 1024);
        }
    };

    f32x16 acc[UM][UN] = {};
    const int b = __float_as_int(INT_BIAS);
    const i32x16 bias = {b, b, b, b, b, b, b, b, b, b, b, b, b, b, b, b};
    // a scale's slots: rows d1 d1 d1 d2 | d2 d2 d3 d3, columns s1 s2 s3 s1 | s2 s3 s1 s2
    const uint32_t xsel0 = half ? 0x03020302u : 0x01000100u, xsel1 = half ? 0x05040504u : 0x03020100u;
    const uint32_t wsel0 = half ? 0x05040302u : 0x03020100u, wsel1 = half ? 0x03020100u : 0x01000504u;
    i32x4 xa[UM], wb[PLANES][UN];
    s16x4 xp[1 + MINS][UM], wp[1 + MINS][UN];     // bf16
    auto slots = [&](const uint8_t* p, uint32_t s0, uint32_t s1) {
        const uint2 w = *reinterpret_cast<const uint2*>(p);
        return __builtin_bit_cast(s16x4, uint2{__builtin_amdgcn_perm(w.y, w.x, s0), __builtin_amdgcn_perm(w.y, w.x, s1)});
    };
    const int x0 = wm * UM * XP + wk * GW * XB, w0 = XS + wn * UN * WP + wk * GW * WB;
    const int xl0 = x0 + lane * 16, xs0 = x0 + 1024 + col * 8, wl0 = w0 + lane * 16, ws0 = w0 + 1024 * PLANES + col * 8;
    auto operands = [&](const uint8_t* stage, int g) {
#pragma unroll
        for (int u = 0; u < UM; u++) {
            xa[u] = *reinterpret_cast<const i32x4*>(stage + (xl0 + (u * XP + g * XB)));
#pragma unroll
            for (int h = 0; h <= MINS; h++) xp[h][u] = slots(stage + (xs0 + (u * XP + g * XB + 256 * h)), xsel0, xsel1);
        }
#pragma unroll
        for (int u = 0; u < UN; u++) {
#pragma unroll
            for (int j = 0; j < PLANES; j++)
                wb[j][u] = *reinterpret_cast<const i32x4*>(stage + (wl0 + (u * WP + g * WB + 1024 * j)));
#pragma unroll
            for (int h = 0; h <= MINS; h++) wp[h][u] = slots(stage + (ws0 + (u * WP + g * WB + 256 * h)), wsel0, wsel1);
        }
    };
    constexpr int UNITS = UM * UN, STEPS = GW * UNITS;
    static_assert(UNITS > 1, "the operands of a group are read two steps ahead");
    f32x16 ds[2];
    i32x16 p[2], ph[2];
    auto scale_step = [&](int s) {
        const int u = s % UNITS;
        ds[s % 2] = __builtin_amdgcn_mfma_f32_32x32x8bf16_1k(xp[0][u / UN], wp[0][u % UN], f32x16{}, 0, 0, 0);
    };
    auto code_step = [&](int s) {
        const int u = s % UNITS;
        p[s % 2] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xa[u / UN], wb[0][u % UN], PLANES == 1 ? bias : i32x16{}, 0, 0, 0);
        if constexpr (PLANES == 2) ph[s % 2] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xa[u / UN], wb[1][u % UN], i32x16{}, 0, 0, 0);
    };
    auto min_step = [&](int s) {
        const int u = s % UNITS;
#pragma unroll
        for (int h = 1; h <= MINS; h++)
            acc[u / UN][u % UN] = __builtin_amdgcn_mfma_f32_32x32x8bf16_1k(xp[h][u / UN], wp[h][u % UN], acc[u / UN][u % UN], 0, 0, 0);
    };
    auto add = [&](int s, int from) {
        const int u = s % UNITS;
#pragma unroll
        for (int i = from; i < from + 8; i++) {
            const float c = PLANES == 1 ? __int_as_float(p[s % 2][i]) - INT_BIAS
                                        : (float)(int)(((uint32_t)ph[s % 2][i] << 7) + (uint32_t)p[s % 2][i]);
            acc[u / UN][u % UN][i] = __builtin_fmaf(c, ds[s % 2][i], acc[u / UN][u % UN][i]);
        }
    };
    auto turn = [&](const uint8_t* stage, uint8_t* next, int after) {
        // this wave's copies of the stage have landed; after the barrier all have,
        // and no wave reads the other stage any more
        __builtin_amdgcn_s_waitcnt(0x0f70);     // vmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        copy(after < stages ? after : stages - 1, next);    // no branch: the last stage again
        __builtin_amdgcn_sched_barrier(0);                  // they go out first
        // The matrix instructions of a step are issued before the vector ones
        // of the step before it, so a wave's vector work covers their latency.
        operands(stage, 0);
        scale_step(0);
        code_step(0);
        min_step(0);
#pragma unroll
        for (int s = 0; s < STEPS; s++) {
            const bool more = s + 1 < STEPS;
            __builtin_amdgcn_sched_barrier(0);
            if (more) scale_step(s + 1);
            __builtin_amdgcn_sched_barrier(0);
            add(s, 0);
            __builtin_amdgcn_sched_barrier(0);
            if (more) code_step(s + 1);
            __builtin_amdgcn_sched_barrier(0);
            add(s, 8);
            __builtin_amdgcn_sched_barrier(0);
            if (more) min_step(s + 1);
            if ((s + 2) % UNITS == 0 && s + 2 < STEPS) operands(stage, (s + 2) / UNITS);
        }
    };
    copy(0, even);
    for (int s = 0; s < stages; s += 2) {       // an even number of stages
        turn(even, odd, s + 1);
        turn(odd, even, s + 2);
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);     // no copy to LDS outlives the workgroup
    if constexpr (ADAPT)
        add_adapters<ADAPT, 3, WK>(adapter_tile(l), acc, t0 + wm * UM * 32, l.t, a.first + n0 + wn * UN * 32, l.n, wk);
    if constexpr (WK > 1) {
        join_waves<WK, WM * WN>(acc, reinterpret_cast<float*>(even), wk, wm * WN + wn);
        static_assert(STAGE >= BM * BN * 4 / UN, "a column of units");
        if (wk > 0) return;
    }
    store_tile(l.dst, l.dst_type, l, acc, t0 + wm * UM * 32, a.first + n0 + wn * UN * 32, a.first + a.count);
}

}  // namespace qsl
