// Products of 8-bit rows with packed weights (gfx950):
//     y[t, n] = sum over groups g of  s[t, g] * (d[n, g] * sum c q - m[n, g] * sum q)
// The inner sums are integers and exact: v_dot4_i32_i8 for a few rows, the
// 8-bit matrix instructions for more. Only their results are scaled, in f32,
// so no value of the weight or of the rows is ever rounded to fewer bits; the
// result is rounded once, when it is stored.
#pragma once

#include <hip/hip_fp16.h>

#include "qs_decode.h"
#include "qs_linear.h"

namespace qsl {

using qsd::Format;
using qsd::Group;
using qsd::Raw;

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int64_t i64x2 __attribute__((ext_vector_type(2)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

QS_DEV int dot4(uint32_t a, uint32_t b, int c) { return __builtin_amdgcn_sdot4((int)a, (int)b, c, false); }

QS_DEV void store_value(const LinearArgs& a, int64_t at, float v) {
    if (a.dst_type == QS_SRC_F32) static_cast<float*>(a.dst)[at] = v;
    else if (a.dst_type == QS_SRC_F16) static_cast<_Float16*>(a.dst)[at] = (_Float16)v;
    else static_cast<__bf16*>(a.dst)[at] = (__bf16)v;
}

QS_DEV float value16(uint32_t bits, int type) {
    return type == QS_SRC_BF16 ? __uint_as_float(bits << 16) : qsd::half_bits(bits);
}

// the adapter of row t, -1 where it has none
QS_DEV int adapter_of(const LinearArgs& a, int64_t t) {
    const int id = a.ids[t];
    return id >= 0 && id < a.adapters ? id : -1;
}

// the part of  sum over r of v[t, r] * B[n, r]  with r / 8 = first, first + step, ...
QS_DEV float adapter_sum(const LinearArgs& a, int id, int64_t t, int64_t n, int first, int step) {
    const int o = a.off[id], rank = a.off[id + 1] - o;
    const uint16_t* b = a.b + a.n * o + n * rank;
    const float* v = a.v + t * a.ldv;
    float sum = 0.0f;
    for (int r = 8 * first; r < rank; r += 8 * step) {
        uint32_t w[4];
        __builtin_memcpy(w, __builtin_assume_aligned(b + r, 16), 16);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            sum = __builtin_fmaf(v[r + 2 * i], value16(w[i] & 0xffffu, a.b_type), sum);
            sum = __builtin_fmaf(v[r + 2 * i + 1], value16(w[i] >> 16, a.b_type), sum);
        }
    }
    return sum;
}

// wait for LDS only: loads from memory stay in flight across the barrier
QS_DEV void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// The sum over each 16 neighbouring lanes, in all of them. Cross-lane moves
// inside the vector unit: a shuffle through LDS takes its latency for every
// doubling.
template <int CTRL>
QS_DEV float add_lane(float v) {
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 15, 15, true));
}
QS_DEV float sum16(float v) {
    v = add_lane<0xb1>(v);          // quad_perm 1 0 3 2
    v = add_lane<0x4e>(v);          // quad_perm 2 3 0 1
    v = add_lane<0x141>(v);         // row_half_mirror
    return add_lane<0x140>(v);      // row_mirror
}

// ---- a few rows ----

// The LDS of a workgroup of k_linear_few: the bytes of its weight rows, up to
// whole 16s at both ends, then x, then the grid.
struct FewPlan {
    int w_bytes;
    int64_t blocks;         // of a workgroup's weight rows
};

// Bytes from .. to of memory, 16 at a time on 16-byte boundaries, through
// registers to LDS, which receives byte from - from % 16 on. Bytes outside the
// weight (lo .. hi) are not read.
struct Run {
    const uint8_t* base;
    int chunks;
};
QS_DEV Run run_of(const uint8_t* from, const uint8_t* to) {
    const uint8_t* base = from - (reinterpret_cast<uintptr_t>(from) & 15);
    return {base, (int)((to - base + 15) / 16)};
}
QS_DEV uint4 read_chunk(const Run& r, int c) { return reinterpret_cast<const uint4*>(r.base)[c]; }
// one that may reach over an end of the weight
QS_DEV uint4 read_end(const Run& r, int c, const uint8_t* lo, const uint8_t* hi) {
    const uint8_t* p = r.base + 16 * (int64_t)c;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint8_t* q = p + 4 * i;
        w[i] = q >= lo && q + 2 <= hi ? qsd::load_u16(q) : 0;
        w[i] |= q + 2 >= lo && q + 4 <= hi ? qsd::load_u16(q + 2) << 16 : 0;
    }
    return uint4{w[0], w[1], w[2], w[3]};
}

// A workgroup takes blocks of 256 / L weight rows in turn. A block is one run
// of bytes: it is copied to LDS whole, 16 bytes a lane (read from memory group
// by group, blocks of 18, 34, 66 .. 210 bytes, which start at any even byte,
// cost several times the loads, each of them split), the next block's bytes in
// flight while one is multiplied. L lanes take the groups of a row in turn. x
// is in LDS too, for each group and row of x 32 codes, the scale and the sums of
// codes that an offset of the weight's integers (OFFSET) or a minimum multiplies:
// 48 bytes, the T of a group together, so that a lane reads them at constant
// offsets, and an odd number of 16s a group, which spreads lanes over the banks.
// One row is bound by reading a large weight (151,936 x 2,560: q8_0 72 us, 5.7
// TB/s; q6_k 65 us, 4.9 TB/s; q4_k 47 us, 4.6 TB/s), of the types under 4 bits by
// decoding it (iq2_xxs 60 us, q3_k 62), and by the latency of what comes one after
// another in a small one (q4_k 9,728 x 2,560, 14 MB: 7.2 us). More rows add LDS
// reads and dot products: five with q6_k 151,936 x 2,560 90 us, 3.6 TB/s.
template <int TYPE, int T, int L>
__global__ __launch_bounds__(256) void k_linear_few(LinearArgs a, FewPlan plan) {
    constexpr int SUB = Format<TYPE>::SUB, AHEAD = 8, ROWS = 256 / L, OFFSET = qsd::offset<TYPE>();
    constexpr bool MIN = Format<TYPE>::MIN;
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    const int groups = (int)(a.k / 32), t1 = (int)a.t - 1, tid = threadIdx.x;
    constexpr int REC = few_record(T);
    uint4* x0 = reinterpret_cast<uint4*>(lds + plan.w_bytes);
    uint16_t* grid = reinterpret_cast<uint16_t*>(x0 + REC * groups);
    const uint8_t *lo_end = a.w, *hi_end = a.w + a.n * a.row_bytes;
    auto rows_of = [&](int64_t block) { return a.n - block * ROWS < ROWS ? (int)(a.n - block * ROWS) : ROWS; };
    auto from_of = [&](int64_t block) { return a.w + block * ROWS * a.row_bytes; };
    auto over_end = [&](const Run& r) { return r.base < lo_end || r.base + 16 * (int64_t)r.chunks > hi_end; };
    uint4 ahead[AHEAD];
    auto read_ahead = [&](int64_t block) {
        const Run run = run_of(from_of(block), from_of(block) + rows_of(block) * a.row_bytes);
        if (over_end(run)) return;
#pragma unroll
        for (int j = 0; j < AHEAD; j++)     // a lane past the end reads the last 16 bytes again
            ahead[j] = read_chunk(run, tid + 256 * j < run.chunks ? tid + 256 * j : run.chunks - 1);
    };
    read_ahead(blockIdx.x);
    qsd::stage_grid<TYPE>(grid, tid, 256);
    for (int t = 0; t < T; t++) {
        const int64_t row = t < t1 ? t : t1;
        for (int g = tid; g < groups; g += 256) {
            const uint4* q = reinterpret_cast<const uint4*>(a.q + row * a.k) + 2 * g;
            const uint4 lo = q[0], hi = q[1];
            const int o0 = dot4(lo.x, qsd::ONES, dot4(lo.y, qsd::ONES, dot4(lo.z, qsd::ONES, dot4(lo.w, qsd::ONES, 0))));
            const int o1 = dot4(hi.x, qsd::ONES, dot4(hi.y, qsd::ONES, dot4(hi.z, qsd::ONES, dot4(hi.w, qsd::ONES, 0))));
            constexpr int F = MIN ? 1 : -OFFSET;
            uint4* x = x0 + REC * g + 3 * t;
            x[0] = lo;
            x[1] = hi;
            x[2] = uint4{__float_as_uint(qsd::scale_of(a.s[row * groups + g])), (uint32_t)(F * (SUB == 2 ? o0 : o0 + o1)), (uint32_t)(F * o1), 0};
        }
    }
    const int lane = tid % L, r0 = tid / L;
    for (int64_t block = blockIdx.x; block < plan.blocks; block += gridDim.x) {
        const int rows = rows_of(block);
        const uint8_t* from = from_of(block);
        const Run run = run_of(from, from + rows * a.row_bytes);
        if (block != blockIdx.x) lds_barrier();     // the block before is done with
        uint4* to = reinterpret_cast<uint4*>(lds);
        if (over_end(run)) {
            for (int c = tid; c < run.chunks; c += 256) to[c] = read_end(run, c, lo_end, hi_end);
        } else {
#pragma unroll
            for (int j = 0; j < AHEAD; j++)
                if (tid + 256 * j < run.chunks) to[tid + 256 * j] = ahead[j];
            // rows longer than the registers hold ahead
            for (int c = tid + 256 * AHEAD; c < run.chunks; c += 256) to[c] = read_chunk(run, c);
        }
        if (block + gridDim.x < plan.blocks) read_ahead(block + gridDim.x);
        lds_barrier();
        const qsd::LdsBytes<Format<TYPE>::BYTES % 4 != 0> at{
            lds, (int)(reinterpret_cast<uintptr_t>(from) & 15) + (r0 < rows ? r0 : rows - 1) * (int)a.row_bytes};
        float acc[T] = {};
        for (int g = lane; g < groups; g += L) {
            Raw<TYPE> raw;
            Group<TYPE> w;
            qsd::load_row_group<TYPE>(at, g, raw);
            qsd::decode_group<TYPE, true>(raw, qsd::group_in_block<TYPE>(g), grid, w);
#pragma unroll
            for (int t = 0; t < T; t++) {
                const uint4 *p = x0 + REC * g + 3 * t, lo = p[0], hi = p[1], rest = p[2];
                const uint32_t x[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                const int o[2] = {(int)rest.y, (int)rest.z};
                int c[SUB];
#pragma unroll
                for (int h = 0; h < SUB; h++) c[h] = OFFSET ? o[h] : 0;
#pragma unroll
                for (int i = 0; i < 8; i++) c[i * SUB / 8] = dot4(w.c[i], x[i], c[i * SUB / 8]);
                float y = 0.0f;
#pragma unroll
                for (int h = 0; h < SUB; h++) {
                    y = h ? __builtin_fmaf(w.d[h], (float)c[h], y) : w.d[h] * (float)c[h];
                    if (MIN) y = __builtin_fmaf(-w.m[h], (float)o[h], y);
                }
                acc[t] = __builtin_fmaf(__uint_as_float(rest.x), y, acc[t]);
            }
        }
        const int64_t n = block * ROWS + r0;
        if (a.v && r0 < rows)
#pragma unroll
            for (int t = 0; t < T; t++) {
                const int id = t <= t1 ? adapter_of(a, t) : -1;
                if (id >= 0) acc[t] += adapter_sum(a, id, t, n, lane, L);
            }
        float y = 0.0f;         // lane t keeps row t's sum, and the lanes store together
#pragma unroll
        for (int t = 0; t < T; t++) {
            float v = sum16(acc[t]);
            if (L == 64) v += __shfl_xor(v, 16), v += __shfl_xor(v, 32);
            y = lane == t ? v : y;
        }
        if (lane <= t1 && r0 < rows) store_value(a, lane * a.n + n, y);
    }
}

// ---- more rows ----

// An int32 matrix product starts from this word in every place, so that the
// result's bits are the float 1.5 * 2^23 + sum (|sum| <= 32 * 128 * 128 < 2^22):
// a subtraction at full rate in place of a conversion at half rate.
constexpr float INT_BIAS = 12582912.0f;

// A minimum is multiplied by s * (sum of codes), which can pass f32's largest number
// where no value does: 2^-12 of it, against 2^12 times the minimum.
constexpr float CODE_SUM_UNIT = 0x1p-12f, MIN_UNIT = 0x1p12f;

// Each sum is scaled by d[n] * s[t]: a product per element and group, as much
// vector work as the sums themselves are matrix work. It is an outer product,
// so the matrix units form it: a factor is cut into three bf16 pieces that add
// up to it exactly (8 bits each of its 24), and eight of the nine products of
// pieces, which bf16 MFMA sums in f32, miss the product by less than 2^-30 of
// it. Slot by slot: d1 d1 d1 d2 d2 d2 d3 d3 against s1 s2 s3 s1 s2 s3 s1 s2.
struct Pieces {
    uint32_t a, b, c;       // the top halves of three floats
};
QS_DEV Pieces pieces(float f) {
    Pieces p;
    p.a = __float_as_uint(f) & 0xffff0000u;
    const float r = f - __uint_as_float(p.a);
    p.b = __float_as_uint(r) & 0xffff0000u;
    p.c = __float_as_uint(r - __uint_as_float(p.b));
    return p;
}
QS_DEV uint32_t two(uint32_t lo, uint32_t hi) { return (lo >> 16) | (hi & 0xffff0000u); }
QS_DEV uint4 weight_slots(float f) {
    const Pieces p = pieces(f);
    return uint4{two(p.a, p.a), two(p.a, p.b), two(p.b, p.b), two(p.c, p.c)};
}
QS_DEV uint4 row_slots(float f) {
    const Pieces p = pieces(f);
    return uint4{two(p.a, p.b), two(p.c, p.a), two(p.b, p.c), two(p.a, p.b)};
}

template <int TYPE, int BM, int BN, int WM, int WN, int WK, int G>
struct Tile {
    static constexpr int THREADS = 64 * WM * WN * WK, SUB = Format<TYPE>::SUB;
    static constexpr bool MIN = Format<TYPE>::MIN;
    static constexpr int UM = BM / WM / 32, UN = BN / WN / 32;
    // Offsets in LDS, bytes. Codes lie in halves of 16 values, a half's rows
    // one after another, so that the 32 lanes of a matrix operand read 512 bytes
    // in a row; 32 bytes between groups spread the threads that write different
    // groups of a row over the banks.
    static constexpr int XQS = BM * 32 + 32, WQS = BN * 32 + 32, XPS = BM * 16 + 32, WPS = BN * 16 + 32;
    static constexpr int XQ = 0, WQ = XQ + G * XQS, XP = WQ + G * WQS, WP = XP + G * XPS, XM = WP + G * SUB * WPS,
                         WMN = XM + (MIN ? G * SUB * XPS : 0), ZERO = WMN + (MIN ? G * SUB * WPS : 0),
                         GRID = ZERO + 16, STAGE = GRID + Format<TYPE>::GRID * 2, JOIN = (WK - 1) * BM * BN * 4,
                         BYTES = STAGE > JOIN ? STAGE : JOIN;
    static constexpr int WTASKS = (BN * G + THREADS - 1) / THREADS, XTASKS = (BM * G + THREADS - 1) / THREADS;
    // matrix steps of a wave between two stages
    static constexpr int UNITS = UM * UN, STEPS = G / WK * UNITS * SUB;
    static constexpr bool PAIR = SUB == 1 && G / WK % 2 == 0;      // minima of two groups in a matrix instruction
    static_assert(G % WK == 0, "groups of a wave");
};

// A tile of BM rows by BN weight rows. The workgroup's WM x WN x WK waves
// stage G groups of 32 values at a time: the weight's are decoded to bytes by
// a thread a group, the rows' copied; the bytes of the next stage are in
// flight while one is multiplied (two or three stages ahead, whose registers
// leave fewer waves, took 5 to 15% longer). WM x WN waves split the tile, WK the
// groups (their sums are joined in LDS at the end, in order). A group's 16
// products a lane are scaled by an outer product of the scales, d * s, that a
// matrix instruction makes from three bf16 pieces of each, exact to f32.
// Bound by the turn of a stage: decode and copies to LDS, a barrier, products, a
// barrier, one after another: with 64 rows of q4_k 9,728 x 2,560 vector
// instructions take about a fifth of the SIMDs' cycles, matrix ones a twentieth,
// with 128 of q6_k 151,936 x 2,560 half and a sixth. 64 rows 21 us, 152 TFLOP/s; 16
// rows 16 us; 128 with q6_k 151,936 x 2,560 493 us, 202 TFLOP/s.
template <int TYPE, int BM, int BN, int WM, int WN, int WK, int G>
__global__ __launch_bounds__(64 * WM * WN * WK, 2) void k_linear_tile(LinearArgs a) {
    using S = Tile<TYPE, BM, BN, WM, WN, WK, G>;
    constexpr int THREADS = S::THREADS, SUB = S::SUB, UM = S::UM, UN = S::UN;
    constexpr bool MIN = S::MIN;
    __shared__ __attribute__((aligned(16))) uint8_t lds[S::BYTES];
    uint16_t* grid = reinterpret_cast<uint16_t*>(lds + S::GRID);
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const int wk = wave % WK, wn = wave / WK % WN, wmr = wave / WK / WN;
    const int col = lane % 32, half = lane / 32;
    // Workgroups go round the 8 XCDs in turn; each XCD takes a run of tiles, in
    // strips of 8 columns of tiles, so that what it works on at a time shares
    // rows and weights in its L2.
    const int64_t tiles_m = (a.t + BM - 1) / BM, tiles_n = (a.n + BN - 1) / BN, tiles = tiles_m * tiles_n;
    const int64_t number = (int64_t)blockIdx.y * gridDim.x + blockIdx.x, workgroups = (int64_t)gridDim.y * gridDim.x;
    const int64_t place = number % 8 * (workgroups / 8) + number / 8, at = place % tiles;
    if (place >= tiles * a.splits) return;
    const int64_t strip = at / (8 * tiles_m), left = tiles_n - 8 * strip, wide = left < 8 ? left : 8;
    const int64_t in = at - strip * 8 * tiles_m;
    const int64_t t0 = in / wide * BM, n0 = (8 * strip + in % wide) * BN;
    const int groups = (int)(a.k / 32), stages = (groups + G - 1) / G, per = (stages + a.splits - 1) / a.splits;
    const int split = (int)(place / tiles), begin = split * per * G, end = (split + 1) * per * G < groups ? (split + 1) * per * G : groups;

    qsd::stage_grid<TYPE>(grid, tid, THREADS);
    if (tid < 4) reinterpret_cast<uint32_t*>(lds + S::ZERO)[tid] = 0;
    // this thread's part of every stage
    const uint8_t* wrow[S::WTASKS];
    const int8_t* xrow[S::XTASKS];
    const float* srow[S::XTASKS];
    Raw<TYPE> wraw[S::WTASKS];
    uint4 xraw[S::XTASKS][2];
    float sraw[S::XTASKS];
#pragma unroll
    for (int j = 0; j < S::WTASKS; j++) {
        const int64_t n = n0 + (tid + j * THREADS) / G;
        wrow[j] = a.w + (n < a.n ? n : a.n - 1) * a.row_bytes;
    }
#pragma unroll
    for (int j = 0; j < S::XTASKS; j++) {
        const int64_t t = t0 + (tid + j * THREADS) / G;
        xrow[j] = a.q + (t < a.t ? t : a.t - 1) * a.k;
        srow[j] = a.s + (t < a.t ? t : a.t - 1) * groups;
    }
    // past the last group: its bytes again, to be placed with scales of 0
    auto load = [&](int g0) {
#pragma unroll
        for (int j = 0; j < S::WTASKS; j++) {
            const int i = tid + j * THREADS, g = g0 + i % G < groups ? g0 + i % G : groups - 1;
            if (BN * G % THREADS == 0 || i < BN * G) qsd::load_row_group<TYPE>(wrow[j], g, wraw[j]);
        }
#pragma unroll
        for (int j = 0; j < S::XTASKS; j++) {
            const int i = tid + j * THREADS, g = g0 + i % G < groups ? g0 + i % G : groups - 1;
            if (BM * G % THREADS == 0 || i < BM * G) {
                const uint4* p = reinterpret_cast<const uint4*>(xrow[j] + 32 * g);
                xraw[j][0] = p[0];
                xraw[j][1] = p[1];
                sraw[j] = srow[j][g];
            }
        }
    };
    auto put = [&](int at, uint4 v) { *reinterpret_cast<uint4*>(lds + at) = v; };
    auto put_stage = [&](int g0) {
#pragma unroll
        for (int j = 0; j < S::WTASKS; j++) {
            const int i = tid + j * THREADS, g = i % G, r = i / G;
            if (!(BN * G % THREADS == 0 || i < BN * G)) continue;
            const bool live = g0 + g < groups;
            Group<TYPE> w;
            qsd::decode_group<TYPE>(wraw[j], qsd::group_in_block<TYPE>(live ? g0 + g : groups - 1), grid, w);
            put(S::WQ + g * S::WQS + r * 16, uint4{w.c[0], w.c[1], w.c[2], w.c[3]});
            put(S::WQ + g * S::WQS + (BN + r) * 16, uint4{w.c[4], w.c[5], w.c[6], w.c[7]});
#pragma unroll
            for (int h = 0; h < SUB; h++) {
                put(S::WP + (g * SUB + h) * S::WPS + r * 16, weight_slots(live ? w.d[h] : 0.0f));
                if constexpr (MIN) put(S::WMN + (g * SUB + h) * S::WPS + r * 16, weight_slots(live ? -w.m[h] * MIN_UNIT : 0.0f));
            }
        }
#pragma unroll
        for (int j = 0; j < S::XTASKS; j++) {
            const int i = tid + j * THREADS, g = i % G, r = i / G;
            if (!(BM * G % THREADS == 0 || i < BM * G)) continue;
            const uint4 lo = xraw[j][0], hi = xraw[j][1];
            const float s = g0 + g < groups ? sraw[j] : 0.0f;
            put(S::XQ + g * S::XQS + r * 16, lo);
            put(S::XQ + g * S::XQS + (BM + r) * 16, hi);
            put(S::XP + g * S::XPS + r * 16, row_slots(s));
            if constexpr (MIN) {
                const int o0 = dot4(lo.x, qsd::ONES, dot4(lo.y, qsd::ONES, dot4(lo.z, qsd::ONES, dot4(lo.w, qsd::ONES, 0))));
                const int o1 = dot4(hi.x, qsd::ONES, dot4(hi.y, qsd::ONES, dot4(hi.z, qsd::ONES, dot4(hi.w, qsd::ONES, 0))));
                put(S::XM + g * SUB * S::XPS + r * 16, row_slots(s * ((float)(SUB == 2 ? o0 : o0 + o1) * CODE_SUM_UNIT)));
                if constexpr (SUB == 2) put(S::XM + (g * SUB + 1) * S::XPS + r * 16, row_slots(s * ((float)o1 * CODE_SUM_UNIT)));
            }
        }
    };

    f32x16 acc[UM][UN] = {};
    const int b = __float_as_int(INT_BIAS);
    const i32x16 bias = {b, b, b, b, b, b, b, b, b, b, b, b, b, b, b, b};
    const int m0 = (wmr * UM * 32 + col) * 16, c0 = (wn * UN * 32 + col) * 16;      // bytes
    // operands of the group in hand
    i32x4 xa[UM], wb[UN];           // SUB 1: 16 of the 32 values a half wave
    i64x2 xa2[UM], wb2[UN];         // SUB 2: 8 of 16, twice
    bf16x8 xp[UM], wp[SUB][UN], xm[UM], wm[UN];
    auto at128 = [&](int at) { return *reinterpret_cast<const i32x4*>(lds + at); };
    auto operands = [&](int g) {
#pragma unroll
        for (int u = 0; u < UM; u++) {
            if constexpr (SUB == 1) xa[u] = at128(S::XQ + g * S::XQS + half * BM * 16 + m0 + 512 * u);
            else
#pragma unroll
                for (int h = 0; h < 2; h++)
                    xa2[u][h] = *reinterpret_cast<const int64_t*>(lds + S::XQ + g * S::XQS + h * BM * 16 + m0 + 512 * u + 8 * half);
            // the upper half wave's slots are not used
            xp[u] = __builtin_bit_cast(bf16x8, at128(half ? S::ZERO : S::XP + g * S::XPS + m0 + 512 * u));
        }
#pragma unroll
        for (int u = 0; u < UN; u++) {
            if constexpr (SUB == 1) wb[u] = at128(S::WQ + g * S::WQS + half * BN * 16 + c0 + 512 * u);
            else
#pragma unroll
                for (int h = 0; h < 2; h++)
                    wb2[u][h] = *reinterpret_cast<const int64_t*>(lds + S::WQ + g * S::WQS + h * BN * 16 + c0 + 512 * u + 8 * half);
#pragma unroll
            for (int h = 0; h < SUB; h++)
                wp[h][u] = __builtin_bit_cast(bf16x8, at128(half ? S::ZERO : S::WP + (g * SUB + h) * S::WPS + c0 + 512 * u));
        }
    };
    // - m * (s * sum of codes) is an outer product too: of two groups, or of the
    // two halves of one, in a matrix instruction, straight into the sums
    auto min_operands = [&](int g) {
        const int mine = SUB == 2 ? g * 2 + half : S::PAIR ? g - (1 - half) * WK : g;
        const bool none = SUB == 1 && !S::PAIR && half;
#pragma unroll
        for (int u = 0; u < UM; u++) xm[u] = __builtin_bit_cast(bf16x8, at128(none ? S::ZERO : S::XM + mine * S::XPS + m0 + 512 * u));
#pragma unroll
        for (int u = 0; u < UN; u++) wm[u] = __builtin_bit_cast(bf16x8, at128(none ? S::ZERO : S::WMN + mine * S::WPS + c0 + 512 * u));
    };
    f32x16 ds[2];
    i32x16 p[2];
    // step s of a stage: group s / (units * SUB) of the wave's, then the unit, then the half
    auto scale_step = [&](int s) {
        const int u = s / SUB % S::UNITS, h = s % SUB;
        ds[s % 2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xp[u / UN], wp[h][u % UN], f32x16{}, 0, 0, 0);
    };
    auto code_step = [&](int s) {
        const int u = s / SUB % S::UNITS, h = s % SUB;
        if constexpr (SUB == 1) p[s % 2] = __builtin_amdgcn_mfma_i32_32x32x32_i8(xa[u / UN], wb[u % UN], bias, 0, 0, 0);
        else p[s % 2] = __builtin_amdgcn_mfma_i32_32x32x16_i8(xa2[u / UN][h], wb2[u % UN][h], bias, 0, 0, 0);
    };
    auto add = [&](int s, int from) {
        const int u = s / SUB % S::UNITS;
#pragma unroll
        for (int i = from; i < from + 8; i++)
            acc[u / UN][u % UN][i] =
                __builtin_fmaf(__int_as_float(p[s % 2][i]) - INT_BIAS, ds[s % 2][i], acc[u / UN][u % UN][i]);
    };

    load(begin);
    for (int g0 = begin; g0 < end; g0 += G) {
        lds_barrier();
        put_stage(g0);
        load(g0 + G);
        lds_barrier();
        // The matrix instructions of a step are issued before the vector ones
        // of the step before it, so a wave's vector work covers their latency.
        operands(wk);
        scale_step(0);
        code_step(0);
        constexpr int PER = S::UNITS * SUB;
        if (PER == 1 && S::STEPS > 1) operands(wk + WK);
#pragma unroll
        for (int s = 0; s < S::STEPS; s++) {
            const int g = wk + s / PER * WK;
            __builtin_amdgcn_sched_barrier(0);
            if (s + 1 < S::STEPS) scale_step(s + 1);
            __builtin_amdgcn_sched_barrier(0);
            add(s, 0);
            __builtin_amdgcn_sched_barrier(0);
            if (s + 1 < S::STEPS) code_step(s + 1);
            // operands of the next group as soon as the last step of this one is issued
            if ((s + 2) % PER == 0 && s + 2 < S::STEPS) operands(g + (PER == 1 ? 2 * WK : WK));
            __builtin_amdgcn_sched_barrier(0);
            add(s, 8);
            if constexpr (MIN) {
                if (!S::PAIR || s / PER % 2 == 1) {
                    if (s % PER == 0) min_operands(g);
                    if (s % SUB == SUB - 1) {
                        const int u = s / SUB % S::UNITS;
                        acc[u / UN][u % UN] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(xm[u / UN], wm[u % UN], acc[u / UN][u % UN], 0, 0, 0);
                    }
                }
            }
        }
    }
    // place of element i of a unit: row 8 (i / 4) + 4 half + i % 4, column `col`
    if (a.delta && a.splits == 1 && wk == 0)        // all at once, before the first store
#pragma unroll
        for (int u = 0; u < UM * UN * 16; u++) {
            const int64_t t = t0 + (wmr * UM + u / 16 / UN) * 32 + 8 * (u % 16 / 4) + 4 * half + u % 4;
            const int64_t n = n0 + (wn * UN + u / 16 % UN) * 32 + col;
            acc[u / 16 / UN][u / 16 % UN][u % 16] += a.delta[(t < a.t ? t : a.t - 1) * a.n + (n < a.n ? n : a.n - 1)];
        }
    if constexpr (WK > 1) {
        float* join = reinterpret_cast<float*>(lds);
        const int mine = (wmr * WN + wn) * UM * UN * 16;
        __syncthreads();
        if (wk > 0)
#pragma unroll
            for (int u = 0; u < UM * UN * 16; u++)
                join[(wk - 1) * BM * BN + (mine + u) * 64 + lane] = acc[u / 16 / UN][u / 16 % UN][u % 16];
        __syncthreads();
        if (wk > 0) return;
        for (int j = 0; j < WK - 1; j++)
#pragma unroll
            for (int u = 0; u < UM * UN * 16; u++)
                acc[u / 16 / UN][u / 16 % UN][u % 16] += join[j * BM * BN + (mine + u) * 64 + lane];
    }
#pragma unroll
    for (int um = 0; um < UM; um++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int64_t t = t0 + (wmr * UM + um) * 32 + 8 * (i / 4) + 4 * half + i % 4;
            if (t >= a.t) continue;
#pragma unroll
            for (int un = 0; un < UN; un++) {
                const int64_t n = n0 + (wn * UN + un) * 32 + col;
                if (n >= a.n) continue;
                float y = acc[um][un][i];
                if (a.splits > 1) {
                    a.parts[(split * a.t + t) * a.n + n] = y;
                    continue;
                }
                store_value(a, t * a.n + n, y);
            }
        }
}

// The sum of a split product's parts, one after another.
static __global__ __launch_bounds__(256) void k_join(LinearArgs a) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, all = a.t * a.n;
    if (i >= all) return;
    float y = a.parts[i];
    for (int s = 1; s < a.splits; s++) y += a.parts[s * all + i];
    if (a.delta) y += a.delta[i];
    store_value(a, i, y);
}

}  // namespace qsl
