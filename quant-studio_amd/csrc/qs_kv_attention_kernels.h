// The attention kernel (gfx950).
//
// A wave takes 32 slots of one key/value head at a time and up to eight of its
// queries (the head's group of query heads, times the new tokens). Two matrix
// products of 16 x 16 x 32 f16 per 16 slots and block of 32 dimensions:
//
//   scores   D[slot][query] = codes[slot][dim] q[dim][query], one product for a
//            block, so that the slot's step multiplies its sum: S += step D
//   values   acc[dim][query] += codes[dim][slot] P[slot][query], one for 16 of a
//            block's dimensions, with P = p step (the step runs along the sum)
//
// The scores' D has its slots where the values' P wants them (a lane: one query,
// slots 4 g .. 4 g + 3 of both sixteens), so nothing moves between lanes. Codes go to
// f16 without a conversion: their bits are a subnormal number, which a multiplication by a
// power of two takes up; from four-bit ones it takes their offset of 8 as well (left on, it
// would have to come off the sums, and these would cancel).
// P is held to 21 bits or more: a query has two of the 16 columns, one takes f16(P),
// the other f16(P - f16(P)). So that the second does not fall below f16's range, p counts
// 2^s times, a power of two that takes the largest step so far to just below 2^15: what
// is lost is under 2^-24 of the largest P, mostly far under. q is rounded to f16 after
// its row is scaled to 2^14 .. 2^15 in the same way: all of a bf16 or f16 q down to 2^-35
// of the row's largest; an f32 q takes two products, 22 bits.
//
// What bounds it (heads of 128, bf16 queries, four to a head): eight-bit codes their bytes,
// 8 sequences of 32,767 slots 570 MB in 114 us with the join, 5.0 TB/s, of which loads
// alone take 111 (a large copy reaches 5.2 TB/s; matrix units 0.08 of the cycles, vector
// units 0.5); four-bit ones, at half the bytes for as many codes, loads and the vector
// instructions that unpack them and make P, which overlap in part: 16 of 8,191 slots 151 MB
// in 46 us, 3.3 TB/s, loads alone 38. Small calls wait for memory one read after another:
// lengths, pages, codes, then the join, 11 to 12 us of split calls, 5 of one of 17 slots.
#pragma once

#include "qs_kv_attention.h"
#include "qs_launch_kernel.h"
#include "qs_rows.h"
#include "qs_wave.h"

namespace qskv {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float LOG2E = 1.44269504088896341f;

QS_DEV f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
}

// f over the four lanes that hold a query's slots (lane ^ 16, ^ 32), for an f
// whose value does not depend on its operands' order
template <typename F>
QS_DEV uint32_t over_slots(uint32_t v, F&& f) {
    const auto a = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = f(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return f(b[0], b[1]);
}
QS_DEV float max_over_slots(float v) {
    return __uint_as_float(over_slots(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
    }));
}
QS_DEV float sum_over_slots(float v) {
    return __uint_as_float(over_slots(__float_as_uint(v), [](uint32_t a, uint32_t b) {
        return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
    }));
}
// the other column of the lane's query (lane ^ 8)
QS_DEV float other_column(float v) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x128, 0xF, 0xF, true));
}

// N bytes of consecutive codes as words, loaded through a buffer descriptor: a lane's
// offset `at` stays the same for every step, and where the step is lies in scalar
// registers
typedef __amdgpu_buffer_rsrc_t Buffer;
template <int N>
struct Codes {
    uint32_t w[N / 4];
};
template <int N>
QS_DEV void load_piece(uint32_t* o, Buffer p, int at, int from) {
    if constexpr (N == 16) {
        const u32x4 v = __builtin_amdgcn_raw_buffer_load_b128(p, at, from, 0);
#pragma unroll
        for (int j = 0; j < 4; j++) o[j] = v[j];
    } else if constexpr (N == 8) {
        const u32x2 v = __builtin_amdgcn_raw_buffer_load_b64(p, at, from, 0);
        o[0] = v[0], o[1] = v[1];
    } else {
        o[0] = __builtin_amdgcn_raw_buffer_load_b32(p, at, from, 0);
    }
}
template <int N>
QS_DEV void load(Codes<N>& o, Buffer p, int at, int from) {
    constexpr int PIECE = N % 16 == 0 ? 16 : N % 8 == 0 ? 8 : 4;
#pragma unroll
    for (int i = 0; i < N; i += PIECE) load_piece<PIECE>(o.w + i / 4, p, at + i, from);
}

// Codes as f16, two at a time: c 2^-CODE_POWER, exactly, and normal numbers. As they come out
// of the bytes they are subnormal, and the matrix units take a subnormal factor's bits where
// they are: what lies far below 2^-14 is lost in their sums. With subnormal codes averages of
// 131,071 slots were off by 1e-4 of their rms (four bits; 3e-5 with eight), now by 3e-7. One
// packed multiplication a pair takes them up (1 x 131,071 slots of eight bits 60.5 us, 59.3
// without it), for four-bit codes in the instruction that takes their offset off.
QS_DEV uint32_t sign_and_magnitude(uint32_t twice) {        // a byte beside itself in each half
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2_t, twice & 0x807f807fu) * half2_t{(_Float16)0x1p15f, (_Float16)0x1p15f});
}
// the four-bit codes i and i + 4 of a word, less 8
QS_DEV uint32_t four_bits(uint32_t w, int i) {
    const uint32_t two = (i & 2 ? w >> 8 : w) & (i & 1 ? 0x00f000f0u : 0x000f000fu);
    const _Float16 up = i & 1 ? (_Float16)0x1p11f : (_Float16)0x1p15f, eight = (_Float16)-0x1p-6f;
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_fma(__builtin_bit_cast(half2_t, two), half2_t{up, up}, half2_t{eight, eight}));
}

// eight codes of a key's block
template <int BITS, int BLOCKS>
QS_DEV u32x4 key_block(const Codes<BITS * BLOCKS>& c, int b) {
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if constexpr (BITS == 8)
            o[i] = sign_and_magnitude(__builtin_amdgcn_perm(0u, c.w[2 * b + (i >> 1)], i & 1 ? 0x03030202u : 0x01010000u));
        else o[i] = four_bits(c.w[b], i);
    }
    return o;
}
// code n of the slots 2 i and 2 i + 1 of four
template <int BITS, int BLOCKS>
QS_DEV uint32_t value_pair(const Codes<BITS * BLOCKS>& c, int i, int n) {
    // `run` bytes of each slot one after another: bytes `x` and `y` have the code
    constexpr int RUN = BITS * BLOCKS / 4;
    const int x = 2 * i * RUN + n * BITS / 8, y = x + RUN;
    if constexpr (BITS == 8) {
        return sign_and_magnitude(
            __builtin_amdgcn_perm(c.w[y >> 2], c.w[x >> 2], (x & 3) * 0x00000101u + (y & 3) * 0x01010000u + 0x04040000u));
    } else {
        // the half words that have it; their codes 0 .. 3 are those from n & ~3 on
        const uint32_t hx = x & 2 ? 0x0302u : 0x0100u, hy = y & 2 ? 0x07060000u : 0x05040000u;
        return four_bits(__builtin_amdgcn_perm(c.w[y >> 2], c.w[x >> 2], hx | hy), n & 3);
    }
}

// Two P as the lane's column takes them: f16(P), cut off, in the first (second = 0); in
// the second (0xffffe000, what of an f32 an f16 has) what that leaves of it, cut off as
// well, which one instruction does for both, or to nearest for f32 results.
template <bool NEAREST>
QS_DEV uint32_t two_halves(float x, float y, uint32_t second) {
    const auto cut = [](float v, uint32_t mask) { return __uint_as_float(__float_as_uint(v) & mask); };
    if constexpr (NEAREST) {
        const float u = cut(x, 0xffffe000u), v = cut(y, 0xffffe000u);
        return __builtin_bit_cast(uint32_t, half2_t{(_Float16)(second ? x - u : u), (_Float16)(second ? y - v : v)});
    }
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x - cut(x, second), y - cut(y, second)));
}

// the queries of a wave, as the scores' products take them
template <int BLOCKS, bool WIDE>
struct Queries {
    u32x4 q[BLOCKS], lo[WIDE ? BLOCKS : 1];
    float scale;                            // of the scores, beside 2^up
    int up;
    int first, last;                        // slots that the lane's query sees: first .. last - 1
};

// as they are in memory, eight of every block to a lane
template <int BLOCKS, bool WIDE>
struct RawQueries {
    qsr::Eight<WIDE ? qs::SRC_F32 : qs::SRC_BF16> b[BLOCKS];
};
template <int BLOCKS, bool WIDE>
QS_DEV void load_queries(const AttentionArgs& a, int seq, int head, int first, RawQueries<BLOCKS, WIDE>& o) {
    const int lane = threadIdx.x & 63, g = lane >> 4, column = first + (lane & 7);
    const bool live = column < a.group * a.fresh;
    const int token = live ? column / a.group : 0, mine = live ? column - token * a.group : 0;
    const int64_t at = ((int64_t)seq * a.fresh + token) * a.q_stride + (int64_t)(head * a.group + mine) * 32 * BLOCKS;
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) qsr::load8<WIDE ? qs::SRC_F32 : qs::SRC_BF16>(a.q, at + 32 * b + 8 * g, o.b[b]);
}
template <int BLOCKS, bool WIDE>
QS_DEV void prepare_queries(const AttentionArgs& a, int first, int length, const RawQueries<BLOCKS, WIDE>& raw,
                            Queries<BLOCKS, WIDE>& o) {
    const int lane = threadIdx.x & 63, column = first + (lane & 7);
    const bool live = column < a.group * a.fresh, bf16 = a.type == QS_SRC_BF16;
    const int token = live ? column / a.group : 0;
    float x[BLOCKS][8];
    float top = 0.0f;
#pragma unroll
    for (int b = 0; b < BLOCKS; b++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if constexpr (WIDE) x[b][i] = qsr::value8<qs::SRC_F32>(raw.b[b], i);
            else {
                const uint32_t h = raw.b[b].w[0][i >> 1] >> (16 * (i & 1));
                x[b][i] = bf16 ? __uint_as_float(h << 16) : half_of(h);
            }
            x[b][i] = live ? x[b][i] : 0.0f;
            top = fmaxf(top, fabsf(x[b][i]));
        }
    top = max_over_slots(top);
    const bool scaled = top > 0.0f && top < __builtin_inff();
    const int e = scaled ? 15 - __builtin_amdgcn_frexp_expf(top) : 0;     // top 2^e in 2^14 .. 2^15
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            half2_t h, l;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                const float v = __builtin_ldexpf(x[b][2 * i + j], e);
                h[j] = (_Float16)v;
                if constexpr (WIDE) l[j] = (_Float16)(v - (float)h[j]);
            }
            o.q[b][i] = __builtin_bit_cast(uint32_t, h);
            if constexpr (WIDE) o.lo[b][i] = __builtin_bit_cast(uint32_t, l);
        }
    }
    o.scale = a.scale * LOG2E;
    o.up = CODE_POWER - e;
    o.last = length - a.fresh + 1 + token;
    o.first = a.window > 0 && o.last > a.window ? o.last - a.window : 0;
}

// what a wave has summed up of its slots
template <int BLOCKS>
struct Sums {
    f32x4 acc[BLOCKS][2];               // dims 32 block + 8 g + 2 r + e at [block][e][r]
    float top, total;                   // running maximum, sum of p; p and P count 2^power times
    int power;
    uint32_t step;                      // the bits of all steps so far, or'ed
};
template <int BLOCKS>
QS_DEV void clear(Sums<BLOCKS>& o) {
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) o.acc[b][0] = o.acc[b][1] = f32x4{0, 0, 0, 0};
    o.top = -__builtin_inff();
    o.total = 0.0f;
    o.power = 0;
    o.step = 0;
}

// What the queries of a wave see: any of them slots first .. last - 1 at most, all of
// them slots all_first .. all_last - 1.
struct Span {
    int first, last, all_first, all_last;
};
QS_DEV Span span_of(const AttentionArgs& a, int first, int columns, int length) {
    const int high = min(a.group * a.fresh, first + columns) - 1;
    Span s;
    s.last = length - a.fresh + 1 + high / a.group;
    s.all_last = length - a.fresh + 1 + first / a.group;
    s.first = a.window > 0 && s.all_last > a.window ? s.all_last - a.window : 0;
    s.all_first = a.window > 0 && s.last > a.window ? s.last - a.window : 0;
    return s;
}

// The calls' tables and lengths: nothing writes them meanwhile, so they may come
// through the scalar cache, and what they give is the same for a wave.
typedef const __attribute__((address_space(4))) int32_t* Ints;
QS_DEV Ints constant(const int32_t* p) { return (Ints)(uintptr_t)p; }

// What a lane loads of a step's 32 slots, both sixteens of which lie in one page each:
// of each sixteen a quarter of key m's codes, and of the slots 4 g .. 4 g + 3 the values'
// codes of two dims of every block. The steps (of quantisation) are wanted by sixteen
// lanes each: one loads them, and LDS gives them to all.
template <int K_BITS, int V_BITS, int BLOCKS>
struct Tile {
    static constexpr int KROW = row_bytes(K_BITS, BLOCKS), VROW = row_bytes(V_BITS, BLOCKS);
    Codes<KROW / 4> keys[2];
    Codes<VROW / 4> values[2];          // of one slot after another
    Codes<2 * BLOCKS> steps;
};
// where they are: the same for the whole wave
struct Place {
    const uint8_t *head0, *head1;   // of the sixteens' pages
    int slot0, slot1;               // in them
    int held;                       // bits 0 and 1: their pages are in the cache
};
// the pages of a step, as the table has them
struct Pages {
    int first, second;
};
QS_DEV Pages pages_of(const AttentionArgs& a, Ints table, int start) {
    const int first = start >> a.c.shift, second = (start + 16) >> a.c.shift;
    return {table[first], table[second < a.pages_each ? second : first]};
}
QS_DEV Place place_of(const AttentionArgs& a, const Pages& pages, int head, int start) {
    Place o;
    const int second = (start + 16) >> a.c.shift;
    const bool held0 = (unsigned)pages.first < (unsigned)a.c.pages;
    const bool held1 = (unsigned)pages.second < (unsigned)a.c.pages && second < a.pages_each;
    // where one is not, page 0, whose slots are not used
    o.head0 = head_of(a.c, held0 ? pages.first : 0, head);
    o.head1 = head_of(a.c, held1 ? pages.second : 0, head);
    o.slot0 = start & (a.c.page - 1);
    o.slot1 = (start + 16) & (a.c.page - 1);
    o.held = (held0 ? 1 : 0) | (held1 ? 2 : 0);
    return o;
}
template <int K_BITS, int V_BITS, int BLOCKS>
QS_DEV Buffer buffer_of(const AttentionArgs& a, const uint8_t* head) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(head), 0, a.c.page * slot_bytes(K_BITS, V_BITS, BLOCKS), 0x00027000);
}
template <int K_BITS, int V_BITS, int BLOCKS>
QS_DEV void load_keys(const AttentionArgs& a, const Place& at, Tile<K_BITS, V_BITS, BLOCKS>& t) {
    typedef Tile<K_BITS, V_BITS, BLOCKS> T;
    const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
    constexpr int RUN = T::KROW / 4, PIECES = RUN / 16 * 16;
#pragma unroll
    for (int s = 0; s < 2; s++) {
        const Buffer p = buffer_of<K_BITS, V_BITS, BLOCKS>(a, s ? at.head1 : at.head0);
        const int from = (s ? at.slot1 : at.slot0) * T::KROW;
#pragma unroll
        for (int i = 0; i < PIECES; i += 16) load_piece<16>(t.keys[s].w + i / 4, p, m * T::KROW + 16 * g + 4 * i, from);
        if constexpr (RUN > PIECES) load_piece<8>(t.keys[s].w + PIECES / 4, p, m * T::KROW + 8 * g + 4 * PIECES, from);
    }
    // half a wave takes a sixteen's
    const int codes = a.c.page * (T::KROW + T::VROW);
    const uint8_t* p = lane < 32 ? at.head0 + (codes + at.slot0 * 4 * BLOCKS) : at.head1 + (codes + at.slot1 * 4 * BLOCKS);
    __builtin_memcpy(t.steps.w, __builtin_assume_aligned(p + (lane & 31) * 2 * BLOCKS, 4), 2 * BLOCKS);
}
template <int K_BITS, int V_BITS, int BLOCKS>
QS_DEV void load_values(const AttentionArgs& a, const Place& at, Tile<K_BITS, V_BITS, BLOCKS>& t) {
    typedef Tile<K_BITS, V_BITS, BLOCKS> T;
    const int lane = threadIdx.x & 63, g = lane >> 4, m = lane & 15;
#pragma unroll
    for (int s = 0; s < 2; s++)
        load(t.values[s], buffer_of<K_BITS, V_BITS, BLOCKS>(a, s ? at.head1 : at.head0), 4 * T::VROW * g + m * (T::VROW / 4),
             a.c.page * T::KROW + (s ? at.slot1 : at.slot0) * T::VROW);
}

// One step: the slots start .. start + 31, in `t`. The next step's keys and values
// (at `next`) are loaded into the registers of this one's as soon as these are done
// with, and arrive while the other half is computed.
// edge: some query does not see all of the slots; to it they count for nothing,
// whatever they hold, since a lane's scores and steps are its query's own copies.
template <bool WIDE, int K_BITS, int V_BITS, int BLOCKS, int SETS>
QS_DEV void attend(const AttentionArgs& a, int start, bool edge, int held, const Place& next,
                   const Queries<BLOCKS, WIDE> (&q)[SETS], uint32_t* lds, Tile<K_BITS, V_BITS, BLOCKS>& t, Sums<BLOCKS> (&sums)[SETS]) {
    const int lane = threadIdx.x & 63, g = lane >> 4;
    // steps of four slots, and one of them
    typedef Codes<8 * BLOCKS> Steps4;
    const auto steps_from = [&](int s, bool value, Steps4& o) {
        const uint32_t* p = lds + (s * 16 + 4 * g) * BLOCKS + (value ? 2 * BLOCKS : 0);
#pragma unroll
        for (int i = 0; i < 2 * BLOCKS; i += 4) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(p + i);
#pragma unroll
            for (int j = 0; j < 4; j++) o.w[i + j] = v[j];
        }
    };
    const auto step_of = [](const Steps4& c, int r, int b) {
        const int n = r * BLOCKS + b;
        return half_of(c.w[n >> 1] >> (16 * (n & 1)));
    };
    // lane after lane they are the two sixteens' steps as they lie in their pages
#pragma unroll
    for (int i = 0; i < BLOCKS / 2; i++) lds[lane * (BLOCKS / 2) + i] = t.steps.w[i];
    qs::wave_sync<true>();
    // scores, in powers of two
    float x[SETS][2][4];
#pragma unroll
    for (int s = 0; s < 2; s++) {
#pragma unroll
        for (int n = 0; n < 4 * SETS; n++) x[n >> 2][s][n & 3] = 0.0f;
        Steps4 ks;
        steps_from(s, false, ks);
#pragma unroll
        for (int b = 0; b < BLOCKS; b++) {
            const u32x4 k = key_block<K_BITS, BLOCKS>(t.keys[s], b);
#pragma unroll
            for (int n = 0; n < SETS; n++) {
                f32x4 d = mfma(k, q[n].q[b], f32x4{0, 0, 0, 0});
                if constexpr (WIDE) d = mfma(k, q[n].lo[b], d);
#pragma unroll
                for (int r = 0; r < 4; r++) x[n][s][r] = __builtin_fmaf(d[r], step_of(ks, r, b), x[n][s][r]);
            }
        }
#pragma unroll
        for (int n = 0; n < SETS; n++)
#pragma unroll
            for (int r = 0; r < 4; r++) x[n][s][r] = __builtin_ldexpf(x[n][s][r] * q[n].scale, q[n].up);
    }
    __builtin_amdgcn_sched_barrier(0);      // loads that move up would need registers of their own
    load_keys(a, next, t);
    Steps4 vs[SETS][2];
#pragma unroll
    for (int n = 0; n < SETS; n++)
#pragma unroll
        for (int s = 0; s < 2; s++) {
            if (n == 0) steps_from(s, true, vs[0][s]);
            else vs[n][s] = vs[0][s];
        }
    if (edge) {
#pragma unroll
        for (int n = 0; n < 8 * SETS; n++) {
            const int set = n >> 3, s = n >> 2 & 1, r = n & 3, p = start + 16 * s + 4 * g + r;
            if (!((held >> s & 1) && p >= q[set].first && p < q[set].last)) {
                x[set][s][r] = -__builtin_inff();
#pragma unroll
                for (int i = 0; i < BLOCKS / 2; i++) vs[set][s].w[r * (BLOCKS / 2) + i] = 0;
            }
        }
    }
    float p[SETS][8];
#pragma unroll
    for (int n = 0; n < SETS; n++) {
        // the running maximum and the power of two
        float top = sums[n].top;
        uint32_t steps = 0;
#pragma unroll
        for (int s = 0; s < 2; s++) {
#pragma unroll
            for (int r = 0; r < 4; r++) top = fmaxf(top, x[n][s][r]);
#pragma unroll
            for (int i = 0; i < 2 * BLOCKS; i++) steps |= vs[n][s].w[i];
        }
        top = max_over_slots(top);
        steps = over_slots(steps, [](uint32_t u, uint32_t v) { return u | v; });
        sums[n].step |= steps | steps >> 16;
        // 2^s takes every step below 2^15. Or'ed exponents bound them all, and are over the
        // largest by 15 at most, by 7 for steps below 2, which takes that much off 39 bits; a
        // subnormal step, or none, counts as 2^-14.
        const int exponent = (int)(sums[n].step >> 10 & 31), s = 29 - (exponent > 1 ? exponent : 1);
        const float base = top > -__builtin_inff() ? top : 0.0f;
        // 0 where nothing was seen yet
        const float shrink = __builtin_ldexpf(__builtin_amdgcn_exp2f(sums[n].top - base), s - sums[n].power);
        sums[n].top = top;
        sums[n].power = s;
        // 2^s multiplies p: in the exponent it would take bits of what is there
        const float power = __uint_as_float((uint32_t)(127 + s) << 23);
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            p[n][i] = __builtin_amdgcn_exp2f(x[n][i >> 2][i & 3] - base) * power;
            total += p[n][i];
        }
        sums[n].total = __builtin_fmaf(sums[n].total, shrink, total);
        if (__any(shrink != 1.0f)) {
#pragma unroll
            for (int b = 0; b < BLOCKS; b++)
#pragma unroll
                for (int e = 0; e < 2; e++)
#pragma unroll
                    for (int r = 0; r < 4; r++) sums[n].acc[b][e][r] *= shrink;
        }
    }
    const uint32_t second = lane & 8 ? 0xffffe000u : 0u;
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) {
        u32x4 w[SETS];
#pragma unroll
        for (int n = 0; n < 4 * SETS; n++) {
            const int set = n >> 2, i = 2 * (n & 3);
            const Steps4& d = vs[set][i >> 2];
            // + 0 makes it one instruction that takes the step as f16
            w[set][n & 3] = two_halves<WIDE>(__builtin_fmaf(p[set][i], step_of(d, i & 3, b), 0.0f),
                                             __builtin_fmaf(p[set][i + 1], step_of(d, (i & 3) + 1, b), 0.0f), second);
        }
#pragma unroll
        for (int e = 0; e < 2; e++) {
            u32x4 c;
#pragma unroll
            for (int i = 0; i < 4; i++) c[i] = value_pair<V_BITS, BLOCKS>(t.values[i >> 1], i & 1, 2 * b + e);
#pragma unroll
            for (int n = 0; n < SETS; n++) sums[n].acc[b][e] = mfma(c, w[n], sums[n].acc[b][e]);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    load_values(a, next, t);
}

// The wave's sums as one: the four lanes of a query's slots, and its two columns;
// p counts 2^power times.
template <int BLOCKS>
QS_DEV void finish(Sums<BLOCKS>& o) {
    const float once = __builtin_ldexpf(1.0f, -o.power);
    o.total = sum_over_slots(o.total) * once;
#pragma unroll
    for (int b = 0; b < BLOCKS; b++)
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                o.acc[b][e][r] = (o.acc[b][e][r] + other_column(o.acc[b][e][r])) * once;
}

QS_DEV int cut_length(const AttentionArgs& a, int n) {
    const int most = a.pages_each << a.c.shift;
    return n < 0 ? 0 : n > most ? most : n;
}
QS_DEV int length_of(const AttentionArgs& a, int seq) { return cut_length(a, constant(a.lengths)[seq]); }
// Steps of a sequence for any of its queries, from step `begin` on: at least one,
// so that queries that see nothing get their zeros.
struct Steps {
    int begin, count;
};
QS_DEV Steps steps_of(const AttentionArgs& a, int length) {
    const int lowest = length - a.fresh + 1;
    Steps s;
    s.begin = (a.window > 0 && lowest > a.window ? lowest - a.window : 0) / TILE;
    s.count = (length + TILE - 1) / TILE - s.begin;
    s.count = s.count < 1 ? 1 : s.count;
    return s;
}

// The call's steps in a row (by sequence, head, tile of columns, then along the
// sequence), dealt to the workgroups in equal runs: `total` of them, `each` to a
// workgroup, this one's first one in sequence `seq`, whose own begin at `base` of one
// head's. A head's steps count `opening` more than they are, which comes first: what
// beginning with another one takes. The lengths are on the device, so every workgroup
// adds them up.
struct Deal {
    int64_t total, each;
    int seq, base;
};
QS_DEV int64_t quotient(int64_t a, int64_t b) {     // of numbers from 0 on
    return (a | b) >> 32 ? a / b : (int64_t)((uint32_t)a / (uint32_t)b);
}
QS_DEV int units_of(const AttentionArgs& a, int opening, int seq) { return opening + steps_of(a, length_of(a, seq)).count; }
QS_DEV Deal deal(const AttentionArgs& a, int groups, int waves, int opening, int heads) {
    // every wave by itself: a lane adds up a run of sequences, and these sums are added along the lanes
    const int lane = threadIdx.x & 63, each_lane = (a.batch + 63) >> 6;
    int sum = 0;
#pragma unroll 4
    for (int i = 0; i < each_lane; i++) {
        const int seq = lane * each_lane + i;
        sum += seq < a.batch ? units_of(a, opening, seq) : 0;
    }
    const int scan = qs::wave_incl_scan(sum);
    Deal d;
    d.total = (int64_t)__builtin_amdgcn_readlane(scan, 63) * heads;
    d.each = quotient(d.total + groups - 1, groups);
    d.each = d.each < waves ? waves : d.each;
    const int64_t begin = blockIdx.x * d.each;
    if (begin >= d.total) return d;
    const int at = (int)quotient(begin, heads);
    const int run = __builtin_ctzll(__ballot(at < scan));       // the lane whose run it is in
    d.seq = run * each_lane;
    d.base = __builtin_amdgcn_readlane(scan - sum, run);
    for (int n = units_of(a, opening, d.seq); at >= d.base + n && d.seq + 1 < a.batch; n = units_of(a, opening, d.seq)) {
        d.base += n;
        d.seq++;
    }
    return d;
}

// A workgroup of four waves or one, which take a segment's steps in turn (a segment:
// what the workgroup has of one head's and column tile's steps of a sequence) and join
// their sums through LDS. A segment that is a whole one is written as the result,
// else as a part that k_kv_join takes.
// SHARE: its segment is the steps that it has of the split's `share`, dealt to their
// waves in turn.
template <int K_BITS, int V_BITS, int BLOCKS, bool WIDE, int SETS, int WAVES, bool SHARE>
__global__ __launch_bounds__(64 * WAVES) __attribute__((amdgpu_waves_per_eu(resident(BLOCKS, 8 * SETS, WIDE))))
void k_kv_attention(AttentionArgs a, Split split) {
    constexpr int COLUMNS = 8 * SETS, D = 32 * BLOCKS, ROW = D + 4;     // 4: the eight columns' words in other banks
    constexpr int OPENING = qskv::OPENING * WAVES;
    __shared__ __attribute__((aligned(16))) float acc[WAVES][COLUMNS][ROW];
    __shared__ float2 stats[WAVES][COLUMNS];
    __shared__ __attribute__((aligned(16))) uint32_t steps_lds[WAVES][TILE * BLOCKS];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, g = lane >> 4;
    const int tiles = (a.group * a.fresh + COLUMNS - 1) / COLUMNS, heads = a.c.heads * tiles;
    int64_t at = 0, end = 1, each = 0;
    int seq, base = 0, which = -1, from = 0;        // which: head and column tile
    int4 going{0, 0, 0, -1};
    if constexpr (SHARE) {
        const int segment = (int)blockIdx.x / split.share;
        seq = segment / heads;
        which = segment - seq * heads;
        from = (int)blockIdx.x - segment * split.share;     // which part
    } else {
        const Deal d = deal(a, split.groups, WAVES, OPENING, heads);
        each = d.each;
        at = blockIdx.x * d.each;
        end = at + d.each < d.total ? at + d.each : d.total;
        seq = d.seq;
        base = d.base;
    }
    const int64_t begin = at;
    while (at < end && seq < a.batch) {
        int length = constant(a.lengths)[seq];
        Steps steps{};
        int to = 0;                                 // from .. to - 1 of them
        if constexpr (!SHARE) {
            length = cut_length(a, length);
            steps = steps_of(a, length);
            if (which < 0) {
                const int64_t rel = at - (int64_t)base * heads;
                which = (int)quotient(rel, OPENING + steps.count);
                at -= rel - (int64_t)which * (OPENING + steps.count);
                from = (int)(begin - at) - OPENING;
            }
            // `at`: where the head's begin, `from` below 0 where they do in this workgroup
            to = steps.count < end - at - OPENING ? steps.count : (int)(end - at) - OPENING;
            from = from < 0 ? 0 : from;
            if (to <= from) break;                  // it ends before they do
        }
        const int head = which / tiles, first = (which - head * tiles) * COLUMNS;    // its first column
        RawQueries<BLOCKS, WIDE> raw[SETS];
        Sums<BLOCKS> sums[SETS];
#pragma unroll
        for (int n = 0; n < SETS; n++) {
            load_queries(a, seq, head, first + 8 * n, raw[n]);
            clear(sums[n]);
        }
        const Ints table = constant(a.tables + seq * a.table_stride);
        // The wave's steps i, i + stride, ... before `stop`, counted from the sequence's
        // start, of those that this column tile's queries see. The first one's codes are
        // asked for as soon as it is known which it is: a part's first step depends on
        // the length only with a window.
        constexpr bool RUN = !SHARE;
        const int stride = RUN ? WAVES : split.share * WAVES, most = ((a.pages_each << a.c.shift) + TILE - 1) / TILE;
        const bool early = SHARE && a.window == 0;
        Span span{};
        int i = RUN ? steps.begin + from + wave : from * WAVES + wave, stop = RUN ? steps.begin + to : most;
        const auto see = [&] {
            if (SHARE) length = cut_length(a, length);
            span = span_of(a, first, COLUMNS, length);
            const int low = span.first / TILE, high = (span.last + TILE - 1) / TILE;
            stop = high < stop ? high : stop;
            if (!early) i = RUN ? (low > steps.begin + from ? low + wave : i) : low + i;
        };
        if (!early) see();
        Place place;
        Pages ahead;
        Tile<K_BITS, V_BITS, BLOCKS> t;
        const bool any = i < stop;
        if (any) {
            place = place_of(a, pages_of(a, table, i * TILE), head, i * TILE);
            ahead = pages_of(a, table, (i + stride < stop ? i + stride : i) * TILE);
            load_keys(a, place, t);
            load_values(a, place, t);
        }
        if (early) see();
        if (any && i < stop) {
            // The pages of a step are asked for two steps ahead, its codes one ahead; after
            // the last step it is that step's again, whose codes are in the caches.
            const int final = i + (stop - 1 - i) / stride * stride;
            const auto start_of = [&](int n) { return (n < final ? n : final) * TILE; };
            Queries<BLOCKS, WIDE> q[SETS];
#pragma unroll
            for (int n = 0; n < SETS; n++) prepare_queries(a, first + 8 * n, length, raw[n], q[n]);
            for (; i < stop; i += stride) {
                const int start = i * TILE, held = place.held;
                place = place_of(a, ahead, head, start_of(i + stride));
                ahead = pages_of(a, table, start_of(i + 2 * stride));
                attend(a, start, start < span.all_first || start + TILE > span.all_last || held != 3, held, place, q, steps_lds[wave], t, sums);
            }
        }
#pragma unroll
        for (int n = 0; n < SETS; n++) {
            finish(sums[n]);
            if (lane & 8) continue;
            const int column = 8 * n + (lane & 7);
#pragma unroll
            for (int b = 0; b < BLOCKS; b++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const f32x4(&v)[2] = sums[n].acc[b];
                    *reinterpret_cast<f32x4*>(&acc[wave][column][32 * b + 8 * g + 4 * h]) =
                        f32x4{v[0][2 * h], v[1][2 * h], v[0][2 * h + 1], v[1][2 * h + 1]};
                }
            if (g == 0) stats[wave][column] = float2{sums[n].top, sums[n].total};
        }
        __syncthreads();
        const bool whole = SHARE ? split.share == 1 : from == 0 && to == steps.count;
        // thread: two dims of every 64 of a column, or of one after another
        const int sub = threadIdx.x & 31;
#pragma unroll
        for (int column = threadIdx.x >> 5; column < COLUMNS; column += 2 * WAVES) {
            float ref = -__builtin_inff(), total = 0.0f, part[WAVES];
#pragma unroll
            for (int w = 0; w < WAVES; w++) ref = fmaxf(ref, stats[w][column].x);
#pragma unroll
            for (int w = 0; w < WAVES; w++) {
                const float2 s = stats[w][column];
                part[w] = s.x > -__builtin_inff() ? __builtin_amdgcn_exp2f(s.x - ref) : s.y;    // s.y: 0, or NaN
                total = __builtin_fmaf(s.y, part[w], total);
            }
            const int64_t row = row_of(a, seq, head, first + column);
            const int64_t slot = ((int64_t)blockIdx.x * 2 + (from == 0)) * COLUMNS + column;
            const float inverse = total != 0.0f ? ONCE / total : 0.0f;    // 0: it sees nothing
#pragma unroll
            for (int i = 0; i < BLOCKS / 2; i++) {
                float2 v{0, 0};
#pragma unroll
                for (int w = 0; w < WAVES; w++) {
                    const float2 u = *reinterpret_cast<const float2*>(&acc[w][column][64 * i + 2 * sub]);
                    v.x = __builtin_fmaf(u.x, part[w], v.x);
                    v.y = __builtin_fmaf(u.y, part[w], v.y);
                }
                if (!whole) *reinterpret_cast<float2*>(split.parts + slot * D + 64 * i + 2 * sub) = v;
                else if (row >= 0) store_two(a, row + 64 * i + 2 * sub, v.x * inverse, v.y * inverse);
            }
            if (!whole && sub == 0) split.stats[slot] = float2{ref, total};
        }
        __syncthreads();
        if constexpr (SHARE) return;
        if (from == 0) {
            if (!whole) going = int4{seq, which, (int)blockIdx.x, (int)quotient(at + OPENING + steps.count - 1, each)};
            if (split.listed && threadIdx.x == 0) split.segments[seq * heads + which] = whole ? int4{0, 0, 0, -1} : going;
        }
        at += OPENING + steps.count;
        from = 0;
        if (++which == heads) {         // only the last segment ends before its steps do
            which = 0;
            seq++;
        }
    }
    if (!split.listed && threadIdx.x == 0) split.segments[blockIdx.x] = going;
}

template <int K_BITS, int V_BITS, int BLOCKS, bool WIDE, int SETS>
hipError_t launch_sets(const AttentionArgs& a, const Split& split, hipStream_t st) {
    const auto kernel = split.waves == 4 ? (split.share ? k_kv_attention<K_BITS, V_BITS, BLOCKS, WIDE, SETS, 4, true>
                                                        : k_kv_attention<K_BITS, V_BITS, BLOCKS, WIDE, SETS, 4, false>)
                                         : (split.share ? k_kv_attention<K_BITS, V_BITS, BLOCKS, WIDE, SETS, 1, true>
                                                        : k_kv_attention<K_BITS, V_BITS, BLOCKS, WIDE, SETS, 1, false>);
    const hipError_t e = qs_host::launch_kernel(kernel, dim3((unsigned)split.groups), dim3((unsigned)(64 * split.waves)), 0, st, a, split);
    return e != hipSuccess || split.share == 1 ? e : launch_join(a, split, st);
}
template <int K_BITS, int V_BITS, int BLOCKS>
hipError_t launch_blocks(const AttentionArgs& a, const Split& split, hipStream_t st) {
    if (a.type == QS_SRC_F32) return launch_sets<K_BITS, V_BITS, BLOCKS, true, 1>(a, split, st);
    if constexpr (BLOCKS <= 4)
        if (columns_of(a) == 16) return launch_sets<K_BITS, V_BITS, BLOCKS, false, 2>(a, split, st);
    return launch_sets<K_BITS, V_BITS, BLOCKS, false, 1>(a, split, st);
}

template <int K_BITS, int V_BITS>
hipError_t launch_attention(const AttentionArgs& a, const Split& split, hipStream_t st) {
    switch (a.c.blocks) {
        case 2: return launch_blocks<K_BITS, V_BITS, 2>(a, split, st);
        case 4: return launch_blocks<K_BITS, V_BITS, 4>(a, split, st);
        case 6: return launch_blocks<K_BITS, V_BITS, 6>(a, split, st);
        default: return launch_blocks<K_BITS, V_BITS, 8>(a, split, st);
    }
}

}  // namespace qskv
