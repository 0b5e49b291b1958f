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
// P is held to 21 bits or more beside the largest of its block of 32 dimensions: a query has
// two of the 16 columns, one takes f16(P), the other f16(P - f16(P)). So that neither leaves
// f16's range, P count by a power of two that follows the largest of them (Sums). q is
// rounded to f16 after its row is scaled to 2^14 .. 2^15 likewise: all of a bf16 or f16 q
// down to 2^-35 of the row's largest; an f32 q takes two products, 22 bits.
//
// What bounds it (heads of 128, bf16 queries, four to a head): eight-bit codes their bytes,
// 8 sequences of 32,767 slots 570 MB in 116 us with the join, 4.9 TB/s, of which loads
// alone take 111 (a large copy reaches 5.2 TB/s; matrix units 0.07 of the cycles, vector
// units 0.54); four-bit ones, at half the bytes for as many codes, loads and the vector
// instructions that unpack them and make P (0.7), which overlap in part: 16 of 8,191 slots
// 151 MB in 48 us, 3.1 TB/s, loads alone 38. Small calls wait for memory one read after
// another: lengths, pages, codes, then the join, 12 to 13 us of split calls, 6 of one of 17
// slots.
#pragma once

#include "qs_kv_attention.h"
#include "qs_launch_kernel.h"
#include "qs_rows.h"
#include "qs_wave.h"

namespace qskv {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
typedef short i16x2 __attribute__((ext_vector_type(2)));

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

// Two P as the lane's column takes them: f16(P) in the first (second = 0); in the second (1)
// what that leaves of it, in f16 as well.
QS_DEV uint32_t two_halves(float x, float y, float second) {
    // Both as f32 hold them: the compiler would form the product that x is and its f16 in one
    // instruction, which rounds once, and where x lies half way the two columns would differ.
    asm("" : "+v"(x), "+v"(y));
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const half2_t h = __builtin_convertvector(f32x2{x, y}, half2_t);
    const half2_t v{(_Float16)__builtin_fmaf((float)h[0], -second, x), (_Float16)__builtin_fmaf((float)h[1], -second, y)};
    return __builtin_bit_cast(uint32_t, v);
}

// the queries of a wave, as the scores' products take them
template <int BLOCKS, bool WIDE>
struct Queries {
    u32x4 q[BLOCKS], lo[WIDE ? BLOCKS : 1];
    float scale;                            // of the scores, beside 2^up
    int up;
    int first, last;                        // slots that the lane's query sees: first .. last - 1
};

// A column without a query takes the last one. No lane branches off for it: where lanes join
// again the compiler (ROCm 7.2's) has saved registers for the joined ones alone.
QS_DEV int column_of(const AttentionArgs& a, int column) { return min(column, a.group * a.fresh - 1); }

// as they are in memory, eight of every block to a lane
template <int BLOCKS, bool WIDE>
struct RawQueries {
    qsr::Eight<WIDE ? qs::SRC_F32 : qs::SRC_BF16> b[BLOCKS];
};
template <int BLOCKS, bool WIDE>
QS_DEV void load_queries(const AttentionArgs& a, int seq, int head, int first, RawQueries<BLOCKS, WIDE>& o) {
    const int lane = threadIdx.x & 63, g = lane >> 4, column = column_of(a, first + (lane & 7));
    const int token = column / a.group, mine = column - token * a.group;
    const int64_t at = ((int64_t)seq * a.fresh + token) * a.q_stride + (int64_t)(head * a.group + mine) * 32 * BLOCKS;
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) qsr::load8<WIDE ? qs::SRC_F32 : qs::SRC_BF16>(a.q, at + 32 * b + 8 * g, o.b[b]);
}
template <int BLOCKS, bool WIDE>
QS_DEV void prepare_queries(const AttentionArgs& a, int first, int length, const RawQueries<BLOCKS, WIDE>& raw,
                            Queries<BLOCKS, WIDE>& o) {
    const int lane = threadIdx.x & 63, column = first + (lane & 7), token = column_of(a, column) / a.group;
    const bool live = column < a.group * a.fresh, bf16 = a.type == QS_SRC_BF16;
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
    // a mantissa and a power of two: scale log2(e) itself may pass f32's range where no score does
    o.scale = __builtin_amdgcn_frexp_mantf(a.scale) * LOG2E;
    o.up = CODE_POWER - e + __builtin_amdgcn_frexp_expf(a.scale);
    o.last = length - a.fresh + 1 + token;
    o.first = a.window > 0 && o.last > a.window ? o.last - a.window : 0;
}

// What a wave has summed up of its slots. P count by 2^power, which follows the largest |P| of
// the query so far: 2^(TARGET - 1) or more as it counts when the power is chosen, by up to
// 2^SLACK less while the running maximum rises, and never 2^LIMIT. A block whose own largest
// is then below 2^(FLOOR - 1), where the second of two f16 would come to lose bits of it,
// counts by a power of its own, 2^MOST times the others' at most. (One power for the largest step seen, whatever its p and its
// block, left blocks of small values and those beside large ones of no weight 6 to 17 bits:
// errors up to 1e-2.) The running maximum is a whole number, so that what it takes off is a
// power of two as well.
//
// What a wave pays: the powers are chosen on its first step of a segment, 0.4 us (1 of 17
// slots 5.4 to 5.8 us, 61 ragged ones 30.2 to 32.2, 16 of 8,191 with four bits 46.3 to 47.6),
// and seldom again: a step asks for it where the maximum rose by more than is left of the
// slack, or a value's step could take a P to 2^LIMIT. Looking at every P of every step took
// 16 of 8,191 slots to 52 us, choosing anew wherever the maximum rises to 55. Where a block has
// a power of its own, values a thousandth of the others', those take 47.0 us for 42.1; a block
// of zeros costs nothing.
constexpr int LIMIT = 15, TARGET = 11, FLOOR = 3, SLACK = 6, MOST = 60;
template <int BLOCKS>
struct Sums {
    f32x4 acc[BLOCKS][2];               // dims 32 block + 8 g + 2 r + e at [block][e][r]
    float top, total;                   // the running maximum, rounded up to a whole number; sum of p
    float up;                           // 2^power
    int slack;                          // what is left of SLACK
};
// When the power was chosen, each block's largest |P| was below 2^(size - 126). Few steps need
// that: it lies in LDS, a lane's own copy 64 words apart.
QS_DEV i16x2 size_at(const uint32_t* sizes, int i) { return __builtin_bit_cast(i16x2, sizes[64 * i]); }
template <int BLOCKS>
QS_DEV void clear(Sums<BLOCKS>& o, uint32_t* sizes) {
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) o.acc[b][0] = o.acc[b][1] = f32x4{0, 0, 0, 0};
    o.top = -__builtin_inff();
    o.total = 0.0f;
    o.up = (float)(INT64_C(1) << MOST);
    o.slack = 0;
#pragma unroll
    for (int i = 0; i < BLOCKS / 2; i++) sizes[64 * i] = 0;
}
QS_DEV i16x2 both(int v) { return i16x2{(short)v, (short)v}; }
QS_DEV i16x2 larger(i16x2 a, i16x2 b) { return __builtin_elementwise_max(a, b); }
QS_DEV int larger_of(i16x2 v) { return max((int)v[0], (int)v[1]); }
QS_DEV int power_of(float up) { return (int)(__float_as_uint(up) >> 23) - 127; }
// which blocks count by their own powers, all bits, and what blocks count by; size 0: nothing but zeros so far
QS_DEV i16x2 own(i16x2 size, int power) { return (i16x2)(size < both(FLOOR + 126 - power)) & (i16x2)(size > both(0)); }
QS_DEV i16x2 powers(i16x2 size, int power) {
    const i16x2 m = own(size, power), alone = __builtin_elementwise_min(both(TARGET + 126) - size, both(power + MOST));
    return (alone & m) | (both(power) & ~m);
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

// The running maximum rose by `fall`, which takes as much off all earlier P; `by`: the powers
// of two that the blocks' sums have to be multiplied by.
template <int BLOCKS>
QS_DEV void lower(Sums<BLOCKS>& o, int fall, i16x2 (&by)[BLOCKS / 2]) {
    o.total = __builtin_ldexpf(o.total, -fall);
    o.slack -= fall;
#pragma unroll
    for (int i = 0; i < BLOCKS / 2; i++) by[i] = both(-fall);
}
// The same, and chooses the powers anew where that is more than the slack, a P reaches LIMIT
// or a block has its first P. For other queries nothing else changes: none depends on what
// another one sees.
// first: there are no sums yet.
template <int BLOCKS, typename F>
QS_DEV void settle(Sums<BLOCKS>& o, uint32_t* sizes, bool first, int fall, const float (&p)[8], F&& step, i16x2 (&by)[BLOCKS / 2]) {
    const int was = power_of(o.up);
    i16x2 now[BLOCKS / 2], most = both(0);
#pragma unroll
    for (int i = 0; i < BLOCKS / 2; i++) {
        uint32_t e[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            float f = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) f = fmaxf(f, fabsf(__builtin_fmaf(p[j], step(j, 2 * i + h), 0.0f)));
            e[h] = __float_as_uint(f) >> 23;
        }
        now[i] = __builtin_bit_cast(i16x2, over_slots(e[0] | e[1] << 16, [](uint32_t u, uint32_t v) {
            return __builtin_bit_cast(uint32_t, larger(__builtin_bit_cast(i16x2, u), __builtin_bit_cast(i16x2, v)));
        }));
    }
    bool anew = true;
    if (!first) {
        i16x2 begins = both(0);
#pragma unroll
        for (int i = 0; i < BLOCKS / 2; i++) {
            const i16x2 then = size_at(sizes, i);
            most = larger(most, now[i] + powers(then, was));
            begins |= (i16x2)(then == both(0)) & now[i];
        }
        anew = fall > o.slack || larger_of(most) > LIMIT + 126 || __builtin_bit_cast(uint32_t, begins) != 0;
        most = both(0);
#pragma unroll
        for (int i = 0; i < BLOCKS / 2; i++) {
            const i16x2 then = size_at(sizes, i);
            now[i] = anew ? larger(then - both(SLACK - o.slack + fall), now[i]) : then;
        }
    }
#pragma unroll
    for (int i = 0; i < BLOCKS / 2; i++) most = larger(most, now[i]);
    const int power = anew ? min(TARGET + 126 - larger_of(most), MOST) : was;
    if (!first) {
        o.total = __builtin_ldexpf(o.total, -fall);
#pragma unroll
        for (int i = 0; i < BLOCKS / 2; i++)
            by[i] = larger(powers(now[i], power) - powers(size_at(sizes, i), was) - both(fall), both(-126));
    }
#pragma unroll
    for (int i = 0; i < BLOCKS / 2; i++) sizes[64 * i] = __builtin_bit_cast(uint32_t, now[i]);
    o.up = __builtin_ldexpf(1.0f, power);
    o.slack = anew ? SLACK : o.slack - fall;
}
// What a wave goes on by: whether a block of a query counts by a power of its own, and the f16
// bits of the least steps of values, block by block, that could take a P to LIMIT or begin a
// block of zeros, less one.
template <int BLOCKS>
struct Pace {
    bool uneven;
    uint32_t under[BLOCKS / 2];
};
template <int BLOCKS, int SETS>
QS_DEV Pace<BLOCKS> pace_of(const Sums<BLOCKS> (&sums)[SETS], const uint32_t* sizes) {
    Pace<BLOCKS> o;
    bool uneven = false;
#pragma unroll
    for (int i = 0; i < BLOCKS / 2; i++) {
        i16x2 up = both(-32768);
#pragma unroll
        for (int n = 0; n < SETS; n++) {
            const int power = power_of(sums[n].up);
            const bool seen = sums[n].top > -__builtin_inff();
            const i16x2 size = size_at(sizes, n * (BLOCKS / 2) + i), zero = (i16x2)(size == both(0));
            uneven |= seen & (__builtin_bit_cast(uint32_t, own(size, power)) != 0);
            up = seen ? larger(up, (powers(size, power) & ~zero) | (both(1000) & zero)) : up;
        }
        // over the eight queries: lanes ^ 1, ^ 2 and, four being alike, ^ 7
        const auto with = [&](uint32_t other) { up = larger(up, __builtin_bit_cast(i16x2, other)); };
        with(qs::quad_xor<1>(__builtin_bit_cast(uint32_t, up)));
        with(qs::quad_xor<2>(__builtin_bit_cast(uint32_t, up)));
        with((uint32_t)__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, up), 0x141, 0xF, 0xF, true));
        const half2_t least{(_Float16)__builtin_ldexpf(1.0f, LIMIT - up[0]), (_Float16)__builtin_ldexpf(1.0f, LIMIT - up[1])};
        const u16x2 under = __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, least), u16x2{1, 1});
        o.under[i] = (uint32_t)__builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, under));
    }
    o.uneven = __any(uneven);
    return o;
}

// One step: the slots start .. start + 31, in `t`. The next step's keys and values
// (at `next`) are loaded into the registers of this one's as soon as these are done
// with, and arrive while the other half is computed.
// edge: some query does not see all of the slots; to it they count for nothing,
// whatever they hold, since a lane's scores and steps are its query's own copies.
// first: of the segment's steps of the wave.
template <bool WIDE, int K_BITS, int V_BITS, int BLOCKS, int SETS>
QS_DEV void attend(const AttentionArgs& a, int start, bool first, bool edge, int held, const Place& next,
                   const Queries<BLOCKS, WIDE> (&q)[SETS], uint32_t* lds, Tile<K_BITS, V_BITS, BLOCKS>& t,
                   Sums<BLOCKS> (&sums)[SETS], uint32_t* wave_sizes, Pace<BLOCKS>& pace) {
    // Where registers are scarce, what comes of the lane's number is worked out anew in each step
    // (16 sequences of 2,048 slots, heads of 256: 43.0 us without, 40.1).
    int lane = threadIdx.x & 63;
    if constexpr (!WIDE && BLOCKS * SETS == 8) asm volatile("" : "+v"(lane));
    const int g = lane >> 4;
    uint32_t* const sizes = wave_sizes + lane;
    // steps of four slots, and one of them
    struct Steps4 {
        u32x4 w[BLOCKS / 2];
    };
    const auto steps_from = [&](int s, bool value, Steps4& o) {
        const uint32_t* p = lds + (s * 16 + 4 * g) * BLOCKS + (value ? 2 * BLOCKS : 0);
#pragma unroll
        for (int i = 0; i < BLOCKS / 2; i++) o.w[i] = *reinterpret_cast<const u32x4*>(p + 4 * i);
    };
    const auto two_of = [](const Steps4& c, int r, int b) {
        const int n = (r * BLOCKS + b) >> 1;
        return c.w[n >> 2][n & 3];
    };
    const auto step_of = [&](const Steps4& c, int r, int b) { return half_of(two_of(c, r, b) >> (16 * (b & 1))); };
    // lane after lane they are the two sixteens' steps as they lie in their pages, four keys', then four values'
    uint32_t over = 0;
#pragma unroll
    for (int i = 0; i < BLOCKS / 2; i++) {
        const uint32_t two = t.steps.w[i];
        lds[lane * (BLOCKS / 2) + i] = two;
        over |= __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(__builtin_bit_cast(u16x2, two & 0x7fff7fffu),
                                                                           __builtin_bit_cast(u16x2, pace.under[i])));
    }
    over = lane & 4 ? over : 0;
    asm volatile("" : "+v"(over));      // from here on, in place of what it comes from
    bool steep = over != 0;
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
    float lowest[SETS];     // of a maximum over slots of which some are seen: scores may all be -infinity
#pragma unroll
    for (int n = 0; n < SETS; n++) lowest[n] = LOWEST;
    if (edge) {
#pragma unroll
        for (int n = 0; n < SETS; n++) lowest[n] = -__builtin_inff();
#pragma unroll
        for (int n = 0; n < 2 * SETS; n++) {
            const int set = n >> 1, s = n & 1;
            uint32_t keep[4];
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int p = start + 16 * s + 4 * g + r;
                const bool sees = (bool)(held >> s & 1) & (p >= q[set].first) & (p < q[set].last);      // lanes do not branch
                x[set][s][r] = sees ? x[set][s][r] : -__builtin_inff();
                keep[r] = sees ? ~0u : 0u;
                lowest[set] = sees ? LOWEST : lowest[set];
            }
#pragma unroll
            for (int i = 0; i < BLOCKS / 2; i++) {
                constexpr int ROW = BLOCKS / 2;     // words of a slot
                vs[set][s].w[i] &= u32x4{keep[4 * i / ROW], keep[(4 * i + 1) / ROW], keep[(4 * i + 2) / ROW], keep[(4 * i + 3) / ROW]};
            }
        }
    }
    float p[SETS][8];
    int fall[SETS];         // the running maximum rose by so much
    bool rose = false;
#pragma unroll
    for (int n = 0; n < SETS; n++) {
        const float was = sums[n].top;
        float top = lowest[n];
#pragma unroll
        for (int i = 0; i < 8; i++) top = fmaxf(top, x[n][i >> 2][i & 3]);
        top = fmaxf(was, __builtin_ceilf(max_over_slots(top)));
        const float base = top > -__builtin_inff() ? top : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) p[n][i] = __builtin_amdgcn_exp2f(x[n][i >> 2][i & 3] - base);
        fall[n] = top != was ? (int)fminf(top - was, 1000.0f) : 0;      // 1000: nothing was seen yet
        rose |= fall[n] != 0;
        steep |= fall[n] > sums[n].slack;
        sums[n].top = top;
    }
    const bool moves = __any(steep | rose), moved = moves && !first;
    i16x2 by[SETS][BLOCKS / 2];
    if (moves) {
        if (__any(steep)) {
#pragma unroll
            for (int n = 0; n < SETS; n++)
                settle(sums[n], sizes + 32 * BLOCKS * n, first, fall[n], p[n], [&](int i, int b) {
                    // a copy: the compiler would keep all steps as f32 for what follows
                    uint32_t two = two_of(vs[n][i >> 2], i & 3, b);
                    asm volatile("" : "+v"(two));
                    return half_of(two >> (16 * (b & 1)));
                }, by[n]);
            pace = pace_of(sums, sizes);
        } else {
#pragma unroll
            for (int n = 0; n < SETS; n++) lower(sums[n], fall[n], by[n]);
        }
    }
#pragma unroll
    for (int n = 0; n < SETS; n++) {
        float total = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            total += p[n][i];
            p[n][i] *= sums[n].up;
        }
        sums[n].total += total;
    }
    const float second = lane & 8 ? 1.0f : 0.0f;
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) {
        u32x4 w[SETS];
#pragma unroll
        for (int n = 0; n < SETS; n++) {
            if (moved) {
                const float f = __builtin_ldexpf(1.0f, by[n][b >> 1][b & 1]);
#pragma unroll
                for (int i = 0; i < 8; i++) sums[n].acc[b][i >> 2][i & 3] *= f;
            }
            if (__builtin_expect(pace.uneven, 0)) {     // p goes on to this block's power
                const int power = power_of(sums[n].up);
                const auto at = [&](int b) { return b < 0 ? power : powers(size_at(sizes, (n * BLOCKS + b) >> 1), power)[b & 1]; };
                const float f = __builtin_ldexpf(1.0f, at(b) - at(b - 1));
#pragma unroll
                for (int i = 0; i < 8; i++) p[n][i] *= f;
            }
            float u[8];
            // + 0 makes it one instruction that takes the step as f16
#pragma unroll
            for (int i = 0; i < 8; i++) u[i] = __builtin_fmaf(p[n][i], step_of(vs[n][i >> 2], i & 3, b), 0.0f);
#pragma unroll
            for (int i = 0; i < 4; i++) w[n][i] = two_halves(u[2 * i], u[2 * i + 1], second);
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

// The wave's sums as one: the four lanes of a query's slots, and its two columns; what
// P count by.
template <int BLOCKS>
QS_DEV void finish(Sums<BLOCKS>& o, const uint32_t* sizes) {
    o.total = sum_over_slots(o.total);
#pragma unroll
    for (int b = 0; b < BLOCKS; b++) {
        const float once = __builtin_ldexpf(1.0f, -powers(size_at(sizes, b >> 1), power_of(o.up))[b & 1]);
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int r = 0; r < 4; r++) o.acc[b][e][r] = (o.acc[b][e][r] + other_column(o.acc[b][e][r])) * once;
    }
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
    Deal d{};
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
    __shared__ uint32_t sizes[WAVES][SETS * BLOCKS / 2][64];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
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
            clear(sums[n], &sizes[wave][n * (BLOCKS / 2)][threadIdx.x & 63]);
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
            Pace<BLOCKS> pace{};
#pragma unroll
            for (int n = 0; n < SETS; n++) prepare_queries(a, first + 8 * n, length, raw[n], q[n]);
            for (bool opens = true; i < stop; i += stride, opens = false) {
                const int start = i * TILE, held = place.held;
                place = place_of(a, ahead, head, start_of(i + stride));
                ahead = pages_of(a, table, start_of(i + 2 * stride));
                const bool edge = start < span.all_first || start + TILE > span.all_last || held != 3;
                attend(a, start, opens, edge, held, place, q, steps_lds[wave], t, sums, sizes[wave][0], pace);
            }
        }
        // anew from here, so that no step holds registers for the addresses of what follows
        int thread = (int)threadIdx.x;
        asm volatile("" : "+v"(thread));
        const int lane = thread & 63, g = lane >> 4;
#pragma unroll
        for (int n = 0; n < SETS; n++) {
            finish(sums[n], &sizes[wave][n * (BLOCKS / 2)][lane]);
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
        const int sub = thread & 31;
#pragma unroll
        for (int k = 0; k < COLUMNS; k += 2 * WAVES) {
            const int column = k + (thread >> 5);
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
            const float inverse = inverse_of(ref, total);
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
