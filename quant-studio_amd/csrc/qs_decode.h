// Packed GGUF blocks back to integers and scales (gfx950): what the products
// with packed weights read. Every format stands for values
//     w = d * c - m
// with c an integer of 8 bits, and d, m constant over 32 or 16 values, so a
// product with 8-bit rows is an integer dot product per group and one f32
// multiplication of its result. decode_group() yields one group of 32.
#pragma once

#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qs_grids.h"
#include "quant_studio.h"

#ifndef QS_DEV
#define QS_DEV __device__ __forceinline__
#endif

namespace qsd {

// BLK values in BYTES bytes; SUB groups of 32 / SUB values with a scale of
// their own in each 32; MIN: there is an m; GRID: entries of the type's grid;
// RAW: words that hold a group's bytes and its block's scales.
template <int TYPE>
struct Format;
#define QS_FORMAT(T, blk, bytes, sub, min, grid, raw)                                     \
    template <>                                                                           \
    struct Format<T> {                                                                    \
        static constexpr int BLK = blk, BYTES = bytes, SUB = sub, GRID = grid, RAW = raw; \
        static constexpr bool MIN = min;                                                  \
    };
QS_FORMAT(QS_TYPE_Q4_0, 32, 18, 1, false, 0, 5)
QS_FORMAT(QS_TYPE_Q4_1, 32, 20, 1, true, 0, 5)
QS_FORMAT(QS_TYPE_Q5_0, 32, 22, 1, false, 0, 6)
QS_FORMAT(QS_TYPE_Q5_1, 32, 24, 1, true, 0, 6)
QS_FORMAT(QS_TYPE_Q8_0, 32, 34, 1, false, 0, 9)
QS_FORMAT(QS_TYPE_IQ4_NL, 32, 18, 1, false, 0, 5)
QS_FORMAT(QS_TYPE_Q2_K, 256, 84, 2, true, 0, 10)
QS_FORMAT(QS_TYPE_Q3_K, 256, 110, 2, false, 0, 20)
QS_FORMAT(QS_TYPE_Q4_K, 256, 144, 1, true, 0, 12)
QS_FORMAT(QS_TYPE_Q5_K, 256, 176, 1, true, 0, 20)
QS_FORMAT(QS_TYPE_Q6_K, 256, 210, 2, false, 0, 18)
QS_FORMAT(QS_TYPE_IQ4_XS, 256, 136, 1, false, 0, 6)
QS_FORMAT(QS_TYPE_IQ2_XXS, 256, 66, 1, false, 256, 3)
QS_FORMAT(QS_TYPE_IQ2_XS, 256, 74, 2, false, 512, 4)
QS_FORMAT(QS_TYPE_IQ2_S, 256, 82, 2, false, 1024, 5)
QS_FORMAT(QS_TYPE_IQ3_XXS, 256, 98, 1, false, 256, 4)
QS_FORMAT(QS_TYPE_IQ3_S, 256, 110, 1, false, 512, 6)
#undef QS_FORMAT

// The grids of the IQ types as device constants; a kernel copies the one it
// needs to LDS (stage_grid), where a lookup per lane costs bank conflicts
// rather than a cache line each.
template <int TYPE>
QS_DEV uint16_t grid_entry(int i) {
    if constexpr (TYPE == QS_TYPE_IQ2_XXS) return QS_GRID2_256[i];
    else if constexpr (TYPE == QS_TYPE_IQ2_XS) return QS_GRID2_512[i];
    else if constexpr (TYPE == QS_TYPE_IQ2_S) return QS_GRID2_1024[i];
    else if constexpr (TYPE == QS_TYPE_IQ3_XXS) return QS_GRID3_256[i];
    else if constexpr (TYPE == QS_TYPE_IQ3_S) return QS_GRID3_512[i];
    else return 0;
}

template <int TYPE>
QS_DEV void stage_grid(uint16_t* lds, int tid, int nthreads) {
    if constexpr (Format<TYPE>::GRID > 0)
        for (int i = tid; i < Format<TYPE>::GRID; i += nthreads) lds[i] = grid_entry<TYPE>(i);
}

// one group of 32: integers in order, four to a word, and the scales
template <int TYPE>
struct Group {
    uint32_t c[8];
    float d[Format<TYPE>::SUB];
    float m[Format<TYPE>::SUB];     // 0 without MIN
};

// ---- bytes ----

// Blocks start at any even address; the hardware takes such loads from memory.
template <int WORDS>
QS_DEV void load_words(const uint8_t* p, uint32_t (&w)[WORDS]) {
    __builtin_memcpy(w, p, 4 * WORDS);
}
QS_DEV uint32_t load_u16(const uint8_t* p) {
    uint16_t v;
    __builtin_memcpy(&v, p, 2);
    return v;
}

// A place in bytes copied to LDS (on whose boundaries the copy keeps memory's).
// An LDS read off its boundary takes several times as long (of Q6_K's 210-byte
// blocks it made four fifths of the LDS time), so where blocks are not whole
// words (SHIFT) the words around are read and shifted together.
template <bool SHIFT>
struct LdsBytes {
    const uint8_t* base;
    int at;
    QS_DEV LdsBytes operator+(int o) const { return {base, at + o}; }
    QS_DEV uint8_t operator[](int o) const { return base[at + o]; }
};
template <int WORDS, bool SHIFT>
QS_DEV void load_words(LdsBytes<SHIFT> p, uint32_t (&w)[WORDS]) {
    if constexpr (!SHIFT) {
        __builtin_memcpy(w, __builtin_assume_aligned(p.base + p.at, 4), 4 * WORDS);
    } else {
        const uint32_t* d = reinterpret_cast<const uint32_t*>(p.base + (p.at & ~3));
        const uint32_t sh = (uint32_t)(p.at & 2) * 8;
        uint32_t lo = d[0];
#pragma unroll
        for (int i = 0; i < WORDS; i++) {
            const uint32_t hi = d[i + 1];
            w[i] = __builtin_amdgcn_alignbit(hi, lo, sh);
            lo = hi;
        }
    }
}
template <bool SHIFT>
QS_DEV uint32_t load_u16(LdsBytes<SHIFT> p) {
    return *reinterpret_cast<const uint16_t*>(p.base + p.at);
}
template <typename P>
QS_DEV uint32_t load_u32(P p) {
    uint32_t w[1];
    load_words(p, w);
    return w[0];
}
QS_DEV float half_bits(uint32_t b) { return __half2float(__ushort_as_half((unsigned short)b)); }

// A scale as it is, NaN where it is infinite: such a scale stands for no values.
// Codes summed before it is applied would else give an infinity where the values
// singly, infinities of both signs and inf * 0, add up to a NaN.
QS_DEV float scale_of(float s) { return __builtin_fmaf(s, 0.0f, s); }
QS_DEV float scale_bits(uint32_t b) { return scale_of(half_bits(b)); }

// ---- four bytes at a time ----

constexpr uint32_t ONES = 0x01010101u;

// v - B in every byte, for bytes v < 0x80: the set top bit takes the borrow
template <uint32_t B>
QS_DEV uint32_t sub_bytes(uint32_t v) {
    return ((v | 0x80808080u) - B * ONES) ^ 0x80808080u;
}
// bits 0..3 of n to bit 0 of the four bytes
QS_DEV uint32_t spread4(uint32_t n) { return __umul24(n & 15u, 0x00204081u) & ONES; }
// 0x00 / 0xff from bit 0 of the four bytes
QS_DEV uint32_t byte_mask(uint32_t b) { return (b << 8) - b; }
// -v in the bytes where n's bit is set (v in 1..127: no carry between bytes)
QS_DEV uint32_t sign4(uint32_t v, uint32_t n) {
    const uint32_t b = spread4(n);
    return (v ^ byte_mask(b)) + b;
}
// the eighth sign of seven stored ones: their parity
QS_DEV uint32_t signs8(uint32_t v7) { return v7 | ((__popc(v7) & 1u) << 7); }

// byte j of the result: byte sel_j (0..7) of the table hi:lo
QS_DEV uint32_t pick8(uint32_t hi, uint32_t lo, uint32_t sel) { return __builtin_amdgcn_perm(hi, lo, sel); }

// the IQ4 levels -127 -104 -83 -65 | -49 -35 -22 -10 | 1 13 25 38 | 53 69 89 113
QS_DEV uint32_t iq4_levels(uint32_t nib) {
    const uint32_t sel = nib & 0x07070707u;
    const uint32_t lo = pick8(0xf6eaddcfu, 0xbfad9881u, sel), hi = pick8(0x71594535u, 0x26190d01u, sel);
    const uint32_t top = byte_mask((nib >> 3) & ONES);
    return (hi & top) | (lo & ~top);
}
// four 2-bit levels 0..2 -> 8, 25, 43
QS_DEV uint32_t iq2_levels(uint32_t code) {
    const uint32_t sel = (code & 3u) | ((code & 0xcu) << 6) | ((code & 0x30u) << 12) | ((code & 0xc0u) << 18);
    return pick8(0, 0x002b1908u, sel);
}
// four 3-bit levels to table bytes
QS_DEV uint32_t iq3_levels(uint32_t code, uint32_t hi, uint32_t lo) {
    const uint32_t sel = (code & 7u) | ((code & 0x38u) << 5) | ((code & 0x1c0u) << 10) | ((code & 0xe00u) << 15);
    return pick8(hi, lo, sel);
}

// 6-bit scale and minimum j of the 12-byte field of Q4_K / Q5_K (words s)
QS_DEV void scale_min(const uint32_t (&s)[3], int j, uint32_t& sc, uint32_t& mn) {
    const int sh = 8 * (j & 3);
    const uint32_t a = s[0] >> sh, b = s[1] >> sh, c = s[2] >> sh;
    const bool low = j < 4;
    sc = low ? (a & 63u) : ((c & 15u) | ((a >> 2) & 0x30u));
    mn = low ? (b & 63u) : (((c >> 4) & 15u) | ((b >> 2) & 0x30u));
}

// The bytes of group g (0 .. BLK/32 - 1) of the block at b, as loaded: what a
// kernel holds between issuing the loads and using them.
template <int TYPE>
struct Raw {
    uint32_t w[Format<TYPE>::RAW];
};

template <int N, int WORDS, typename P>
QS_DEV void load_at(uint32_t (&w)[WORDS], int at, P p) {
    uint32_t v[N];
    load_words(p, v);
#pragma unroll
    for (int i = 0; i < N; i++) w[at + i] = v[i];
}

template <int TYPE, typename P>
QS_DEV void load_group(P b, int g, Raw<TYPE>& o) {
    if constexpr (TYPE == QS_TYPE_Q4_0 || TYPE == QS_TYPE_IQ4_NL) {
        load_at<4>(o.w, 0, b + 2);
        o.w[4] = load_u16(b);
    } else if constexpr (TYPE == QS_TYPE_Q4_1) {
        load_at<4>(o.w, 0, b + 4);
        o.w[4] = load_u32(b);
    } else if constexpr (TYPE == QS_TYPE_Q5_0) {
        load_at<5>(o.w, 0, b + 2);      // the fifth bits, then 16 bytes of nibbles
        o.w[5] = load_u16(b);
    } else if constexpr (TYPE == QS_TYPE_Q5_1) {
        load_at<5>(o.w, 0, b + 4);
        o.w[5] = load_u32(b);
    } else if constexpr (TYPE == QS_TYPE_Q8_0) {
        load_at<8>(o.w, 0, b + 2);
        o.w[8] = load_u16(b);
    } else if constexpr (TYPE == QS_TYPE_Q2_K) {
        load_at<8>(o.w, 0, b + 16 + 32 * (g >> 2));
        o.w[8] = load_u32(b + 80);
        o.w[9] = load_u16(b + 2 * g);
    } else if constexpr (TYPE == QS_TYPE_Q3_K) {
        load_at<8>(o.w, 0, b + 32 + 32 * (g >> 2));
        load_at<8>(o.w, 8, b);
        load_at<3>(o.w, 16, b + 96);
        o.w[19] = load_u16(b + 108);
    } else if constexpr (TYPE == QS_TYPE_Q4_K) {
        load_at<8>(o.w, 0, b + 16 + 32 * (g >> 1));
        load_at<4>(o.w, 8, b);          // d, dmin, 12 bytes of scales
    } else if constexpr (TYPE == QS_TYPE_Q5_K) {
        load_at<8>(o.w, 0, b + 48 + 32 * (g >> 1));
        load_at<4>(o.w, 8, b);
        load_at<8>(o.w, 12, b + 16);
    } else if constexpr (TYPE == QS_TYPE_Q6_K) {
        load_at<8>(o.w, 0, b + 64 * (g >> 2) + 32 * (g & 1));
        load_at<8>(o.w, 8, b + 128 + 32 * (g >> 2));
        o.w[16] = load_u16(b + 192 + 2 * g);
        o.w[17] = load_u16(b + 208);
    } else if constexpr (TYPE == QS_TYPE_IQ4_XS) {
        load_at<4>(o.w, 0, b + 8 + 16 * g);
        load_at<2>(o.w, 4, b);
    } else if constexpr (TYPE == QS_TYPE_IQ2_XXS) {
        load_at<2>(o.w, 0, b + 2 + 8 * g);      // four grid indices; four times seven signs and the scale
        o.w[2] = load_u16(b);
    } else if constexpr (TYPE == QS_TYPE_IQ2_XS) {
        load_at<2>(o.w, 0, b + 2 + 8 * g);      // four entries: grid index (9 bits), seven signs
        o.w[2] = load_u16(b);
        o.w[3] = b[66 + g];
    } else if constexpr (TYPE == QS_TYPE_IQ2_S) {
        o.w[0] = load_u32(b + 2 + 4 * g);
        o.w[1] = load_u32(b + 34 + 4 * g);
        o.w[2] = load_u16(b);
        o.w[3] = b[66 + g];
        o.w[4] = b[74 + g];
    } else if constexpr (TYPE == QS_TYPE_IQ3_XXS) {
        load_at<2>(o.w, 0, b + 2 + 8 * g);      // eight grid indices
        o.w[2] = load_u32(b + 66 + 4 * g);
        o.w[3] = load_u16(b);
    } else {
        static_assert(TYPE == QS_TYPE_IQ3_S, "format");
        load_at<2>(o.w, 0, b + 2 + 8 * g);
        o.w[2] = load_u32(b + 74 + 4 * g);
        o.w[3] = load_u16(b);
        o.w[4] = b[66 + g];
        o.w[5] = b[106 + (g >> 1)];
    }
}

// scale k (of 16) of a Q3_K block: the low nibbles of bytes 0..7, then their
// high ones; two more bits from bytes 8..11
template <int TYPE>
QS_DEV int q3_scale(const Raw<TYPE>& r, int k) {
    const int by = 8 * (k & 3);
    const uint32_t lo = ((((k >> 2) & 1) ? r.w[17] : r.w[16]) >> (by + 4 * (k >> 3))) & 15u;
    const uint32_t hi = (r.w[18] >> (by + 2 * (k >> 2))) & 3u;
    return (int)(lo | (hi << 4)) - 32;
}

// What the codes of a format are less than the bits that store them (they have
// a minimum, are signed, or come from a table: 0).
template <int TYPE>
constexpr int offset() {
    return TYPE == QS_TYPE_Q4_0 ? 8 : TYPE == QS_TYPE_Q5_0 ? 16 : TYPE == QS_TYPE_Q3_K ? 4 : TYPE == QS_TYPE_Q6_K ? 32 : 0;
}
template <int TYPE, bool STORED>
QS_DEV uint32_t codes(uint32_t stored) {
    if constexpr (STORED || offset<TYPE>() == 0) return stored;
    else return sub_bytes<offset<TYPE>()>(stored);
}

// Group g of a block from its bytes. `grid` is the staged table of the IQ
// types. STORED: the codes as stored, offset() too large.
template <int TYPE, bool STORED = false>
QS_DEV void decode_group(const Raw<TYPE>& r, int g, const uint16_t* grid, Group<TYPE>& o) {
    const uint32_t(&w)[Format<TYPE>::RAW] = r.w;
    o.m[0] = o.m[Format<TYPE>::SUB - 1] = 0.0f;
    if constexpr (TYPE == QS_TYPE_Q4_0 || TYPE == QS_TYPE_Q4_1 || TYPE == QS_TYPE_IQ4_NL) {
        o.d[0] = scale_bits(w[4] & 0xffffu);
        if constexpr (TYPE == QS_TYPE_Q4_1) o.m[0] = -scale_bits(w[4] >> 16);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t lo = w[i] & 0x0f0f0f0fu, hi = (w[i] >> 4) & 0x0f0f0f0fu;
            if constexpr (TYPE == QS_TYPE_IQ4_NL) o.c[i] = iq4_levels(lo), o.c[4 + i] = iq4_levels(hi);
            else o.c[i] = codes<TYPE, STORED>(lo), o.c[4 + i] = codes<TYPE, STORED>(hi);
        }
    } else if constexpr (TYPE == QS_TYPE_Q5_0 || TYPE == QS_TYPE_Q5_1) {
        o.d[0] = scale_bits(w[5] & 0xffffu);
        if constexpr (TYPE == QS_TYPE_Q5_1) o.m[0] = -scale_bits(w[5] >> 16);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t lo = (w[1 + i] & 0x0f0f0f0fu) | (spread4(w[0] >> (4 * i)) << 4);
            const uint32_t hi = ((w[1 + i] >> 4) & 0x0f0f0f0fu) | (spread4(w[0] >> (16 + 4 * i)) << 4);
            o.c[i] = codes<TYPE, STORED>(lo), o.c[4 + i] = codes<TYPE, STORED>(hi);
        }
    } else if constexpr (TYPE == QS_TYPE_Q8_0) {
#pragma unroll
        for (int i = 0; i < 8; i++) o.c[i] = w[i];
        o.d[0] = scale_bits(w[8]);
    } else if constexpr (TYPE == QS_TYPE_Q2_K) {
        const uint32_t sc = w[9];
        const float d = scale_bits(w[8] & 0xffffu), dmin = scale_bits(w[8] >> 16);
        o.d[0] = d * (float)(sc & 15u), o.m[0] = dmin * (float)((sc >> 4) & 15u);
        o.d[1] = d * (float)((sc >> 8) & 15u), o.m[1] = dmin * (float)(sc >> 12);
        const int sh = 2 * (g & 3);
#pragma unroll
        for (int i = 0; i < 8; i++) o.c[i] = (w[i] >> sh) & 0x03030303u;
    } else if constexpr (TYPE == QS_TYPE_Q3_K) {
        const float d = scale_bits(w[19]);
        const int sh = 2 * (g & 3);
#pragma unroll
        for (int i = 0; i < 8; i++)
            o.c[i] = codes<TYPE, STORED>(((w[i] >> sh) & 0x03030303u) | (((w[8 + i] >> g) & ONES) << 2));
#pragma unroll
        for (int j = 0; j < 2; j++) o.d[j] = d * (float)q3_scale(r, 2 * g + j);
    } else if constexpr (TYPE == QS_TYPE_Q4_K || TYPE == QS_TYPE_Q5_K) {
        uint32_t sc, mn;
        const uint32_t s[3] = {w[9], w[10], w[11]};
        scale_min(s, g, sc, mn);
        o.d[0] = scale_bits(w[8] & 0xffffu) * (float)sc;
        o.m[0] = scale_bits(w[8] >> 16) * (float)mn;
        const int sh = 4 * (g & 1);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            o.c[i] = (w[i] >> sh) & 0x0f0f0f0fu;
            if constexpr (TYPE == QS_TYPE_Q5_K) o.c[i] |= ((w[12 + i] >> g) & ONES) << 4;
        }
    } else if constexpr (TYPE == QS_TYPE_Q6_K) {
        const float d = scale_bits(w[17]);
        o.d[0] = d * (float)(int8_t)(w[16] & 0xffu), o.d[1] = d * (float)(int8_t)(w[16] >> 8);
        const int sl = 4 * ((g >> 1) & 1), sh = 2 * (g & 3);
#pragma unroll
        for (int i = 0; i < 8; i++)
            o.c[i] = codes<TYPE, STORED>(((w[i] >> sl) & 0x0f0f0f0fu) | (((w[8 + i] >> sh) & 0x03030303u) << 4));
    } else if constexpr (TYPE == QS_TYPE_IQ4_XS) {
        const uint32_t ls = ((w[5] >> (4 * g)) & 15u) | (((w[4] >> (16 + 2 * g)) & 3u) << 4);
        o.d[0] = scale_bits(w[4] & 0xffffu) * (float)((int)ls - 32);
#pragma unroll
        for (int i = 0; i < 4; i++)
            o.c[i] = iq4_levels(w[i] & 0x0f0f0f0fu), o.c[4 + i] = iq4_levels((w[i] >> 4) & 0x0f0f0f0fu);
    } else if constexpr (TYPE == QS_TYPE_IQ2_XXS) {
        o.d[0] = scale_bits(w[2]) * (0.5f + (float)(w[1] >> 28)) * 0.25f;
#pragma unroll
        for (int l = 0; l < 4; l++) {
            const uint32_t e = grid[(w[0] >> (8 * l)) & 255u], s = signs8((w[1] >> (7 * l)) & 127u);
            o.c[2 * l] = sign4(iq2_levels(e), s), o.c[2 * l + 1] = sign4(iq2_levels(e >> 8), s >> 4);
        }
    } else if constexpr (TYPE == QS_TYPE_IQ2_XS) {
        const float d = scale_bits(w[2]);
        o.d[0] = d * (0.5f + (float)(w[3] & 15u)) * 0.25f, o.d[1] = d * (0.5f + (float)(w[3] >> 4)) * 0.25f;
#pragma unroll
        for (int l = 0; l < 4; l++) {
            const uint32_t v = (w[l >> 1] >> (16 * (l & 1))) & 0xffffu;
            const uint32_t e = grid[v & 511u], s = signs8(v >> 9);
            o.c[2 * l] = sign4(iq2_levels(e), s), o.c[2 * l + 1] = sign4(iq2_levels(e >> 8), s >> 4);
        }
    } else if constexpr (TYPE == QS_TYPE_IQ2_S) {
        const float d = scale_bits(w[2]);
        o.d[0] = d * (0.5f + (float)(w[4] & 15u)) * 0.25f, o.d[1] = d * (0.5f + (float)(w[4] >> 4)) * 0.25f;
#pragma unroll
        for (int l = 0; l < 4; l++) {
            const uint32_t e = grid[((w[0] >> (8 * l)) & 255u) | (((w[3] >> (2 * l)) & 3u) << 8)], s = w[1] >> (8 * l);
            o.c[2 * l] = sign4(iq2_levels(e), s), o.c[2 * l + 1] = sign4(iq2_levels(e >> 8), s >> 4);
        }
    } else if constexpr (TYPE == QS_TYPE_IQ3_XXS) {
        o.d[0] = scale_bits(w[3]) * (0.5f + (float)(w[2] >> 28)) * 0.5f;
#pragma unroll
        for (int l = 0; l < 4; l++) {
            const uint32_t s = signs8((w[2] >> (7 * l)) & 127u), i2 = w[l >> 1] >> (16 * (l & 1));
            // levels 4 12 20 28 36 44 52 62
            o.c[2 * l] = sign4(iq3_levels(grid[i2 & 255u], 0x3e342c24u, 0x1c140c04u), s);
            o.c[2 * l + 1] = sign4(iq3_levels(grid[(i2 >> 8) & 255u], 0x3e342c24u, 0x1c140c04u), s >> 4);
        }
    } else {
        static_assert(TYPE == QS_TYPE_IQ3_S, "format");
        o.d[0] = scale_bits(w[3]) * (float)(1 + 2 * ((w[5] >> (4 * (g & 1))) & 15u));
#pragma unroll
        for (int l = 0; l < 4; l++) {
            const uint32_t s = w[2] >> (8 * l), i2 = w[l >> 1] >> (16 * (l & 1)), h = w[4] >> (2 * l);
            // levels 1 3 5 ... 15
            o.c[2 * l] = sign4(iq3_levels(grid[(i2 & 255u) | ((h & 1u) << 8)], 0x0f0d0b09u, 0x07050301u), s);
            o.c[2 * l + 1] =
                sign4(iq3_levels(grid[((i2 >> 8) & 255u) | ((h & 2u) << 7)], 0x0f0d0b09u, 0x07050301u), s >> 4);
        }
    }
}

// the group of 32 values number `gi` of a row, and its number in its block
template <int TYPE, typename P>
QS_DEV void load_row_group(P row, int gi, Raw<TYPE>& o) {
    constexpr int PER = Format<TYPE>::BLK / 32;
    load_group<TYPE>(row + gi / PER * Format<TYPE>::BYTES, gi % PER, o);    // a row is under 2^31 bytes
}
template <int TYPE>
QS_DEV int group_in_block(int gi) {
    return gi % (Format<TYPE>::BLK / 32);
}

}  // namespace qsd
