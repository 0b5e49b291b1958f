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
// their own in each 32; MIN: there is an m.
template <int TYPE>
struct Format;
#define QS_FORMAT(T, blk, bytes, sub, min, grid)                                          \
    template <>                                                                           \
    struct Format<T> {                                                                    \
        static constexpr int BLK = blk, BYTES = bytes, SUB = sub, GRID = grid;            \
        static constexpr bool MIN = min;                                                  \
    };
QS_FORMAT(QS_TYPE_Q4_0, 32, 18, 1, false, 0)
QS_FORMAT(QS_TYPE_Q4_1, 32, 20, 1, true, 0)
QS_FORMAT(QS_TYPE_Q5_0, 32, 22, 1, false, 0)
QS_FORMAT(QS_TYPE_Q5_1, 32, 24, 1, true, 0)
QS_FORMAT(QS_TYPE_Q8_0, 32, 34, 1, false, 0)
QS_FORMAT(QS_TYPE_IQ4_NL, 32, 18, 1, false, 0)
QS_FORMAT(QS_TYPE_Q2_K, 256, 84, 2, true, 0)
QS_FORMAT(QS_TYPE_Q3_K, 256, 110, 2, false, 0)
QS_FORMAT(QS_TYPE_Q4_K, 256, 144, 1, true, 0)
QS_FORMAT(QS_TYPE_Q5_K, 256, 176, 1, true, 0)
QS_FORMAT(QS_TYPE_Q6_K, 256, 210, 2, false, 0)
QS_FORMAT(QS_TYPE_IQ4_XS, 256, 136, 1, false, 0)
QS_FORMAT(QS_TYPE_IQ2_XXS, 256, 66, 1, false, 256)
QS_FORMAT(QS_TYPE_IQ2_XS, 256, 74, 2, false, 512)
QS_FORMAT(QS_TYPE_IQ2_S, 256, 82, 2, false, 1024)
QS_FORMAT(QS_TYPE_IQ3_XXS, 256, 98, 1, false, 256)
QS_FORMAT(QS_TYPE_IQ3_S, 256, 110, 1, false, 512)
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

// Blocks start at any even address; the hardware takes such loads.
template <int WORDS>
QS_DEV void load_words(const uint8_t* p, uint32_t (&w)[WORDS]) {
    __builtin_memcpy(w, p, 4 * WORDS);
}
QS_DEV uint32_t load_u32(const uint8_t* p) {
    uint32_t v;
    __builtin_memcpy(&v, p, 4);
    return v;
}
QS_DEV uint32_t load_u16(const uint8_t* p) {
    uint16_t v;
    __builtin_memcpy(&v, p, 2);
    return v;
}
QS_DEV float half_bits(uint32_t b) { return __half2float(__ushort_as_half((unsigned short)b)); }
QS_DEV float load_f16(const uint8_t* p) { return half_bits(load_u16(p)); }

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

// Group g (0 .. BLK/32 - 1) of the block at b. `grid` is the staged table of
// the IQ types.
template <int TYPE>
QS_DEV void decode_group(const uint8_t* b, int g, const uint16_t* grid, Group<TYPE>& o) {
    o.m[0] = 0.0f;
    if constexpr (TYPE == QS_TYPE_Q4_0 || TYPE == QS_TYPE_Q4_1 || TYPE == QS_TYPE_IQ4_NL) {
        uint32_t w[4];
        load_words(b + (TYPE == QS_TYPE_Q4_1 ? 4 : 2), w);
        o.d[0] = load_f16(b);
        if constexpr (TYPE == QS_TYPE_Q4_1) o.m[0] = -load_f16(b + 2);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t lo = w[i] & 0x0f0f0f0fu, hi = (w[i] >> 4) & 0x0f0f0f0fu;
            if constexpr (TYPE == QS_TYPE_Q4_0) o.c[i] = sub_bytes<8>(lo), o.c[4 + i] = sub_bytes<8>(hi);
            else if constexpr (TYPE == QS_TYPE_Q4_1) o.c[i] = lo, o.c[4 + i] = hi;
            else o.c[i] = iq4_levels(lo), o.c[4 + i] = iq4_levels(hi);
        }
    } else if constexpr (TYPE == QS_TYPE_Q5_0 || TYPE == QS_TYPE_Q5_1) {
        constexpr int AT = TYPE == QS_TYPE_Q5_0 ? 2 : 4;
        uint32_t w[5];
        load_words(b + AT, w);      // the fifth bits, then 16 bytes of nibbles
        o.d[0] = load_f16(b);
        if constexpr (TYPE == QS_TYPE_Q5_1) o.m[0] = -load_f16(b + 2);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t lo = (w[1 + i] & 0x0f0f0f0fu) | (spread4(w[0] >> (4 * i)) << 4);
            const uint32_t hi = ((w[1 + i] >> 4) & 0x0f0f0f0fu) | (spread4(w[0] >> (16 + 4 * i)) << 4);
            o.c[i] = TYPE == QS_TYPE_Q5_0 ? sub_bytes<16>(lo) : lo;
            o.c[4 + i] = TYPE == QS_TYPE_Q5_0 ? sub_bytes<16>(hi) : hi;
        }
    } else if constexpr (TYPE == QS_TYPE_Q8_0) {
        load_words(b + 2, o.c);
        o.d[0] = load_f16(b);
    } else if constexpr (TYPE == QS_TYPE_Q2_K) {
        uint32_t w[8];
        load_words(b + 16 + 32 * (g >> 2), w);
        const uint32_t sc = load_u16(b + 2 * g), dd = load_u32(b + 80);
        const float d = half_bits(dd & 0xffffu), dmin = half_bits(dd >> 16);
        o.d[0] = d * (float)(sc & 15u), o.m[0] = dmin * (float)((sc >> 4) & 15u);
        o.d[1] = d * (float)((sc >> 8) & 15u), o.m[1] = dmin * (float)(sc >> 12);
        const int sh = 2 * (g & 3);
#pragma unroll
        for (int i = 0; i < 8; i++) o.c[i] = (w[i] >> sh) & 0x03030303u;
    } else if constexpr (TYPE == QS_TYPE_Q3_K) {
        uint32_t w[8], h[8], s[3];
        load_words(b + 32 + 32 * (g >> 2), w);
        load_words(b, h);
        load_words(b + 96, s);
        const float d = load_f16(b + 108);
        const int sh = 2 * (g & 3);
#pragma unroll
        for (int i = 0; i < 8; i++)
            o.c[i] = sub_bytes<4>(((w[i] >> sh) & 0x03030303u) | (((h[i] >> g) & ONES) << 2));
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const int k = 2 * g + j, by = 8 * (k & 3);
            // scale k: the low nibbles of bytes 0..7, then their high ones; two more bits from bytes 8..11
            const uint32_t lo = ((((k >> 2) & 1) ? s[1] : s[0]) >> (by + 4 * (k >> 3))) & 15u;
            const uint32_t hi = (s[2] >> (by + 2 * (k >> 2))) & 3u;
            o.d[j] = d * (float)((int)(lo | (hi << 4)) - 32);
        }
        o.m[1] = 0.0f;
    } else if constexpr (TYPE == QS_TYPE_Q4_K || TYPE == QS_TYPE_Q5_K) {
        uint32_t head[4], w[8], h[8], sc, mn;
        load_words(b, head);        // d, dmin, 12 bytes of scales
        load_words(b + (TYPE == QS_TYPE_Q4_K ? 16 : 48) + 32 * (g >> 1), w);
        if constexpr (TYPE == QS_TYPE_Q5_K) load_words(b + 16, h);
        const uint32_t s[3] = {head[1], head[2], head[3]};
        scale_min(s, g, sc, mn);
        o.d[0] = half_bits(head[0] & 0xffffu) * (float)sc;
        o.m[0] = half_bits(head[0] >> 16) * (float)mn;
        const int sh = 4 * (g & 1);
#pragma unroll
        for (int i = 0; i < 8; i++) {
            o.c[i] = (w[i] >> sh) & 0x0f0f0f0fu;
            if constexpr (TYPE == QS_TYPE_Q5_K) o.c[i] |= ((h[i] >> g) & ONES) << 4;
        }
    } else if constexpr (TYPE == QS_TYPE_Q6_K) {
        const int n = g >> 2, quad = g & 3;
        uint32_t w[8], h[8];
        load_words(b + 64 * n + 32 * (quad & 1), w);
        load_words(b + 128 + 32 * n, h);
        const uint32_t sc = load_u16(b + 192 + 2 * g);
        const float d = load_f16(b + 208);
        o.d[0] = d * (float)(int8_t)(sc & 0xffu), o.d[1] = d * (float)(int8_t)(sc >> 8);
        o.m[1] = 0.0f;
        const int sl = 4 * (quad >> 1), sh = 2 * quad;
#pragma unroll
        for (int i = 0; i < 8; i++)
            o.c[i] = sub_bytes<32>(((w[i] >> sl) & 0x0f0f0f0fu) | (((h[i] >> sh) & 0x03030303u) << 4));
    } else if constexpr (TYPE == QS_TYPE_IQ4_XS) {
        uint32_t w[4];
        load_words(b + 8 + 16 * g, w);
        const uint32_t head = load_u32(b), sl = load_u32(b + 4);
        const uint32_t ls = ((sl >> (4 * g)) & 15u) | (((head >> (16 + 2 * g)) & 3u) << 4);
        o.d[0] = half_bits(head & 0xffffu) * (float)((int)ls - 32);
#pragma unroll
        for (int i = 0; i < 4; i++)
            o.c[i] = iq4_levels(w[i] & 0x0f0f0f0fu), o.c[4 + i] = iq4_levels((w[i] >> 4) & 0x0f0f0f0fu);
    } else if constexpr (TYPE == QS_TYPE_IQ2_XXS) {
        uint32_t w[2];              // four grid indices; four times seven signs and the scale
        load_words(b + 2 + 8 * g, w);
        o.d[0] = load_f16(b) * (0.5f + (float)(w[1] >> 28)) * 0.25f;
#pragma unroll
        for (int l = 0; l < 4; l++) {
            const uint32_t e = grid[(w[0] >> (8 * l)) & 255u], s = signs8((w[1] >> (7 * l)) & 127u);
            o.c[2 * l] = sign4(iq2_levels(e), s), o.c[2 * l + 1] = sign4(iq2_levels(e >> 8), s >> 4);
        }
    } else if constexpr (TYPE == QS_TYPE_IQ2_XS) {
        uint32_t w[2];              // four entries: grid index (9 bits), seven signs
        load_words(b + 2 + 8 * g, w);
        const float d = load_f16(b);
        const uint32_t sc = b[66 + g];
        o.d[0] = d * (0.5f + (float)(sc & 15u)) * 0.25f, o.d[1] = d * (0.5f + (float)(sc >> 4)) * 0.25f;
        o.m[1] = 0.0f;
#pragma unroll
        for (int l = 0; l < 4; l++) {
            const uint32_t v = (w[l >> 1] >> (16 * (l & 1))) & 0xffffu;
            const uint32_t e = grid[v & 511u], s = signs8(v >> 9);
            o.c[2 * l] = sign4(iq2_levels(e), s), o.c[2 * l + 1] = sign4(iq2_levels(e >> 8), s >> 4);
        }
    } else if constexpr (TYPE == QS_TYPE_IQ2_S) {
        const uint32_t idx = load_u32(b + 2 + 4 * g), sg = load_u32(b + 34 + 4 * g);
        const uint32_t qh = b[66 + g], sc = b[74 + g];
        const float d = load_f16(b);
        o.d[0] = d * (0.5f + (float)(sc & 15u)) * 0.25f, o.d[1] = d * (0.5f + (float)(sc >> 4)) * 0.25f;
        o.m[1] = 0.0f;
#pragma unroll
        for (int l = 0; l < 4; l++) {
            const uint32_t e = grid[((idx >> (8 * l)) & 255u) | (((qh >> (2 * l)) & 3u) << 8)], s = sg >> (8 * l);
            o.c[2 * l] = sign4(iq2_levels(e), s), o.c[2 * l + 1] = sign4(iq2_levels(e >> 8), s >> 4);
        }
    } else if constexpr (TYPE == QS_TYPE_IQ3_XXS) {
        uint32_t w[2];              // eight grid indices
        load_words(b + 2 + 8 * g, w);
        const uint32_t aux = load_u32(b + 66 + 4 * g);
        o.d[0] = load_f16(b) * (0.5f + (float)(aux >> 28)) * 0.5f;
#pragma unroll
        for (int l = 0; l < 4; l++) {
            const uint32_t s = signs8((aux >> (7 * l)) & 127u), i2 = w[l >> 1] >> (16 * (l & 1));
            // levels 4 12 20 28 36 44 52 62
            o.c[2 * l] = sign4(iq3_levels(grid[i2 & 255u], 0x3e342c24u, 0x1c140c04u), s);
            o.c[2 * l + 1] = sign4(iq3_levels(grid[(i2 >> 8) & 255u], 0x3e342c24u, 0x1c140c04u), s >> 4);
        }
    } else {
        static_assert(TYPE == QS_TYPE_IQ3_S, "format");
        uint32_t w[2];
        load_words(b + 2 + 8 * g, w);
        const uint32_t sg = load_u32(b + 74 + 4 * g), qh = b[66 + g], sc = b[106 + (g >> 1)];
        o.d[0] = load_f16(b) * (float)(1 + 2 * ((sc >> (4 * (g & 1))) & 15u));
#pragma unroll
        for (int l = 0; l < 4; l++) {
            const uint32_t s = sg >> (8 * l), i2 = w[l >> 1] >> (16 * (l & 1)), h = qh >> (2 * l);
            // levels 1 3 5 ... 15
            o.c[2 * l] = sign4(iq3_levels(grid[(i2 & 255u) | ((h & 1u) << 8)], 0x0f0d0b09u, 0x07050301u), s);
            o.c[2 * l + 1] =
                sign4(iq3_levels(grid[((i2 >> 8) & 255u) | ((h & 2u) << 7)], 0x0f0d0b09u, 0x07050301u), s >> 4);
        }
    }
}

// the group of 32 values number `gi` of a row
template <int TYPE>
QS_DEV void decode_row_group(const uint8_t* row, int gi, const uint16_t* grid, Group<TYPE>& o) {
    constexpr int PER = Format<TYPE>::BLK / 32;
    decode_group<TYPE>(row + (int64_t)(gi / PER) * Format<TYPE>::BYTES, gi % PER, grid, o);
}

}  // namespace qsd
