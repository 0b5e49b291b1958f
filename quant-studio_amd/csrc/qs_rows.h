// Rows of f32, f16 or bf16 values, eight at a time: their values in f32 and back.
#pragma once

#include "qs_device.h"

namespace qsr {

using qs::u32x4;

// eight values of the source type in f32
template <int SRC>
struct Eight {
    u32x4 w[SRC == qs::SRC_F32 ? 2 : 1];
};
template <int SRC>
QS_DEV void load8(const void* p, int64_t at, Eight<SRC>& o) {
    const u32x4* s = reinterpret_cast<const u32x4*>(static_cast<const char*>(p) + at * (SRC == qs::SRC_F32 ? 4 : 2));
    o.w[0] = s[0];
    if constexpr (SRC == qs::SRC_F32) o.w[1] = s[1];
}
// values that are read or written once: around the caches' other contents
template <int SRC>
QS_DEV void load8_once(const void* p, int64_t at, Eight<SRC>& o) {
    const u32x4* s = reinterpret_cast<const u32x4*>(static_cast<const char*>(p) + at * (SRC == qs::SRC_F32 ? 4 : 2));
    o.w[0] = __builtin_nontemporal_load(s);
    if constexpr (SRC == qs::SRC_F32) o.w[1] = __builtin_nontemporal_load(s + 1);
}
template <int SRC>
QS_DEV float value8(const Eight<SRC>& o, int i) {
    if constexpr (SRC == qs::SRC_F32) return __uint_as_float(o.w[i >> 2][i & 3]);
    const uint32_t h = (o.w[0][i >> 1] >> (16 * (i & 1))) & 0xffffu;
    if constexpr (SRC == qs::SRC_BF16) return __uint_as_float(h << 16);
    return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
// f32 to bf16, to nearest even; a NaN stays one
QS_DEV uint32_t bf16_bits(float f) {
    return (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)f);
}
// two of them, the first in the low half: one instruction (rows of 2,560 values normalised with a
// residual, 2,048 of them 11.5 us, 11.8 with two; 64 and 16,384 of them the same with both)
QS_DEV uint32_t bf16_pair(float lo, float hi) {
    using f32x2 = float __attribute__((ext_vector_type(2)));
    using bf16x2 = __bf16 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}
template <int DST>
QS_DEV uint32_t bits16(float f) {
    if constexpr (DST == qs::SRC_BF16) return bf16_bits(f);
    // the f32 result is rounded again, as torch's is: the compiler would
    // otherwise form it and the f16 in one mixed-precision instruction
    qs::keep_in_register(f);
    return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f);
}
template <int DST, bool ONCE = false>
QS_DEV void store8(void* p, int64_t at, const float (&v)[8]) {
    u32x4* d = reinterpret_cast<u32x4*>(static_cast<char*>(p) + at * (DST == qs::SRC_F32 ? 4 : 2));
    const auto put = [&](int i, const u32x4& o) {
        if constexpr (ONCE) __builtin_nontemporal_store(o, d + i);
        else d[i] = o;
    };
    if constexpr (DST == qs::SRC_F32) {
        put(0, u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])});
        put(1, u32x4{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])});
    } else {
        u32x4 o;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            if constexpr (DST == qs::SRC_BF16) o[i] = bf16_pair(v[2 * i], v[2 * i + 1]);
            else o[i] = bits16<DST>(v[2 * i]) | (bits16<DST>(v[2 * i + 1]) << 16);
        }
        put(0, o);
    }
}

}  // namespace qsr
