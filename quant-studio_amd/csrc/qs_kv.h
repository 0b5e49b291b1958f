// The quantised key-value cache (include/quant_studio.h): its layout and what
// the kernels that write, read and attend over it share (gfx950).
//
// A page holds, for each key/value head one after another, the codes of its
// keys, their steps (f16, one for 32 codes), the codes of its values and their
// steps, each a row per slot. A row's codes are in the order in which the matrix
// instructions of the attention take them, so that no lane ever moves a code to
// another one (dim = 32 block + ...):
//   keys    unit (quarter, block) of eight codes, dim 8 quarter + 0..7:
//           lane quarter of a token reads its units of all blocks in one run
//   values  unit (pair, block) of two codes, dim 2 pair + 0..1: the sixteen
//           lanes of a product's rows read theirs of all blocks in one run
// Eight-bit codes lie as sign and magnitude: the byte beside itself, but for the
// bits between them, is then the code as a subnormal f16, which costs one
// instruction less than an offset that has to be taken off again. Four-bit codes
// lie as they are, 0..15, and what stands for 0 is 8.
#pragma once

#include "qs_device.h"
#include "quant_studio.h"

namespace qskv {

using qs::u32x2;
using qs::u32x4;

// a cache as the kernels see it; `row` of K or V: code bytes of a slot's row
struct Cache {
    uint8_t* data;
    int64_t page_bytes;
    int32_t pages, page, shift;     // shift: log2 of the page's slots
    int32_t heads, blocks;          // blocks: of 32 values in a head
    int32_t k_bits, v_bits;
};

__host__ __device__ constexpr int row_bytes(int bits, int blocks) { return 4 * bits * blocks; }
__host__ __device__ constexpr int slot_bytes(int k_bits, int v_bits, int blocks) {
    return row_bytes(k_bits, blocks) + row_bytes(v_bits, blocks) + 4 * blocks;
}

// first byte of a head's keys in a page; its key steps, values and value steps follow
QS_DEV uint8_t* head_of(const Cache& c, int page, int head) {
    return c.data + page * c.page_bytes + (int64_t)head * (c.page * slot_bytes(c.k_bits, c.v_bits, c.blocks));
}

// where a unit of eight codes of the keys' rows lies
QS_DEV int k_unit(int bits, int blocks, int quarter, int block) { return (quarter * blocks + block) * bits; }
// where a unit of two codes of the values' rows lies: bits / 4 bytes
QS_DEV int v_unit(int bits, int blocks, int pair, int block) { return (pair * blocks + block) * bits / 4; }

// the f32 value of an eight-bit code (sign and magnitude) and of a four-bit one
QS_DEV float code8(uint32_t b) {
    const float m = (float)(b & 127u);
    return b & 128u ? -m : m;
}
QS_DEV float code4(uint32_t n) { return (float)((int)(n & 15u) - 8); }

QS_DEV float half_of(uint32_t bits) { return (float)__builtin_bit_cast(_Float16, (uint16_t)bits); }

}  // namespace qskv
