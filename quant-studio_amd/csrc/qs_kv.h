// The quantised key-value cache (include/quant_studio.h): its layout and what
// the kernels that write, read and attend over it share (gfx950).
//
// A page holds, for each key/value head one after another, the codes of its keys,
// the codes of its values and the steps of both (f16, one for 32 codes). They lie as
// the matrix instructions of the attention take them, so that a lane loads what it
// needs in runs of up to 16 bytes that are next to its neighbours' and never moves a
// code to another lane. Of a head of `blocks` blocks of 32 dims, dim = 32 block + ...
//   keys    a row for each slot, of units (quarter, block) of eight codes, dim
//           8 quarter + 0..7; a quarter's units of all blocks, in pieces of 16 bytes
//           (the last of 8, if need be), a piece of each quarter after another
//   values  four slots together: for each pair of dims, for each of the slots, the
//           units (pair, block) of two codes, dim 2 pair + 0..1, of all blocks
//   steps   four slots together: the keys' steps of each, then the values'
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

// a cache as the kernels see it
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

// first byte of a head in a page: its keys' codes; the values' and the steps follow
QS_DEV uint8_t* head_of(const Cache& c, int page, int head) {
    return c.data + page * c.page_bytes + (int64_t)head * (c.page * slot_bytes(c.k_bits, c.v_bits, c.blocks));
}

// Bytes in a head, of a slot of the page: a unit of eight codes of a key ...
QS_DEV int k_unit(const Cache& c, int slot, int quarter, int block) {
    const int run = c.blocks * c.k_bits, at = block * c.k_bits, piece = at & ~15;
    return slot * 4 * run + 4 * piece + quarter * (run - piece < 16 ? run - piece : 16) + (at & 15);
}
// ... a unit of two codes of a value ...
QS_DEV int v_unit(const Cache& c, int slot, int pair, int block) {
    const int run = c.blocks * c.v_bits / 4;
    return c.page * row_bytes(c.k_bits, c.blocks) + (slot >> 2) * 64 * run + (4 * pair + (slot & 3)) * run + block * c.v_bits / 4;
}
// ... the step of a block.
QS_DEV int step_at(const Cache& c, int slot, bool value, int block) {
    return c.page * (row_bytes(c.k_bits, c.blocks) + row_bytes(c.v_bits, c.blocks)) +
           2 * (((slot >> 2) * 8 + (value ? 4 : 0) + (slot & 3)) * c.blocks + block);
}

QS_DEV float half_of(uint32_t bits) { return (float)__builtin_bit_cast(_Float16, (uint16_t)bits); }

}  // namespace qskv
