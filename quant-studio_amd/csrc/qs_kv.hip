// Rows of keys and values quantised into a cache's pages and read back
// (declarations: include/quant_studio.h; the layout: qs_kv.h).
#include <hip/hip_runtime.h>

#include <type_traits>

#include "qs_host.h"
#include "qs_kernels.h"
#include "qs_kv.h"
#include "qs_kv_attention.h"
#include "qs_launch_kernel.h"
#include "qs_rows.h"

namespace {

using namespace qsr;
using qs_host::fail;
using qskv::Cache;

struct RowsArgs {
    Cache c;
    void *k, *v;                    // rows of heads x 32 blocks values
    int64_t k_stride, v_stride;     // between rows, in values
    const int32_t* slots;
    int32_t rows, units;            // units: of eight values in a row's keys and values
    int32_t group;                  // rows of a workgroup at a time
    int32_t wide, together;         // threads on a row, rows at a time
    uint32_t per_wide, per_block;   // 2^20 / wide and 2^18 / blocks, rounded up: threads and units divide by them
};

// the eight values of a thread: a quarter of a block, keys or values
struct Unit {
    int head, block, quarter, bits;
    bool value;
    int codes, step;            // bytes in a page of the first slot's: its codes, its step
    int four, one, step_four;   // bytes to the slot four on, to the next of four
    int pair;                   // values: bytes between its four units of two codes
};
QS_DEV Unit unit_of(const RowsArgs& a, uint32_t u) {
    const Cache& c = a.c;
    const uint32_t blocks = (uint32_t)c.blocks, of_keys = __umul24(4 * blocks, c.heads);
    Unit o;
    o.value = u >= of_keys;
    u -= o.value ? of_keys : 0;
    o.quarter = (int)(u & 3);
    o.head = (int)(__umul24(u >> 2, a.per_block) >> 18);
    o.block = (int)((u >> 2) - __umul24(o.head, blocks));
    o.bits = o.value ? c.v_bits : c.k_bits;
    const uint32_t head = __umul24(o.head, c.page * qskv::slot_bytes(c.k_bits, c.v_bits, c.blocks));
    // the layout's distances: a slot's keys take 4 runs and its values one of a quarter of theirs
    const uint32_t run = __umul24(blocks, o.bits);
    o.codes = (int)head + (o.value ? qskv::v_unit(c, 0, 4 * o.quarter, o.block) : qskv::k_unit(c, 0, o.quarter, o.block));
    o.four = 16 * run;
    o.one = o.value ? run >> 2 : 4 * run;
    o.pair = (int)run;
    o.step = (int)head + qskv::step_at(c, 0, o.value, o.block);
    o.step_four = 16 * blocks;
    return o;
}
// The rows of keys or of values. Both are read first: the compiler would choose
// between their addresses, and load what it chose with a wait of its own.
struct Side {
    void* data;
    int64_t stride;
};
QS_DEV Side side_of(const RowsArgs& a, bool value) {
    using Global = __attribute__((address_space(1))) void*;
    Global k = (Global)a.k, v = (Global)a.v;
    int64_t k_stride = a.k_stride, v_stride = a.v_stride;
    asm("" : "+s"(k), "+s"(v), "+s"(k_stride), "+s"(v_stride));
    return {(void*)(value ? v : k), value ? v_stride : k_stride};
}
// where the unit of a slot has its codes and its step
struct Place {
    uint8_t *codes, *step;
};
QS_DEV Place place_of(const Cache& c, const Unit& u, int slot) {
    uint8_t* page = c.data + (uint64_t)(uint32_t)(slot >> c.shift) * (uint32_t)c.page_bytes;
    const uint32_t in = (uint32_t)slot & (uint32_t)(c.page - 1), fours = in >> 2, rest = in & 3;
    return {page + (u.codes + __umul24(fours, u.four) + __umul24(rest, u.one)),
            page + (u.step + __umul24(fours, u.step_four) + __umul24(rest, 2 * c.blocks))};
}

// How threads are laid over rows: `wide` of them (whole heads' keys or values, so at
// most all and a multiple of a head's units) on one row, `together` rows at a time,
// BATCH times over.
constexpr int BATCH = 4;
// Calls of no more rows, and no more workgroups than the GPU holds at a time, take one row
// at a time: 1,000 rows of eight heads of 128 read in 4.2 us, 4.4 in batches; 4,000 of one
// head 3.6 and 4.4; but 2,100 of eight heads 6.1 and 5.1.
constexpr int FEW_ROWS = 4096, HELD = 2048;
// Rows of a launch that writes: what a workgroup looks its slots up among, a turn of four for
// each thread. Twice as many are better for narrow rows and worse for wide ones, which have
// more threads that look: 65,535 rows of one head of 64, written and read back, 101 us, 121
// with 4,096 and 76 with 16,384; 8,191 of eight heads of 128 30.1, 34.3 and 33.0, 32,767
// 119, 128 and 122.
constexpr int64_t MOST_ROWS = 8192;
constexpr int WRITERS = 512;      // threads of a workgroup that writes many rows
struct Shape {
    int wide, together, columns;    // columns: workgroups for a row
};
__host__ __device__ inline Shape shape_of(int units, int blocks, int threads) {
    const int most = threads / (4 * blocks) * (4 * blocks);
    Shape s;
    s.wide = units < most ? units : most;
    s.together = threads / s.wide;
    s.columns = (units + s.wide - 1) / s.wide;
    return s;
}

// a byte of a word from the whole part of f: 0 of a negative one and of NaN, 255 above
template <int AT>
QS_DEV uint32_t byte_of(float f, uint32_t w) {
    return __builtin_amdgcn_cvt_pk_u8_f32(__builtin_truncf(f), AT, w);
}
// 1 / d of a step that f16 holds, correctly rounded: one step of Newton's method on the
// hardware's reciprocal, which is as good from 2^-60 to 2^60 (every f32 of them compared
// with the division, which takes twice the instructions). The codes of smaller steps
// stand for zeros, those of larger ones for no values, whatever they are.
QS_DEV float inverse_of(float d) {
    const float y = __builtin_amdgcn_rcpf(d);
    return __builtin_fmaf(__builtin_fmaf(-d, y, 1.0f), y, y);
}
// m / 127, correctly rounded (compared likewise): the product with 1 / 127 and what it is off by
QS_DEV float of_127(float m) {
    const float q = m * (1.0f / 127.0f);
    return __builtin_fmaf(__builtin_fmaf(-127.0f, q, m), 1.0f / 127.0f, q);
}

// largest magnitude of a block as f32 bits, a NaN above all
template <int SRC>
QS_DEV float top_of(const Eight<SRC>& in, const float (&x)[8]) {
    uint32_t m;
    if constexpr (SRC == qs::SRC_F32) {
        m = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
    } else {
        // the order of the 16-bit types' magnitudes is that of their bits
        using u16x2 = uint16_t __attribute__((ext_vector_type(2)));
        u16x2 h = __builtin_bit_cast(u16x2, in.w[0][0] & 0x7fff7fffu);
#pragma unroll
        for (int j = 1; j < 4; j++) h = __builtin_elementwise_max(h, __builtin_bit_cast(u16x2, in.w[0][j] & 0x7fff7fffu));
        m = max((uint32_t)h[0], (uint32_t)h[1]);
    }
    m = max(m, qs::quad_xor<1>(m));
    m = max(m, qs::quad_xor<2>(m));
    if constexpr (SRC == qs::SRC_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)m);
    return __uint_as_float(SRC == qs::SRC_BF16 ? m << 16 : m);
}
// the value of the largest magnitude, the first of them, a NaN above all
template <int SRC>
QS_DEV float peak_of(const float (&x)[8], int quarter) {
    if constexpr (SRC == qs::SRC_F32) return qs::quad_absmax_first(x, quarter);
    // The f32 bits of 16-bit types end in 13 zeros at least: turned left by one, the
    // sign is last, and between it and the magnitude is room for the place, first ones above.
    const uint32_t place = (uint32_t)(31 - 8 * quarter) << 1;
    uint32_t key = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const uint32_t b = __float_as_uint(x[j]);
        key = max(key, __builtin_rotateleft32(b, 1) | (place - 2 * j));
    }
    key = max(key, qs::quad_xor<1>(key));
    key = max(key, qs::quad_xor<2>(key));
    return __uint_as_float(__builtin_rotateright32(key & ~0x3eu, 1));
}

// Codes of eight values as the cache holds them, and their block's step, which four
// threads find together: eight bits as two words of four codes each; four bits as a
// word of four pairs, a key's (0, 2) (4, 6) (1, 3) (5, 7), a value's (0, 1) (2, 3) ...
// The steps and roundings are those of the quantizers' b32_block, in other instructions; the
// tests compare them bit for bit, at ties too.
template <int SRC>
QS_DEV float codes_of(const Eight<SRC>& in, const Unit& u, uint32_t (&code)[2]) {
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = value8<SRC>(in, j);
    if (u.bits == 8) {
        const float d = of_127(top_of<SRC>(in, x)), id = inverse_of(d);
        // Half away from zero, of the magnitude: m + the largest f32 below 0.5 passes a
        // whole number exactly where m + 0.5 does (m + 0.5 itself would also take 0.5's
        // predecessor to 1). Over 127 only where the codes do not matter.
        const auto four = [&](int j) {
            const auto of = [&](int e) { return fabsf(x[j + e] * id) + 0x1.fffffep-2f; };
            const uint32_t w = byte_of<3>(of(3), byte_of<2>(of(2), byte_of<1>(of(1), byte_of<0>(of(0), 0))));
            const auto high = [&](int e) { return __float_as_uint(x[j + e]); };
            const uint32_t low2 = __builtin_amdgcn_perm(high(1), high(0), 0x0c0c0703u);
            const uint32_t signs = __builtin_amdgcn_perm(high(3), high(2), 0x07030c0cu) | low2;
            return w | (signs & 0x80808080u);
        };
        code[0] = four(0);
        code[1] = four(4);
        return d;
    }
    const float d = peak_of<SRC>(x, u.quarter) * -0.125f, id = inverse_of(d);
    const auto level = [&](int j) { return fminf(x[j] * id + 8.5f, 15.5f); };
    uint32_t low, high;
    if (u.value) {
        low = byte_of<3>(level(6), byte_of<2>(level(4), byte_of<1>(level(2), byte_of<0>(level(0), 0))));
        high = byte_of<3>(level(7), byte_of<2>(level(5), byte_of<1>(level(3), byte_of<0>(level(1), 0))));
    } else {
        low = byte_of<3>(level(5), byte_of<2>(level(1), byte_of<1>(level(4), byte_of<0>(level(0), 0))));
        high = byte_of<3>(level(7), byte_of<2>(level(3), byte_of<1>(level(6), byte_of<0>(level(2), 0))));
    }
    code[0] = low | high << 4;
    return d;
}

// A thread takes eight values, four threads a block of 32: its step from their
// largest magnitude, then eight codes each, in the order of the cache's rows.
// Of rows with the same slot the last is written: every workgroup looks all later
// slots up in a table of its own rows' (16,383 rows of one head of 64 in any order, written
// and read back, take 27.6 us; 82 with every own slot compared with every later one). With
// MANY rows a workgroup has WRITERS threads, which share that work among more rows: 8,191
// rows of eight heads of 128 in any order, written and read back, take 29.9 us, 35.4 with
// 256 threads, 29.4 with 1,024; 1,025 rows 10.2, 9.9 and 12.0.
//
// 8,191 such rows in order, bf16 to keys of 8 and values of 4 bits, are 47 MB and take
// 15 us, 3.1 TB/s; a copy of as many bytes takes 11.3. All rows are on their way at once,
// so that reading, 600 instructions a wave for the codes (2.5 us of it) and the
// scattered stores (5 us of it) overlap little. Staging the values' codes in LDS for wide stores
// took 1.4 us more, a row or two at a time instead of BATCH 0.4 to 8 us more.
template <int SRC, bool MANY>
__global__ __launch_bounds__(MANY ? WRITERS : 256) void k_kv_write(RowsArgs a) {
    constexpr int THREADS = MANY ? WRITERS : 256, TIMES = MANY ? BATCH : 1;
    constexpr int TURN = 4 * THREADS, TURNS = MANY ? (int)(MOST_ROWS / TURN) : FEW_ROWS / TURN;
    constexpr int MOST_GROUP = TIMES * THREADS / 16;       // a row has 16 units at least
    __shared__ __attribute__((aligned(16))) int mine[MOST_GROUP];
    __shared__ int replaced[MOST_GROUP], chain[MOST_GROUP], heads[THREADS];
    const int first = (int)blockIdx.x * a.group;
    const int count = a.rows - first < a.group ? a.rows - first : a.group;
    const int slots = a.c.pages << a.c.shift;
    const int sub = (int)(__umul24(threadIdx.x, a.per_wide) >> 20);
    const int at = (int)blockIdx.y * a.wide + ((int)threadIdx.x - (int)__umul24(sub, a.wide));
    const bool live = sub < a.together && at < a.units;
    const Unit u = unit_of(a, live ? at : 0);
    const Side src = side_of(a, u.value);
    const int64_t from = first * src.stride + (__umul24(u.head, 32 * a.c.blocks) + 32 * u.block + 8 * u.quarter);
    // unsigned: behind the last row, where nothing is read, it may pass 2^63
    const uint64_t next = (uint64_t)src.stride * a.together;
    uint64_t from_row = from + (uint64_t)src.stride * sub;
    // The slots of the workgroup's rows and of all later ones, which a launch has few
    // enough of for four turns, then the rows' values: all are on their way before
    // anything waits, and the slots are looked up meanwhile.
    const int s0 = (int)threadIdx.x < count ? a.slots[first + threadIdx.x] : -1;
    int later[TURNS][4];
#pragma unroll
    for (int j = 0; j < TURNS; j++) {
#pragma unroll
        for (int e = 0; e < 4; e++) later[j][e] = -1;
        if (first + count + TURN * j >= a.rows) continue;       // the same for all
        const int r = first + count + TURN * j + 4 * (int)threadIdx.x;
        if (r + 3 < a.rows) __builtin_memcpy(later[j], a.slots + r, 16);
        else
#pragma unroll
            for (int e = 0; e < 3; e++)
                if (r + e < a.rows) later[j][e] = a.slots[r + e];
    }
    Eight<SRC> in[TIMES];
#pragma unroll
    for (int i = 0; i < TIMES; i++) {
        const int row = sub + i * a.together;
        // others' rows are the first one's, so that no load waits in a branch
        load8_once<SRC>(src.data, live && row < count ? (int64_t)from_row : from, in[i]);
        from_row += next;
    }
    // The workgroup's rows by their slots: chains from a table of as many heads as threads.
    const auto place_in = [&](int slot) { return ((uint32_t)slot * 0x9e3779b1u) / (0x80000000u / THREADS * 2); };
    const bool held = (unsigned)s0 < (unsigned)slots;
    heads[threadIdx.x] = -1;
    if ((int)threadIdx.x < MOST_GROUP) {
        mine[threadIdx.x] = held ? s0 : -1;
        replaced[threadIdx.x] = 0;
    }
    __syncthreads();
    if (a.rows - first > 1) {
        if (held) chain[threadIdx.x] = atomicExch(&heads[place_in(s0)], (int)threadIdx.x);
        // most often the later slots are all outside the range of the workgroup's own
        uint32_t low = ~0u, high = 0, near = ~0u;
        for (int i = 0; i < count; i += 4) {
            const int4 m = *reinterpret_cast<const int4*>(mine + i);
            low = min(min(min(low, (uint32_t)m.x), min((uint32_t)m.y, (uint32_t)m.z)), (uint32_t)m.w);
            high = (uint32_t)max(max(max((int)high, m.x), max(m.y, m.z)), m.w);
        }
        __syncthreads();
        // a row's slot is in a later one: of the workgroup's own, or behind them
        const auto look_up = [&](int slot, int before) {
            for (int i = heads[place_in(slot)]; i >= 0; i = chain[i])
                if (i < before && mine[i] == slot) replaced[i] = 1;
        };
        if (held) look_up(s0, (int)threadIdx.x);
#pragma unroll
        for (int j = 0; j < TURNS; j++) {
            if (first + count + TURN * j >= a.rows) break;
#pragma unroll
            for (int e = 0; e < 4; e++) near = min(near, (uint32_t)later[j][e] - low);
        }
        if (near <= high - low) {
#pragma unroll
            for (int j = 0; j < TURNS; j++) {
                if (first + count + TURN * j >= a.rows) break;
#pragma unroll
                for (int e = 0; e < 4; e++) look_up(later[j][e], count);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < TIMES; i++) {
        const int row = sub + i * a.together;
        const int slot = live && row < count && !replaced[row] ? mine[row] : -1;
        if (slot < 0) continue;     // the same for the four threads of a block
        uint32_t code[2];
        const float d = codes_of<SRC>(in[i], u, code);
        const Place p = place_of(a.c, u, slot);
        // a step that f16 cannot hold, like a NaN or an infinity in the block, stands for no values
        const uint32_t h = qs::f16_bits(d);
        if (u.quarter == 0) *reinterpret_cast<uint16_t*>(p.step) = (uint16_t)((h & 0x7fffu) < 0x7c00u ? h : 0x7e00u);
        if (!u.value) {
            if (u.bits == 8) *reinterpret_cast<uint2*>(p.codes) = uint2{code[0], code[1]};
            else *reinterpret_cast<uint32_t*>(p.codes) = code[0];
        } else if (u.bits == 8) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                *reinterpret_cast<uint16_t*>(p.codes + j * u.pair) = (uint16_t)(code[j >> 1] >> (16 * (j & 1)));
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) p.codes[j * u.pair] = (uint8_t)(code[0] >> (8 * j));
        }
    }
}

// The values of some slots' rows; a slot outside the cache gives zeros. Eight to a
// thread, of BATCH rows at a time, whose loads are all on their way before the first
// is waited for. Bound by HBM: 65,535 rows of eight heads of 128, 8 bits to bf16, 411 MB,
// take 78.6 us, 5.2 TB/s, as fast as a large copy.
template <int DST, bool MANY>
__global__ __launch_bounds__(256) void k_kv_read(RowsArgs a) {
    constexpr int TIMES = MANY ? BATCH : 1;
    const int slots = a.c.pages << a.c.shift;
    const int sub = (int)(__umul24(threadIdx.x, a.per_wide) >> 20);
    const int at = (int)blockIdx.y * a.wide + ((int)threadIdx.x - (int)__umul24(sub, a.wide));
    if (sub >= a.together || at >= a.units) return;
    const Unit u = unit_of(a, at);
    const Side dst = side_of(a, u.value);
    const int first = (int)blockIdx.x * a.group;
    const int64_t next = a.together * dst.stride;
    int64_t to = (first + sub) * dst.stride + (__umul24(u.head, 32 * a.c.blocks) + 32 * u.block + 8 * u.quarter);
    const int count = a.rows - first < a.group ? a.rows - first : a.group;
    int slot[TIMES];
#pragma unroll
    for (int i = 0; i < TIMES; i++) {
        const int row = sub + i * a.together;
        slot[i] = a.slots[first + (row < count ? row : 0)];
    }
    uint32_t w[TIMES][4];       // keys: their words; values: a unit each
    uint16_t step[TIMES];
    const uint8_t* codes[TIMES];
#pragma unroll
    for (int i = 0; i < TIMES; i++) {
        // a slot outside is read as the first, and its step as 0
        const Place p = place_of(a.c, u, (unsigned)slot[i] < (unsigned)slots ? slot[i] : 0);
        step[i] = *reinterpret_cast<const uint16_t*>(p.step);
        codes[i] = p.codes;
    }
    // one branch around all rows' loads: none waits for another
    if (u.value && u.bits == 8) {
#pragma unroll
        for (int i = 0; i < TIMES; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) w[i][j] = *reinterpret_cast<const uint16_t*>(codes[i] + j * u.pair);
    } else if (u.value) {
#pragma unroll
        for (int i = 0; i < TIMES; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) w[i][j] = codes[i][j * u.pair];
    } else if (u.bits == 8) {
#pragma unroll
        for (int i = 0; i < TIMES; i++) {
            const uint2 c = *reinterpret_cast<const uint2*>(codes[i]);
            w[i][0] = c.x, w[i][1] = c.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < TIMES; i++) w[i][0] = *reinterpret_cast<const uint32_t*>(codes[i]);
    }
#pragma unroll
    for (int i = 0; i < TIMES; i++) {
        const int row = sub + i * a.together;
        if (row >= count) break;
        // Codes go through f16 two at a time, as subnormals c 2^-24, and c d is exact in
        // f32: a magnitude of 7 bits times a step of 11.
        const float d = (unsigned)slot[i] < (unsigned)slots ? qskv::half_of(step[i]) : 0.0f, large = d * 0x1p24f;
        const float less = u.bits == 8 ? 0.0f : -8.0f * d;
        float x[8];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            uint32_t two;
            if (u.bits == 8) {
                const uint32_t c = u.value ? w[i][j] : w[i][j >> 1];
                two = __builtin_amdgcn_perm(0, c, u.value || j % 2 == 0 ? 0x01010000u : 0x03030202u) & 0x807f807fu;
            } else {
                two = (u.value ? w[i][j] | w[i][j] << 12 : w[i][0] >> (4 * j)) & 0x000f000fu;
            }
            using f16x2 = _Float16 __attribute__((ext_vector_type(2)));
            const f16x2 h = __builtin_bit_cast(f16x2, two);
            x[2 * j] = __builtin_fmaf((float)h[0], large, less);
            x[2 * j + 1] = __builtin_fmaf((float)h[1], large, less);
        }
        store8<DST, true>(dst.data, to, x);
        to += next;
    }
}

template <typename F>
hipError_t launch_rows(const RowsArgs& all, int64_t most, int threads, int esz, F&& few, F&& many, hipStream_t st) {
    for (int64_t first = 0; first < all.rows; first += most) {
        RowsArgs a = all;
        a.rows = (int32_t)(all.rows - first < most ? all.rows - first : most);
        a.k = static_cast<char*>(all.k) + first * all.k_stride * esz;
        a.v = static_cast<char*>(all.v) + first * all.v_stride * esz;
        a.slots = all.slots + first;
        Shape shape = shape_of(all.units, all.c.blocks, 256);
        const bool much = a.rows > FEW_ROWS || (int64_t)a.rows * shape.columns > HELD * shape.together;
        if (much) shape = shape_of(all.units, all.c.blocks, threads);
        a.group = shape.together * (much ? BATCH : 1);
        a.wide = shape.wide;
        a.together = shape.together;
        a.per_wide = (uint32_t)(((1 << 20) + shape.wide - 1) / shape.wide);
        a.per_block = (uint32_t)(((1 << 18) + a.c.blocks - 1) / a.c.blocks);
        const dim3 grid((unsigned)((a.rows + a.group - 1) / a.group), (unsigned)shape.columns);
        const hipError_t e = qs_host::launch_kernel(much ? many : few, grid, dim3(much ? threads : 256), 0, st, a);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

constexpr int64_t kMaxRows = INT64_C(1) << 24, kMaxBatch = INT64_C(1) << 14, kMaxSpan = INT64_C(1) << 62;
bool off16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 != 0; }
bool off4(const void* p) { return reinterpret_cast<uintptr_t>(p) % 4 != 0; }
int bits_of(int type) { return type == QS_TYPE_Q8_0 ? 8 : type == QS_TYPE_Q4_0 ? 4 : 0; }
int size_of(int src) { return src == QS_SRC_F32 ? 4 : (src == QS_SRC_F16 || src == QS_SRC_BF16) ? 2 : 0; }

int bad_layout(int k_type, int v_type, int heads, int head_dim, int page_size) {
    if (!bits_of(k_type) || !bits_of(v_type))
        return fail(QS_ENOTSUP, "cache types %d and %d: Q8_0 (8) or Q4_0 (2)", k_type, v_type);
    if (heads < 1 || heads > 1024) return fail(QS_EINVAL, "%d heads, not 1..1024", heads);
    if (head_dim < 64 || head_dim > 256 || head_dim % 64)
        return fail(QS_EINVAL, "head size %d is not 64, 128, 192 or 256", head_dim);
    if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)))
        return fail(QS_EINVAL, "page of %d slots: not a power of two in 16..1024", page_size);
    return 0;
}

int attention_sizes(const qs_kv_cache* cache, int64_t batch, int64_t fresh, int64_t query_heads, int64_t pages_each,
                    qskv::AttentionArgs& a) {
    const int bad = qskv::cache_of(cache, a.c);
    if (bad) return bad;
    if (batch < 0 || batch > kMaxBatch) return fail(QS_EINVAL, "%lld sequences: negative, or over 2^14", (long long)batch);
    if (fresh < 0 || fresh > 16) return fail(QS_EINVAL, "%lld new tokens of a sequence: not 0..16", (long long)fresh);
    if (query_heads < 1 || query_heads % a.c.heads || query_heads / a.c.heads > 128)
        return fail(QS_EINVAL, "%lld query heads: not 1 to 128 for each of %d key/value heads", (long long)query_heads, a.c.heads);
    if (pages_each < 0 || pages_each > (INT32_C(1) << 30) / a.c.page)
        return fail(QS_EINVAL, "tables of %lld pages of %d slots: negative, or over 2^30 slots", (long long)pages_each, a.c.page);
    if (batch * pages_each * a.c.page > INT64_C(1) << 34)
        return fail(QS_EINVAL, "%lld tables of %lld pages of %d slots: over 2^34 slots", (long long)batch, (long long)pages_each, a.c.page);
    // workgroups may be as many: a launch has under 2^32 threads
    if (batch * a.c.heads * ((query_heads / a.c.heads * fresh + 7) / 8) > INT64_C(1) << 25)
        return fail(QS_EINVAL, "%lld sequences of %d heads with %lld queries each: over 2^25 eights of queries", (long long)batch,
                    a.c.heads, (long long)(query_heads / a.c.heads * fresh));
    a.batch = (int32_t)batch;
    a.fresh = (int32_t)fresh;
    a.group = (int32_t)(query_heads / a.c.heads);
    a.pages_each = (int32_t)pages_each;
    return 0;
}

}  // namespace

namespace qskv {

static int64_t round_up(int64_t n, int64_t to) { return (n + to - 1) / to * to; }

extern template hipError_t launch_attention<8, 8>(const AttentionArgs&, const Split&, hipStream_t);
extern template hipError_t launch_attention<8, 4>(const AttentionArgs&, const Split&, hipStream_t);
extern template hipError_t launch_attention<4, 8>(const AttentionArgs&, const Split&, hipStream_t);
extern template hipError_t launch_attention<4, 4>(const AttentionArgs&, const Split&, hipStream_t);

int cache_of(const qs_kv_cache* cache, Cache& c) {
    if (!cache) return fail(QS_EINVAL, "null cache");
    const int bad = bad_layout(cache->k_type, cache->v_type, cache->heads, cache->head_dim, cache->page_size);
    if (bad) return bad;
    if (cache->pages < 1 || cache->pages > INT32_MAX / cache->page_size)
        return fail(QS_EINVAL, "%d pages of %d slots: none, or over 2^31 - 1 slots", cache->pages, cache->page_size);
    if (!cache->data || off16(cache->data)) return fail(QS_EINVAL, "cache data %p is null or not 16-byte aligned", cache->data);
    c.data = static_cast<uint8_t*>(cache->data);
    c.pages = cache->pages;
    c.page = cache->page_size;
    c.shift = __builtin_ctz(cache->page_size);
    c.heads = cache->heads;
    c.blocks = cache->head_dim / 32;
    c.k_bits = bits_of(cache->k_type);
    c.v_bits = bits_of(cache->v_type);
    c.page_bytes = (int64_t)c.page * c.heads * slot_bytes(c.k_bits, c.v_bits, c.blocks);
    return 0;
}

Split split_of(const AttentionArgs& a, void* workspace) {
    // As many workgroups of four waves as the GPU holds at a time, unless even the
    // longest sequences would not give each a step for every wave.
    //
    // Sequences of `whole` steps at most are not split: one segment to a workgroup, so that
    // nothing is joined. Of 8 heads of 128 in 8 bits: 8 sequences of 600 slots take 13.0 us,
    // 13.9 split, 40 take 19.9, 25.0 split, 150 take 45.4, 56.8 split (ragged ones 28.2, 36.7
    // split); but 8 of 900 slots 17.3 and 16.3, ragged ones 16.4 and 13.4. A lone one of
    // 290 slots takes 9.0, 9.1 split, of 420 slots 10.7 and 9.4. Longer ones are whole where
    // there are so many that the longest cannot take much longer than all together: 40 of 900
    // slots 25.5, 29.4 split (ragged ones 18.4, 21.6 split), 150 of 1,500 slots 97 and 111
    // (ragged 49 and 54), 600 of 1,200 slots 304 and 347; 65 ragged ones of 1,300 30.8 and
    // 29.4. Up to twice `whole` for workgroups of four waves, since lengths may be far below
    // the tables' width but for a few: 190 of 3,000 slots are 257 us split, 244 whole, but
    // ragged ones 99 and 107, and one such with 189 of 17 slots 32 and 40 (39 of 17 slots and
    // one of 900: 12.5, 16.2 whole).
    //
    // A lone sequence is in equal parts, which each workgroup knows before it knows the
    // length; more of them are in equal runs of all their steps, since the longest may be of
    // any share.
    //
    // Where there are more segments than workgroups, waves take them by themselves: opening
    // one is most of what a short one takes (700 ragged sequences of 250 slots: 49.3 us, 65.9
    // with four waves to each; 8 of 500 slots, with fewer: 27.4, and 11.4 with four). Those of
    // more than FEW steps only where every wave has one (700 ragged ones of 500 slots: 78.9,
    // 85.2 with four; 200: 40.3, and 32.4 with four); in tables wider than `whole`, where most
    // may be short all the same, with half as many, in runs (300 of 17 slots in tables for
    // 3,000: 20 us, with four waves 32 in runs and 25 whole, and where one has 3,000 23, 39 and
    // 46; ragged ones up to tables of 1,200: 77, 81 and 70).
    constexpr int64_t CUS = 256, FEW = 8;
    const int64_t whole = a.batch > 1 ? 24 : 12;
    const int64_t steps = ((int64_t)a.pages_each * a.c.page + TILE - 1) / TILE;
    const int64_t segments = (int64_t)a.batch * a.c.heads * column_tiles(a);
    const int64_t full = CUS * resident(a.c.blocks, columns_of(a), a.type == QS_SRC_F32);
    Split s{};
    if (a.batch == 0 || a.fresh == 0) return s;
    s.waves = segments > (steps <= FEW ? 1 : steps <= whole ? 4 : 2) * full && a.batch > 1 ? 1 : 4;
    // Where loads are all that bounds it, eight-bit codes of heads of 128 or 256 for eight
    // 16-bit queries, one workgroup less on each CU streams better: 8 sequences of 32,767
    // slots 116.2 and 118.1 us, of heads of 256 and 16,000 slots 121 and 129; four-bit ones
    // of 128 take 48.0, 45.3 with all, heads of 64 with 8 bits 38.0 and 39.0.
    const bool lean = s.waves == 4 && a.c.k_bits + a.c.v_bits == 16 && a.c.blocks % 4 == 0 && columns_of(a) == 8 &&
                      a.type != QS_SRC_F32;
    const int64_t held = s.waves == 4 ? full - lean * CUS : 4 * full;
    const int64_t more = whole * segments / held;
    if (steps <= whole + (a.batch == 1 ? 0 : s.waves == 4 ? (more < whole ? more : whole) : segments < held ? 0 : more)) {
        s.share = 1;
    } else if (a.batch == 1) {
        const int64_t share = held / segments, most = (steps + s.waves - 1) / s.waves;
        s.share = (int32_t)(share < 1 ? 1 : share < most ? share : most);
    }
    const int64_t most = segments * (steps / s.waves + 1 + OPENING);
    s.groups = (int32_t)(s.share ? segments * s.share : most < held ? most : held);
    if (s.share == 1) return s;
    const int64_t parts = round_up((int64_t)s.groups * 2 * columns_of(a) * 32 * a.c.blocks * 4, 256);
    const int64_t stats = round_up((int64_t)s.groups * 2 * columns_of(a) * 8, 256);
    uint8_t* base = static_cast<uint8_t*>(workspace);
    s.parts = reinterpret_cast<float*>(base);
    s.stats = reinterpret_cast<float2*>(base + parts);
    s.segments = reinterpret_cast<int4*>(base + parts + stats);
    s.listed = (int32_t)(segments <= s.groups ? segments : 0);
    s.bytes = parts + stats + (int64_t)s.groups * 16;
    return s;
}

}  // namespace qskv

extern "C" {

int64_t qs_kv_page_bytes(int k_type, int v_type, int heads, int head_dim, int page_size) {
    qs_host::clear_error();
    const int bad = bad_layout(k_type, v_type, heads, head_dim, page_size);
    if (bad) return bad;
    return (int64_t)page_size * heads * qskv::slot_bytes(bits_of(k_type), bits_of(v_type), head_dim / 32);
}

int qs_kv_write(const qs_kv_cache* cache, int src_type, const void* k, int64_t k_row_stride_bytes, const void* v,
                int64_t v_row_stride_bytes, const int32_t* slots, int64_t rows, void* hip_stream) {
    qs_host::clear_error();
    RowsArgs a{};
    const int bad = qskv::cache_of(cache, a.c);
    if (bad) return bad;
    const int esz = size_of(src_type);
    if (!esz) return fail(QS_EINVAL, "unsupported source type %d (F32=0, F16=1, BF16=30)", src_type);
    if (rows < 0 || rows > kMaxRows) return fail(QS_EINVAL, "%lld rows: negative, or over 2^24", (long long)rows);
    if (rows == 0) return 0;
    if (!k || !v || !slots) return fail(QS_EINVAL, "null k, v or slots");
    if (off16(k) || off16(v) || off4(slots)) return fail(QS_EINVAL, "k and v must be 16-byte aligned, slots 4-byte");
    const int64_t width = (int64_t)a.c.heads * 32 * a.c.blocks * esz;
    for (int64_t s : {k_row_stride_bytes, v_row_stride_bytes})
        if ((s < width && rows > 1) || s < 0 || s % 16 || s > kMaxSpan / rows)
            return fail(QS_EINVAL, "row stride %lld must be >= %lld, a multiple of 16 and in a 2^62-byte span", (long long)s,
                        (long long)width);
    a.k = const_cast<void*>(k);
    a.v = const_cast<void*>(v);
    a.k_stride = k_row_stride_bytes / esz;
    a.v_stride = v_row_stride_bytes / esz;
    a.slots = slots;
    a.rows = (int32_t)rows;
    a.units = 8 * a.c.heads * a.c.blocks;
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const auto launch = [&](auto type) {
        constexpr int T = decltype(type)::value;
        return launch_rows(a, MOST_ROWS, WRITERS, esz, k_kv_write<T, false>, k_kv_write<T, true>, st);
    };
    const hipError_t e = src_type == QS_SRC_F32   ? launch(std::integral_constant<int, qs::SRC_F32>{})
                         : src_type == QS_SRC_F16 ? launch(std::integral_constant<int, qs::SRC_F16>{})
                                                  : launch(std::integral_constant<int, qs::SRC_BF16>{});
    if (e != hipSuccess) return fail(QS_EIO, "kv_write: launch failed: %s", hipGetErrorString(e));
    return 0;
}

int qs_kv_read(const qs_kv_cache* cache, const int32_t* slots, int64_t rows, int dst_type, void* k, void* v,
               void* hip_stream) {
    qs_host::clear_error();
    RowsArgs a{};
    const int bad = qskv::cache_of(cache, a.c);
    if (bad) return bad;
    const int esz = size_of(dst_type);
    if (!esz) return fail(QS_EINVAL, "unsupported destination type %d (F32=0, F16=1, BF16=30)", dst_type);
    if (rows < 0 || rows > kMaxRows) return fail(QS_EINVAL, "%lld rows: negative, or over 2^24", (long long)rows);
    if (rows == 0) return 0;
    if (!k || !v || !slots) return fail(QS_EINVAL, "null k, v or slots");
    if (off16(k) || off16(v) || off4(slots)) return fail(QS_EINVAL, "k and v must be 16-byte aligned, slots 4-byte");
    a.k = k;
    a.v = v;
    a.k_stride = a.v_stride = (int64_t)a.c.heads * 32 * a.c.blocks;
    a.slots = slots;
    a.rows = (int32_t)rows;
    a.units = 8 * a.c.heads * a.c.blocks;
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const auto launch = [&](auto type) {
        constexpr int T = decltype(type)::value;
        return launch_rows(a, kMaxRows, 256, esz, k_kv_read<T, false>, k_kv_read<T, true>, st);
    };
    const hipError_t e = dst_type == QS_SRC_F32   ? launch(std::integral_constant<int, qs::SRC_F32>{})
                         : dst_type == QS_SRC_F16 ? launch(std::integral_constant<int, qs::SRC_F16>{})
                                                  : launch(std::integral_constant<int, qs::SRC_BF16>{});
    if (e != hipSuccess) return fail(QS_EIO, "kv_read: launch failed: %s", hipGetErrorString(e));
    return 0;
}

int64_t qs_kv_attention_workspace(const qs_kv_cache* cache, int64_t batch, int64_t new_tokens, int64_t query_heads,
                                  int64_t pages_each) {
    qs_host::clear_error();
    qskv::AttentionArgs a{};
    const int bad = attention_sizes(cache, batch, new_tokens, query_heads, pages_each, a);
    if (bad) return bad;
    int64_t most = 0;           // of any type
    for (int type : {QS_SRC_F32, QS_SRC_BF16}) {
        a.type = type;
        const int64_t n = qskv::split_of(a, nullptr).bytes;
        most = n > most ? n : most;
    }
    return most;
}

int qs_kv_attention(const qs_kv_cache* cache, int type, const void* q, int64_t q_token_stride_bytes, int64_t batch,
                    int64_t new_tokens, int64_t query_heads, const int32_t* tables, int64_t pages_each,
                    int64_t table_stride, const int32_t* lengths, float scale, int64_t window, void* out,
                    int64_t out_bytes, void* workspace, int64_t workspace_bytes, void* hip_stream) {
    qs_host::clear_error();
    qskv::AttentionArgs a{};
    const int bad = attention_sizes(cache, batch, new_tokens, query_heads, pages_each, a);
    if (bad) return bad;
    const int esz = size_of(type);
    if (!esz) return fail(QS_EINVAL, "unsupported query type %d (F32=0, F16=1, BF16=30)", type);
    if (window < 0) return fail(QS_EINVAL, "window %lld < 0", (long long)window);
    const int64_t tokens = batch * new_tokens, width = query_heads * cache->head_dim * esz;
    if (tokens == 0) return 0;
    if (!q || !lengths || !out || (pages_each > 0 && !tables)) return fail(QS_EINVAL, "null q, tables, lengths or out");
    if (off16(q) || off16(out) || off4(tables) || off4(lengths))
        return fail(QS_EINVAL, "q and out must be 16-byte aligned, tables and lengths 4-byte");
    if ((q_token_stride_bytes < width && tokens > 1) || q_token_stride_bytes < 0 || q_token_stride_bytes % 16 ||
        q_token_stride_bytes > kMaxSpan / tokens)
        return fail(QS_EINVAL, "token stride %lld must be >= %lld, a multiple of 16 and in a 2^62-byte span",
                    (long long)q_token_stride_bytes, (long long)width);
    if (table_stride < pages_each || table_stride > kMaxSpan / batch / 4)
        return fail(QS_EINVAL, "table stride %lld must be >= %lld and in a 2^62-byte span", (long long)table_stride,
                    (long long)pages_each);
    if (out_bytes < tokens * width)
        return fail(QS_EINVAL, "out holds %lld bytes, %lld needed", (long long)out_bytes, (long long)(tokens * width));
    a.q = q;
    a.out = out;
    a.tables = tables;
    a.lengths = lengths;
    a.q_stride = q_token_stride_bytes / esz;
    a.table_stride = table_stride;
    a.window = (int32_t)(window < INT32_MAX ? window : 0);      // as long as any sequence: none
    a.type = type;
    a.scale = scale;
    const qskv::Split split = qskv::split_of(a, workspace);
    if (split.bytes && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 256 || workspace_bytes < split.bytes))
        return fail(QS_EINVAL, "workspace holds %lld bytes at %p, %lld needed, 256-byte aligned", (long long)workspace_bytes,
                    workspace, (long long)split.bytes);
    hipStream_t st = static_cast<hipStream_t>(hip_stream);
    const hipError_t e = a.c.k_bits == 8 ? (a.c.v_bits == 8 ? qskv::launch_attention<8, 8>(a, split, st) : qskv::launch_attention<8, 4>(a, split, st))
                                         : (a.c.v_bits == 8 ? qskv::launch_attention<4, 8>(a, split, st) : qskv::launch_attention<4, 4>(a, split, st));
    if (e != hipSuccess) return fail(QS_EIO, "kv_attention: launch failed: %s", hipGetErrorString(e));
    return 0;
}

}  // extern "C"
