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

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

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

// ---- one to four rows ----

// L lanes share a weight row and take its groups of 32 in turn; each of them
// holds R weight rows, so a group of x is read once for R of the weight's.
template <int TYPE, int T, int L, int R>
__global__ __launch_bounds__(256) void k_linear_few(LinearArgs a) {
    constexpr int SUB = Format<TYPE>::SUB;
    __shared__ uint16_t grid[Format<TYPE>::GRID ? Format<TYPE>::GRID : 1];
    qsd::stage_grid<TYPE>(grid, threadIdx.x, 256);
    if (Format<TYPE>::GRID) __syncthreads();
    const int lane = threadIdx.x % L;
    const int64_t n0 = ((int64_t)blockIdx.x * (256 / L) + threadIdx.x / L) * R;
    const int groups = (int)(a.k / 32), t1 = (int)a.t - 1;
    float acc[T][R] = {};
    for (int g = lane; g < groups; g += L) {
        uint32_t x[T][8];
        float s[T];
#pragma unroll
        for (int t = 0; t < T; t++) {
            const int64_t row = t < t1 ? t : t1;
            __builtin_memcpy(x[t], __builtin_assume_aligned(a.q + row * a.k + 32 * g, 16), 32);
            s[t] = a.s[row * groups + g];
        }
#pragma unroll
        for (int r = 0; r < R; r++) {
            const int64_t n = n0 + r < a.n ? n0 + r : a.n - 1;
            Group<TYPE> w;
            qsd::decode_row_group<TYPE>(a.w + n * a.row_bytes, g, grid, w);
#pragma unroll
            for (int t = 0; t < T; t++) {
                float y = 0.0f;
#pragma unroll
                for (int h = 0; h < SUB; h++) {
                    int c = 0, o = 0;
#pragma unroll
                    for (int i = 8 / SUB * h; i < 8 / SUB * (h + 1); i++) {
                        c = dot4(w.c[i], x[t][i], c);
                        if (Format<TYPE>::MIN) o = dot4(x[t][i], qsd::ONES, o);
                    }
                    y = __builtin_fmaf(w.d[h], (float)c, y);
                    if (Format<TYPE>::MIN) y = __builtin_fmaf(-w.m[h], (float)o, y);
                }
                acc[t][r] = __builtin_fmaf(s[t], y, acc[t][r]);
            }
        }
    }
    if (a.ids)
#pragma unroll
        for (int t = 0; t < T; t++) {
            const int id = t <= t1 ? adapter_of(a, t) : -1;
            if (id >= 0)
#pragma unroll
                for (int r = 0; r < R; r++)
                    if (n0 + r < a.n) acc[t][r] += adapter_sum(a, id, t, n0 + r, lane, L);
        }
#pragma unroll
    for (int t = 0; t < T; t++)
#pragma unroll
        for (int r = 0; r < R; r++) {
#pragma unroll
            for (int o = 1; o < L; o *= 2) acc[t][r] += __shfl_xor(acc[t][r], o);
            if (lane == 0 && t <= t1 && n0 + r < a.n) store_value(a, (int64_t)t * a.n + n0 + r, acc[t][r]);
        }
}

// ---- more rows ----

// An int32 matrix product starts from this word in every place, so that the
// result's bits are the float 1.5 * 2^23 + sum (|sum| <= 32 * 128 * 128 < 2^22):
// a subtraction at full rate in place of a conversion at half rate.
constexpr float INT_BIAS = 12582912.0f;

// A tile of BM rows by BN weight rows. The workgroup's WM x WN x WK waves
// stage G groups of 32 values at a time: the weight's are decoded to bytes by
// a thread a group, the rows' copied. WM x WN waves split the tile, WK the
// groups (their sums are joined in LDS at the end, in order).
template <int TYPE, int BM, int BN, int WM, int WN, int WK, int G>
__global__ __launch_bounds__(64 * WM * WN * WK) void k_linear_tile(LinearArgs a) {
    constexpr int THREADS = 64 * WM * WN * WK, SUB = Format<TYPE>::SUB;
    constexpr bool MIN = Format<TYPE>::MIN;
    constexpr int UM = BM / WM / 32, UN = BN / WN / 32;
    // a group's rows of 32 bytes one after another; 32 bytes between groups keep
    // threads that write different groups of a row off each other's banks
    constexpr int XP = BM * 32 + 32, WP = BN * 32 + 32;
    __shared__ __attribute__((aligned(16))) uint8_t xq[G * XP], wq[G * WP];
    __shared__ __attribute__((aligned(16))) float xs[G][BM], wd[G][SUB][BN];
    __shared__ __attribute__((aligned(16))) float xo[MIN ? G : 1][MIN ? SUB : 1][MIN ? BM : 4];
    __shared__ float wm[MIN ? G : 1][MIN ? SUB : 1][MIN ? BN : 1];
    __shared__ float join[WK > 1 ? WK - 1 : 1][WK > 1 ? BM * BN : 1];
    __shared__ uint16_t grid[Format<TYPE>::GRID ? Format<TYPE>::GRID : 1];
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const int wk = wave % WK, wn = wave / WK % WN, wmr = wave / WK / WN;
    const int col = lane % 32, half = lane / 32;
    const int64_t tiles_m = (a.t + BM - 1) / BM;
    const int64_t t0 = (int64_t)blockIdx.x % tiles_m * BM, n0 = (int64_t)blockIdx.x / tiles_m * BN;
    const int groups = (int)(a.k / 32);
    qsd::stage_grid<TYPE>(grid, tid, THREADS);
    if (Format<TYPE>::GRID) __syncthreads();
    float acc[UM][UN][16] = {};
    for (int g0 = 0; g0 < groups; g0 += G) {
        const int now = groups - g0 < G ? groups - g0 : G;
        for (int i = tid; i < BN * G; i += THREADS) {
            const int g = i % G, r = i / G;
            if (g >= now) continue;
            const int64_t n = n0 + r < a.n ? n0 + r : a.n - 1;
            Group<TYPE> w;
            qsd::decode_row_group<TYPE>(a.w + n * a.row_bytes, g0 + g, grid, w);
            uint4* d = reinterpret_cast<uint4*>(wq + g * WP + r * 32);
            d[0] = uint4{w.c[0], w.c[1], w.c[2], w.c[3]};
            d[1] = uint4{w.c[4], w.c[5], w.c[6], w.c[7]};
#pragma unroll
            for (int h = 0; h < SUB; h++) {
                wd[g][h][r] = w.d[h];
                if constexpr (MIN) wm[g][h][r] = w.m[h];
            }
        }
        for (int i = tid; i < BM * G; i += THREADS) {
            const int g = i % G, r = i / G;
            if (g >= now) continue;
            const int64_t t = t0 + r < a.t ? t0 + r : a.t - 1;
            const uint4* p = reinterpret_cast<const uint4*>(a.q + t * a.k + 32 * (g0 + g));
            const uint4 lo = p[0], hi = p[1];
            const float s = a.s[t * groups + g0 + g];
            uint4* d = reinterpret_cast<uint4*>(xq + g * XP + r * 32);
            d[0] = lo;
            d[1] = hi;
            xs[g][r] = s;
            if constexpr (MIN) {
                const int o0 = dot4(lo.x, qsd::ONES, dot4(lo.y, qsd::ONES, dot4(lo.z, qsd::ONES, dot4(lo.w, qsd::ONES, 0))));
                const int o1 = dot4(hi.x, qsd::ONES, dot4(hi.y, qsd::ONES, dot4(hi.z, qsd::ONES, dot4(hi.w, qsd::ONES, 0))));
                if constexpr (SUB == 2) xo[g][0][r] = s * (float)o0, xo[g][1][r] = s * (float)o1;
                else xo[g][0][r] = s * (float)(o0 + o1);
            }
        }
        __syncthreads();
        for (int g = wk; g < now; g += WK) {
#pragma unroll
            for (int um = 0; um < UM; um++) {
                const int m0 = (wmr * UM + um) * 32;
                const uint8_t* xrow = xq + g * XP + (m0 + col) * 32;
                f32x4 sx[4];
#pragma unroll
                for (int j = 0; j < 4; j++) sx[j] = *reinterpret_cast<const f32x4*>(&xs[g][m0 + 8 * j + 4 * half]);
#pragma unroll
                for (int un = 0; un < UN; un++) {
                    const int c = (wn * UN + un) * 32 + col;
                    const uint8_t* wrow = wq + g * WP + c * 32;
                    const int b = __float_as_int(INT_BIAS);
                    const i32x16 bias = {b, b, b, b, b, b, b, b, b, b, b, b, b, b, b, b};
#pragma unroll
                    for (int h = 0; h < SUB; h++) {
                        i32x16 p;
                        if constexpr (SUB == 1) {
                            const i32x4 av = *reinterpret_cast<const i32x4*>(xrow + 16 * half);
                            const i32x4 bv = *reinterpret_cast<const i32x4*>(wrow + 16 * half);
                            p = __builtin_amdgcn_mfma_i32_32x32x32_i8(av, bv, bias, 0, 0, 0);
                        } else {
                            const long av = *reinterpret_cast<const long*>(xrow + 16 * h + 8 * half);
                            const long bv = *reinterpret_cast<const long*>(wrow + 16 * h + 8 * half);
                            p = __builtin_amdgcn_mfma_i32_32x32x16_i8(av, bv, bias, 0, 0, 0);
                        }
                        const float d = wd[g][h][c];
#pragma unroll
                        for (int i = 0; i < 16; i++)
                            acc[um][un][i] = __builtin_fmaf(__int_as_float(p[i]) - INT_BIAS, d * sx[i / 4][i % 4], acc[um][un][i]);
                        if constexpr (MIN) {
                            const float m = wm[g][h][c];
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const f32x4 o = *reinterpret_cast<const f32x4*>(&xo[g][h][m0 + 8 * j + 4 * half]);
#pragma unroll
                                for (int i = 0; i < 4; i++) acc[um][un][4 * j + i] = __builtin_fmaf(-m, o[i], acc[um][un][4 * j + i]);
                            }
                        }
                    }
                }
            }
        }
        __syncthreads();
    }
    // place of element i of a unit: row 8 (i / 4) + 4 half + i % 4, column `col`
    if constexpr (WK > 1) {
        if (wk > 0)
#pragma unroll
            for (int u = 0; u < UM * UN * 16; u++)
                join[wk - 1][((wmr * WN + wn) * UM * UN * 16 + u) * 64 + lane] = acc[u / 16 / UN][u / 16 % UN][u % 16];
        __syncthreads();
        if (wk > 0) return;
        for (int j = 0; j < WK - 1; j++)
#pragma unroll
            for (int u = 0; u < UM * UN * 16; u++)
                acc[u / 16 / UN][u / 16 % UN][u % 16] += join[j][((wmr * WN + wn) * UM * UN * 16 + u) * 64 + lane];
    }
#pragma unroll
    for (int um = 0; um < UM; um++)
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const int64_t t = t0 + (wmr * UM + um) * 32 + 8 * (i / 4) + 4 * half + i % 4;
            if (t >= a.t) continue;
            const int id = a.ids ? adapter_of(a, t) : -1;
#pragma unroll
            for (int un = 0; un < UN; un++) {
                const int64_t n = n0 + (wn * UN + un) * 32 + col;
                if (n >= a.n) continue;
                float y = acc[um][un][i];
                if (id >= 0) y += adapter_sum(a, id, t, n, 0, 1);
                store_value(a, t * a.n + n, y);
            }
        }
}

}  // namespace qsl
