// Launches of the products with packed weights, per format. Built several
// times (-DQS_LINEAR_SET=<0..5>), so the formats compile in parallel.
#include <hip/hip_runtime.h>

#include "qs_launch_kernel.h"
#include "qs_linear_kernels.h"
#include "qs_matrix16.h"

namespace qsl {

using qs_host::launch_kernel;

namespace {

template <int TYPE, int L>
FewPlan few_plan(const LinearArgs& a) {
    const int64_t rows = 256 / L, w = (rows * a.row_bytes + 15 + 4 + 15) / 16 * 16;    // a shifted read takes the word after its last
    return {(int)(w < 1 << 20 ? w : 1 << 20), (a.n + rows - 1) / rows};
}
template <int TYPE>
size_t few_lds(const FewPlan& p, int t, int64_t k) {
    return (size_t)(p.w_bytes + k / 32 * few_record(t) * 16 + Format<TYPE>::GRID * 2);
}

template <int TYPE, int T, int L>
hipError_t few(const LinearArgs& a, const FewPlan& p, hipStream_t st) {
    const size_t lds = few_lds<TYPE>(p, T, a.k);
    // as many workgroups as the 256 CUs hold at a time: x is staged once by each
    const int64_t held = 256 * (int64_t)(160 * 1024 / lds < 8 ? 160 * 1024 / lds : 8);
    return launch_kernel(k_linear_few<TYPE, T, L>, dim3((unsigned)(p.blocks < held ? p.blocks : held)), dim3(256), lds,
                         st, a, p);
}

template <int TYPE, int L>
hipError_t few_rows(int t, const LinearArgs& a, const FewPlan& p, hipStream_t st) {
    switch (t) {
    case 1: return few<TYPE, 1, L>(a, p, st);
    case 2: return few<TYPE, 2, L>(a, p, st);
    case 3: return few<TYPE, 3, L>(a, p, st);
    case 4: return few<TYPE, 4, L>(a, p, st);
    case 5: return few<TYPE, 5, L>(a, p, st);
    case 6: return few<TYPE, 6, L>(a, p, st);
    default: return few<TYPE, 8, L>(a, p, st);
    }
}

template <int TYPE, int BM, int BN, int WM, int WN, int WK, int G>
hipError_t tile(const LinearArgs& a, hipStream_t st) {
    const int64_t tiles = ((a.t + BM - 1) / BM) * ((a.n + BN - 1) / BN) * a.splits;
    // a multiple of the 8 XCDs: each takes a run of tiles; 2^23 workgroups at most
    // in a row of the grid, whose threads are under 2^32
    const int64_t rows = (tiles + (1 << 23) - 1) >> 23, row = ((tiles + rows - 1) / rows + 7) / 8 * 8;
    return launch_kernel(k_linear_tile<TYPE, BM, BN, WM, WN, WK, G>, dim3((unsigned)row, (unsigned)rows),
                         dim3(64 * WM * WN * WK), 0, st, a);
}

template <int TYPE>
hipError_t matrix(const LinearArgs& a, void* work, hipStream_t st) {
    const MatrixPlan plan = matrix_plan(TYPE, false, a.n, a.k, a.t);
    uint8_t *xl = static_cast<uint8_t*>(work), *wl = xl + plan.x_bytes;
    const int64_t per = (plan.groups + 7) / 8;
    for (int64_t first = 0; first < a.n; first += plan.slice) {
        const int64_t count = a.n - first < plan.slice ? a.n - first : plan.slice;
        const LayoutArgs lay{a.w + first * a.row_bytes, wl, a.q, a.s, xl, a.row_bytes, count, a.t, a.k,
                             (count + 31) / 32 * per, plan.groups};
        const int64_t blocks = lay.w_blocks + (first ? 0 : (a.t + 31) / 32 * per);      // the rows once
        hipError_t e = launch_kernel(k_lay_out<TYPE>, dim3((unsigned)blocks), dim3(256), 0, st, lay);
        if (e != hipSuccess) return e;
        using M = MatrixFormat<TYPE>;
        e = launch_matrix(M::PLANES, M::MINS, MatrixArgs{a, xl, wl, first, count, plan.groups}, st);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

template <int TYPE>
hipError_t matrix16(const LinearArgs& a, void* work, hipStream_t st) {
    const MatrixPlan plan = matrix_plan(TYPE, true, a.n, a.k, a.t);
    float *xs = static_cast<float*>(work), *ws = xs + a.t;
    uint8_t *xl = static_cast<uint8_t*>(work) + plan.scale_bytes, *wl = xl + plan.x_bytes;
    const int64_t per = (plan.groups + 7) / 8;
    for (int64_t first = 0; first < a.n; first += plan.slice) {
        const int64_t count = a.n - first < plan.slice ? a.n - first : plan.slice, rows = first ? 0 : a.t;   // the rows once
        const uint8_t* w = a.w + first * a.row_bytes;
        const ScaleArgs sc{w, a.s, ws, xs, a.row_bytes, count, a.t, a.k, (count + 31) / 32};
        hipError_t e = launch_kernel(k_row_scales<TYPE>, dim3((unsigned)(sc.w_blocks + (rows + 31) / 32)), dim3(256), 0, st, sc);
        if (e != hipSuccess) return e;
        const Layout16Args lay{w, a.q, a.s, ws, xs, wl, xl, a.row_bytes, count, a.t, a.k, (count + 31) / 32 * per, plan.groups};
        e = launch_kernel(k_lay_out16<TYPE>, dim3((unsigned)(lay.w_blocks + (rows + 31) / 32 * per)), dim3(256), 0, st, lay);
        if (e != hipSuccess) return e;
        e = launch_matrix16(Matrix16Args{a, xl, wl, ws, xs, first, count, plan.groups}, st);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

template <int TYPE>
hipError_t launch_linear(const LinearArgs& a, void* work, hipStream_t st) {
    // 16 lanes to a weight row, or a wave where that leaves too few workgroups or
    // rows too long for LDS (a row with q4_k, us for 16 lanes and 64: 9,728 x 2,560
    // 7.2 and 10.1; 4,096 x 2,560 4.8 and 5.2; 1,024 x 2,560 4.3 and 3.9).
    if (takes_few(a.row_bytes, a.t, a.k)) {
        static_assert(Format<TYPE>::GRID * 2 <= FEW_GRID, "the code book's place");
        const int t = a.t <= 6 ? (int)a.t : 8;
        const FewPlan p16 = few_plan<TYPE, 16>(a), p64 = few_plan<TYPE, 64>(a);
        if (p16.blocks >= 256 && few_lds<TYPE>(p16, t, a.k) <= 80 * 1024) return few_rows<TYPE, 16>(t, a, p16, st);
        return few_rows<TYPE, 64>(t, a, p64, st);
    }
    if (takes_matrix(a.t, a.n, a.k)) return a.f16 ? matrix16<TYPE>(a, work, st) : matrix<TYPE>(a, work, st);
    // Up to 64 rows in one tile, so that the weight is decoded once. 64 columns
    // halve what each thread does to stage the rows (64 rows with q4_k 9,728 x 2,560
    // 21.5 us, 32 columns 24.5; q6_k 2,560 x 9,728 27 and 29), 32 make enough tiles of
    // a narrow weight (61 rows with q8_0 1,024 x 2,560 9.7 us, 64 columns 10.7). 32 x
    // 32 to 32 rows: 16 with q6_k 151,936 x 2,560 164 us, in 64 x 32 242, 64 x 64 250.
    const hipError_t e = a.t <= 32      ? tile<TYPE, 32, 32, 1, 1, 4, 8>(a, st)
                         : a.n >= 2048 ? tile<TYPE, 64, 64, 2, 2, 2, 8>(a, st)
                                       : tile<TYPE, 64, 32, 2, 1, 2, 8>(a, st);
    return e != hipSuccess || a.splits == 1 ? e : launch_join(a, st);
}

#define QS_LINEAR(T) template hipError_t launch_linear<T>(const LinearArgs&, void*, hipStream_t);
#if QS_LINEAR_SET == 0
QS_LINEAR(QS_TYPE_Q4_0) QS_LINEAR(QS_TYPE_Q4_1) QS_LINEAR(QS_TYPE_Q8_0)
#elif QS_LINEAR_SET == 1
QS_LINEAR(QS_TYPE_Q5_0) QS_LINEAR(QS_TYPE_Q5_1) QS_LINEAR(QS_TYPE_IQ4_NL)
#elif QS_LINEAR_SET == 2
QS_LINEAR(QS_TYPE_Q2_K) QS_LINEAR(QS_TYPE_Q3_K) QS_LINEAR(QS_TYPE_Q4_K)
#elif QS_LINEAR_SET == 3
QS_LINEAR(QS_TYPE_Q5_K) QS_LINEAR(QS_TYPE_Q6_K) QS_LINEAR(QS_TYPE_IQ4_XS)
#elif QS_LINEAR_SET == 4
QS_LINEAR(QS_TYPE_IQ2_XXS) QS_LINEAR(QS_TYPE_IQ2_XS) QS_LINEAR(QS_TYPE_IQ2_S)
#else
QS_LINEAR(QS_TYPE_IQ3_XXS) QS_LINEAR(QS_TYPE_IQ3_S)
#endif

}  // namespace qsl
