// Launches of the products with packed weights, per format. Built several
// times (-DQS_LINEAR_SET=<0..5>), so the formats compile in parallel.
#include <hip/hip_runtime.h>

#include "qs_launch_kernel.h"
#include "qs_linear_kernels.h"

namespace qsl {

using qs_host::launch_kernel;

namespace {

template <int TYPE, int T, int L, int R>
hipError_t few(const LinearArgs& a, hipStream_t st) {
    constexpr int ROWS = 256 / L * R;
    return launch_kernel(k_linear_few<TYPE, T, L, R>, dim3((unsigned)((a.n + ROWS - 1) / ROWS)), dim3(256), 0, st, a);
}

template <int TYPE, int BM, int BN, int WM, int WN, int WK, int G>
hipError_t tile(const LinearArgs& a, hipStream_t st) {
    const int64_t tiles = ((a.t + BM - 1) / BM) * ((a.n + BN - 1) / BN);
    return launch_kernel(k_linear_tile<TYPE, BM, BN, WM, WN, WK, G>, dim3((unsigned)tiles),
                         dim3(64 * WM * WN * WK), 0, st, a);
}

}  // namespace

template <int TYPE>
hipError_t launch_linear(const LinearArgs& a, hipStream_t st) {
    if (a.t == 1) return few<TYPE, 1, 16, 1>(a, st);
    if (a.t == 2) return few<TYPE, 2, 16, 1>(a, st);
    if (a.t <= 4) return few<TYPE, 4, 16, 1>(a, st);
    // 128 x 128 tiles where they fill the 256 CUs, else 32 x 32 ones whose
    // eight waves share the groups
    const int64_t large = ((a.t + 127) / 128) * ((a.n + 127) / 128);
    if (a.t > 64 && large >= 192) return tile<TYPE, 128, 128, 2, 2, 1, 4>(a, st);
    return tile<TYPE, 32, 32, 1, 1, 8, 16>(a, st);
}

#define QS_LINEAR(T) template hipError_t launch_linear<T>(const LinearArgs&, hipStream_t);
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
