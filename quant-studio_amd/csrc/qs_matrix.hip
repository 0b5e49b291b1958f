// Launches of the product of laid-out factors; it does not depend on the format.
#include <hip/hip_runtime.h>

#include "qs_launch_kernel.h"
#include "qs_matrix.h"

namespace qsl {

namespace {

template <int PLANES, int MINS, int BM, int BN, int WM, int WN, int OCC>
hipError_t product(const MatrixArgs& a, hipStream_t st) {
    const int64_t tiles = ((a.l.t + BM - 1) / BM) * ((a.count + BN - 1) / BN);
    // a multiple of the 8 XCDs: each takes a run of tiles
    return qs_host::launch_kernel(k_matrix<PLANES, MINS, BM, BN, WM, WN, STAGE_GROUPS, OCC>,
                                  dim3((unsigned)((tiles + 7) / 8 * 8)), dim3(64 * WM * WN), 0, st, a);
}

template <int PLANES, int MINS>
hipError_t any(const MatrixArgs& a, hipStream_t st) {
    const int64_t large = ((a.l.t + 127) / 128) * ((a.count + 127) / 128);
    if (large >= 400) return product<PLANES, MINS, 128, 128, 2, 2, 2>(a, st);
    return product<PLANES, MINS, 64, 64, 1, 2, 2>(a, st);
}

}  // namespace

hipError_t launch_matrix(int planes, int mins, const MatrixArgs& a, hipStream_t st) {
    if (planes == 2) return any<2, 0>(a, st);
    return mins == 0 ? any<1, 0>(a, st) : mins == 1 ? any<1, 1>(a, st) : any<1, 2>(a, st);
}

}  // namespace qsl
