// Launches of the products of laid-out factors and of the adapters' products;
// they do not depend on the weight's format.
#include <hip/hip_runtime.h>

#include "qs_launch_kernel.h"
#include "qs_matrix16.h"

namespace qsl {

using qs_host::launch_kernel;

namespace {

// a multiple of the 8 XCDs: each takes a run of tiles
dim3 grid_of(int64_t tiles) { return dim3((unsigned)((tiles + 7) / 8 * 8)); }

// The tile whose rounds over the 256 CUs cost least.
template <int N>
int choose(const Tiles (&choices)[N], int64_t t, int64_t n) {
    int best = 0;
    int64_t least = INT64_MAX;
    for (int i = 0; i < N; i++) {
        const Tiles& c = choices[i];
        const int64_t cost = (tile_count(t, n, c.bm, c.bn) + c.held - 1) / c.held * c.cost;
        if (cost < least) least = cost, best = i;
    }
    return best;
}

template <int PLANES, int MINS, int BM, int BN, int WM, int WN, int WK, int G>
hipError_t product(const MatrixArgs& a, hipStream_t st) {
    const dim3 grid = grid_of(tile_count(a.l.t, a.count, BM, BN)), block(64 * WM * WN * WK);
    if (!a.l.ids) return launch_kernel(k_matrix<PLANES, MINS, BM, BN, WM, WN, WK, G, 0>, grid, block, 0, st, a);
    if (a.l.b_type == QS_SRC_BF16) return launch_kernel(k_matrix<PLANES, MINS, BM, BN, WM, WN, WK, G, QS_SRC_BF16>, grid, block, 0, st, a);
    return launch_kernel(k_matrix<PLANES, MINS, BM, BN, WM, WN, WK, G, QS_SRC_F16>, grid, block, 0, st, a);
}

template <int PLANES, int MINS>
hipError_t any(const MatrixArgs& a, hipStream_t st) {
    constexpr Tiles choices[] = {{128, 128, 512, 690}, {128, 128, 256, 430}, {64, 64, 512, 230}};
    switch (choose(choices, a.l.t, a.count)) {
    case 0: return product<PLANES, MINS, 128, 128, 2, 2, 1, 2>(a, st);
    case 1: return product<PLANES, MINS, 128, 128, 2, 2, 2, 4>(a, st);
    default: return product<PLANES, MINS, 64, 64, 1, 2, 2, 4>(a, st);
    }
}

template <int BM, int BN, int WM, int WN, int WK, int S>
hipError_t product16(const Matrix16Args& a, hipStream_t st) {
    const dim3 grid = grid_of(tile_count(a.l.t, a.count, BM, BN) * a.l.splits), block(64 * WM * WN * WK);
    if (!a.l.ids) return launch_kernel(k_matrix16<BM, BN, WM, WN, WK, S, 0>, grid, block, 0, st, a);
    if constexpr (BN / WN / 32 * (BM / WM / 32) > 8) return hipErrorInvalidValue;       // not chosen with adapters
    else if (a.l.b_type == QS_SRC_BF16) return launch_kernel(k_matrix16<BM, BN, WM, WN, WK, S, QS_SRC_BF16>, grid, block, 0, st, a);
    else return launch_kernel(k_matrix16<BM, BN, WM, WN, WK, S, QS_SRC_F16>, grid, block, 0, st, a);
}

template <int TYPE>
hipError_t adapters(const AdapterArgs& a, hipStream_t st) {
    if (takes_matrix(a.t, a.n, a.k)) {
        const unsigned ranks = (unsigned)((a.ldv + 31) / 32);
        const hipError_t e = launch_kernel(k_adapter_many<TYPE>, dim3((unsigned)((a.t + 31) / 32), ranks, (unsigned)a.parts),
                                           dim3(512), 0, st, a);
        return e != hipSuccess ? e : launch_kernel(k_adapter_join<TYPE>, dim3((unsigned)((a.t + 15) / 16), ranks), dim3(256), 0, st, a);
    }
    const hipError_t e = launch_kernel(k_adapter_few<TYPE>, dim3((unsigned)a.t, (unsigned)(a.ldv / 8)), dim3(256), 0, st, a);
    if (e != hipSuccess || a.few) return e;
    return launch_kernel(k_adapter_delta<TYPE>, dim3((unsigned)((a.n + 255) / 256), (unsigned)a.t), dim3(256), 0, st, a);
}

}  // namespace

hipError_t launch_matrix(int planes, int mins, const MatrixArgs& a, hipStream_t st) {
    if (planes == 2) return any<2, 0>(a, st);
    return mins == 0 ? any<1, 0>(a, st) : mins == 1 ? any<1, 1>(a, st) : any<1, 2>(a, st);
}

static hipError_t tile16(int tile, const Matrix16Args& a, hipStream_t st) {
    switch (tile) {
    case 0: return product16<256, 320, 4, 2, 1, 4>(a, st);
    case 1: return product16<256, 256, 2, 4, 1, 4>(a, st);
    case 2: return product16<128, 160, 4, 1, 2, 8>(a, st);
    case 3: return product16<128, 96, 2, 1, 4, 8>(a, st);
    default: return product16<64, 64, 1, 1, 8, 8>(a, st);
    }
}

hipError_t launch_matrix16(const Matrix16Args& a, hipStream_t st) {
    // a product of one slice was split with its workspace in view
    const int tile = choose16(a.l.ids, a.l.t, a.count, a.l.k, a.count < a.l.n ? 1 : MOST_PARTS).tile;
    const hipError_t e = tile16(tile, a, st);
    return e != hipSuccess || a.l.splits == 1 ? e : launch_join(a.l, st);
}

hipError_t launch_join(const LinearArgs& a, hipStream_t st) {
    return launch_kernel(k_join, dim3((unsigned)((a.t * a.n + 255) / 256)), dim3(256), 0, st, a);
}

hipError_t launch_adapters(int type, const AdapterArgs& a, hipStream_t st) {
    return type == QS_SRC_BF16 ? adapters<QS_SRC_BF16>(a, st) : adapters<QS_SRC_F16>(a, st);
}

}  // namespace qsl
