// Kernel launch of the operators on packed weights.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <tuple>
#include <utility>

namespace qs_host {

// Launch through hipLaunchKernel so its status comes back as the return
// value: the caller's pending hipGetLastError() state is neither read nor
// reset by this library. A dimension of 2^32 threads or more is refused here:
// the runtime takes their number modulo 2^32 and reports nothing unless that is 0.
template <typename... P, typename... A>
hipError_t launch_kernel(void (*kernel)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t st, A&&... args) {
    static_assert(sizeof...(P) == sizeof...(A), "kernel argument count");
    if ((uint64_t)grid.x * block.x >> 32 || (uint64_t)grid.y * block.y >> 32 || (uint64_t)grid.z * block.z >> 32)
        return hipErrorInvalidConfiguration;
    std::tuple<P...> vals(std::forward<A>(args)...);
    void* argv[sizeof...(P)];
    std::apply([&](auto&... v) {
        int i = 0;
        ((argv[i++] = static_cast<void*>(&v)), ...);
    }, vals);
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, argv, lds, st);
}

}  // namespace qs_host
