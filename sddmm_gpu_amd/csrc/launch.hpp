// Kernel launches that return their own error: hipLaunchKernelGGL leaves it to be fetched by hipGetLastError, a call
// that costs 0.4 us next to 2.6 us for the launch itself -- on a small matrix the calls take as long as the kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <cstdint>
#include <type_traits>

namespace sddmm {

// A launch holds less than 2^32 threads in each dimension.  The runtime takes more without an error and runs what is left of their number
// modulo 2^32 (measured: of 2^24 + 3 workgroups of 256 threads three), so entry points refuse such sizes, and `launch` in case one does not.
inline bool launchable(int64_t workgroups, int64_t threads) { return workgroups <= (int64_t)UINT32_MAX / threads; }

template <class... P>
inline hipError_t launch(void (*fn)(P...), dim3 grid, dim3 block, size_t lds, hipStream_t stream, std::type_identity_t<P>... args)
{
    if (!launchable(grid.x, block.x) || !launchable(grid.y, block.y) || !launchable(grid.z, block.z)) return hipErrorInvalidConfiguration;
    void *p[] = {(void *)&args...};
    return hipLaunchKernel((const void *)fn, grid, block, p, lds, stream);
}

}  // namespace sddmm
