// Kernel launch that reports its own status.  The <<<>>> form followed by
// hipGetLastError() returns, and clears, whatever error an earlier call on this
// thread left behind (another library's, for instance), which would then be blamed
// on this launch or lost to its owner; hipLaunchKernel returns the result of this
// launch alone and leaves the thread's error state as it found it.
#pragma once

#include <hip/hip_runtime.h>

namespace kmc_host {

template <typename Args>
inline hipError_t launch(void (*kernel)(const Args), dim3 grid, dim3 block, hipStream_t stream, const Args &args)
{
    void *kernel_args[] = {const_cast<Args *>(&args)};
    return hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, kernel_args, 0, stream);
}

// Several launches of one grid, each of at most `most` workgroups, which find their first in args.first_block.
template <typename Args>
inline hipError_t launch_in_parts(void (*kernel)(const Args), int grid, int most, dim3 block, hipStream_t stream, const Args &args)
{
    if (grid <= most) return launch(kernel, dim3(static_cast<unsigned>(grid)), block, stream, args);
    Args part = args;
    for (int left = grid; left > 0; left -= most) {
        part.first_block = grid - left;
        const hipError_t status = launch(kernel, dim3(static_cast<unsigned>(left < most ? left : most)), block, stream, part);
        if (status != hipSuccess || left <= most) return status;
    }
    return hipSuccess;
}

}  // namespace kmc_host
