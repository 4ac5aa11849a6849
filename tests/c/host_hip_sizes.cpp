/* host_hip.cpp with the runtime's limit on a launch: fewer than 2^32 threads in
 * each dimension, else hipErrorInvalidConfiguration. */
#define __HIP_PLATFORM_AMD__ 1
#include <hip/hip_runtime_api.h>
#define hipLaunchKernel launch_of_any_size
#include "host_hip.cpp"
#undef hipLaunchKernel

extern "C" hipError_t hipLaunchKernel(const void* f, dim3 g, dim3 b, void** args, size_t shared, hipStream_t st) {
  for (const auto& [grid, block] : {std::pair(g.x, b.x), std::pair(g.y, b.y), std::pair(g.z, b.z)})
    if ((uint64_t)grid * block >> 32 || !grid || !block) return g_last = hipErrorInvalidConfiguration;
  return launch_of_any_size(f, g, b, args, shared, st);
}
