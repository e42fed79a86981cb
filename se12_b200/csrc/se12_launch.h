// What every launch with dynamic shared memory has in common. Not part of the
// public interface (include/se12.h is).
#pragma once

#include <cstddef>
#include <cuda_runtime.h>

namespace se12 {

constexpr size_t kMaxSmemPerCta = 227 * 1024;  // one CTA per SM (sm_100 opt-in maximum)

// Lets `kernel` be launched with any amount of dynamic shared memory that fits
// beside its `fixed` bytes of static shared memory. The limit belongs to the kernel
// on its device and is shared by all threads and captured graphs: set to a call's own
// size it may be lowered by another thread before the launch, which then fails. Every
// call sets the same.
template <typename... Params>
inline cudaError_t allow_shared_memory(void (*kernel)(Params...), size_t fixed = 0) {
  return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMaxSmemPerCta - fixed));
}

}  // namespace se12
