#pragma once
#include <hip/hip_runtime.h>

#include <stdint.h>

namespace af3 {

// n workgroups as a grid whose sides, times 1024 threads, stay inside the 32 bits that a launch has for each: workgroup y * gridDim.x + x, those from n on have nothing to do
inline dim3 grid_of(int64_t n) { return n <= (1 << 20) ? dim3((uint32_t)n) : dim3(1u << 20, (uint32_t)((n + (1 << 20) - 1) >> 20)); }

}  // namespace af3
