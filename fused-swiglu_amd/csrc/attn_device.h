// Device code that the attention kernels share.
#pragma once
#include <hip/hip_runtime.h>

namespace fsw {

// Largest value of lanes l, l ^ 16, l ^ 32, l ^ 48: a lane swap of a register with a copy of itself leaves two groups' values side by
// side, one in either register. Written out: of the builtins' two results the compiler used the first alone here, so that the maximum was
// group 0's and weights of fp16 overflowed where another group's scores lay 16 powers of two above. (The wait states are those
// that a swap needs behind a vector write of its operands.)
__device__ __forceinline__ float max_over_groups(float x) {
  float y = x;
  asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(x), "+v"(y));
  x = fmaxf(x, y);
  y = x;
  asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(x), "+v"(y));
  return fmaxf(x, y);
}

}  // namespace fsw
