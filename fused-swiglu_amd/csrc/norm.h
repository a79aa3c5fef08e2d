// Internal launcher interface of the norms around a block (norm_api.hip -> kernels_norm.hip). Nothing here is exported; the public
// surface is include/fsw.h.
#pragma once
#include <hip/hip_runtime.h>

namespace fsw {

struct NormArgs {
  int rows, d;
  const void* x;
  const void* y;     // NULL: the rows are x
  const void* gate;  // NULL: one
  const void* post;  // NULL: y as it is
  const void* pre;   // NULL: one
  long long ldx, ldy, ldg;
  float scale, eps;
  void* x_out;  // may be NULL
  void* h;      // may be NULL
  long long ldxo, ldh;
};
hipError_t launch_add_norm(int dtype, const NormArgs& a, hipStream_t stream);

}  // namespace fsw
