// C entry points of the norms around a block (include/fsw.h): argument validation on the host, then the launcher.
#include <hip/hip_runtime.h>
#include <float.h>
#include <math.h>
#include <stdint.h>

#include "fsw.h"
#include "fsw_internal.h"
#include "norm.h"

namespace {

constexpr int64_t MAX_D = 32768, MAX_LD = 1LL << 31;

// rows of d elements
int check_rows(const void* p, int64_t ld, int64_t rows, int64_t d, bool written) {
  if (!p) return FSW_E_NULL;
  if (ld < 0 || (written && rows > 1 && ld < d)) return FSW_E_LD;
  if (ld > MAX_LD) return FSW_E_SHAPE;
  return ld % 8 || ((uintptr_t)p & 15) ? FSW_E_ALIGN : FSW_OK;
}

#define CHECK(e)                    \
  do {                              \
    const int rc_ = (e);            \
    if (rc_ != FSW_OK) return rc_;  \
  } while (0)

}  // namespace

extern "C" {

int fsw_validate_add_norm(int dtype, int64_t M, int64_t D, const void* X, int64_t ldx, const void* Y, int64_t ldy, const void* gate,
                          int64_t ld_gate, const void* post, const void* pre, float scale, float eps, const void* Xout, int64_t ldxo,
                          const void* H, int64_t ldh) {
  if (dtype != FSW_BF16 && dtype != FSW_FP16) return FSW_E_DTYPE;
  if (M < 0 || M > (1 << 30) || D < 1 || D > MAX_D) return FSW_E_SHAPE;
  if (D % 8) return FSW_E_ALIGN;
  if (!isfinite(scale) || !isfinite(eps) || eps < FLT_MIN) return FSW_E_SHAPE;
  if (M == 0) return FSW_OK;
  CHECK(check_rows(X, ldx, M, D, false));
  if (Y) {
    CHECK(check_rows(Y, ldy, M, D, false));
  } else if (gate || post || Xout) {
    return FSW_E_NULL;
  }
  if (gate) {
    CHECK(check_rows(gate, ld_gate, M, D, false));
    if (ld_gate != 0 && ld_gate < D) return FSW_E_LD;
  }
  if (post) CHECK(check_rows(post, 0, 1, D, false));
  if (pre) CHECK(check_rows(pre, 0, 1, D, false));
  if (!Xout && !H) return FSW_E_NULL;
  if (Xout) CHECK(check_rows(Xout, ldxo, M, D, true));
  if (H) CHECK(check_rows(H, ldh, M, D, true));
  return FSW_OK;
}

int fsw_add_norm(int dtype, int64_t M, int64_t D, const void* X, int64_t ldx, const void* Y, int64_t ldy, const void* gate, int64_t ld_gate,
                 const void* post, const void* pre, float scale, float eps, void* Xout, int64_t ldxo, void* H, int64_t ldh, void* stream) {
  CHECK(fsw_validate_add_norm(dtype, M, D, X, ldx, Y, ldy, gate, ld_gate, post, pre, scale, eps, Xout, ldxo, H, ldh));
  if (M == 0) return FSW_OK;
  CHECK(fsw::device_status());
  const fsw::NormArgs a = {(int)M, (int)D, X, Y, gate, post, pre, ldx, ldy, ld_gate, scale, eps, Xout, H, ldxo, ldh};
  return fsw::launch_status(fsw::launch_add_norm(dtype, a, (hipStream_t)stream));
}

}  // extern "C"
