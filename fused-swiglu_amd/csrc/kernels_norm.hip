// Norms around a block of a layer with its gate and residual scale, in one launch:
//   b = y r(y) post  (or y),  x' = x + scale gate b,  h = x' r(x') pre,  r(z) = (mean z^2 + eps)^(-1/2)
// in fp32, x' and h rounded once each; h is made of the unrounded x'.
//
// Every element is read and written once: memory traffic bounds it, and latency where rows are few. A workgroup owns a row at a time and
// keeps it in registers between the two sums, so the row is never read again; workgroups of many rows keep the weights of
// their channels in registers as well. Squares are summed in 64 bits: they are exact there and neither overflow nor vanish for any values that the types
// have, and beside the memory traffic they cost nothing. Measured, both norms: 8192 rows of 8192 channels with a gate of their own 130 us (5.2 TB/s, two fifths of it written; a
// copy reaches 4.9), of 4096 with one gate for all 49 (5.5), of 1024 17 (3.9); 2048 of 16384 66 (4.1: bf16 holds 130 registers there, so a CU has one
// workgroup of eight waves, not two; of 1024 half of the threads have nothing to do); one row of 4096 3.4 us on the device.
#include "attn_device.h"
#include "fsw.h"
#include "fsw_device.h"
#include "fsw_internal.h"
#include "norm.h"

namespace fsw {
namespace {

template <int CTRL>
__device__ __forceinline__ double add_moved(double x) {
  const u32x2 u = __builtin_bit_cast(u32x2, x);
  const u32x2 v = {(unsigned)__builtin_amdgcn_mov_dpp((int)u[0], CTRL, 0xf, 0xf, true),
                   (unsigned)__builtin_amdgcn_mov_dpp((int)u[1], CTRL, 0xf, 0xf, true)};
  return x + __builtin_bit_cast(double, v);
}

// sum over a wave: neighbours, pairs, halves of 16 lanes, then the four groups of 16
__device__ __forceinline__ double wave_sum(double x) {
  x = add_moved<0xb1>(x);
  x = add_moved<0x4e>(x);
  x = add_moved<0x141>(x);
  x = add_moved<0x140>(x);
  x += __shfl_xor(x, 16);
  return x + __shfl_xor(x, 32);
}

// 1 / sqrt(m) as factor a power of two: mean squares of rows reach 2^256, where a float's reciprocal root has no bits left
struct Root {
  float power, factor;
};
__device__ __forceinline__ Root inverse_root(double m) {
  const int e = __builtin_amdgcn_frexp_exp(m) & ~1;
  return Root{__builtin_amdgcn_ldexpf(1.0f, -e / 2), __builtin_amdgcn_rsqf((float)__builtin_amdgcn_ldexp(m, -e))};
}

template <class T, int THREADS, int VECS>
__global__ __launch_bounds__(THREADS) void add_norm_kernel(NormArgs a, double per_channel) {
  constexpr int WAVES = THREADS / 64;
  __shared__ double parts[2][WAVES];
  const int tid = threadIdx.x, vecs = a.d / 8;
  int turn = 0;
  auto row_sum = [&](double s) -> double {
    s = wave_sum(s);
    if constexpr (WAVES > 1) {
      // sums alternate between two sets of places: the barrier of the next one is behind every read of this one
      if ((tid & 63) == 0) parts[turn][tid >> 6] = s;
      __syncthreads();
      s = 0.0;
#pragma unroll
      for (int w = 0; w < WAVES; ++w) s += parts[turn][w];
      turn ^= 1;
    }
    return s;
  };

  u32x4 post[VECS], pre[VECS];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = i * THREADS + tid;
    post[i] = pre[i] = u32x4{0, 0, 0, 0};
    if (v < vecs && a.post) post[i] = *((const u32x4*)a.post + v);
    if (v < vecs && a.pre) pre[i] = *((const u32x4*)a.pre + v);
  }
  for (int row = blockIdx.x; row < a.rows; row += gridDim.x) {
    // the weights stay as they are, two in a register, until they are needed: unpacked before the loop they are twice the registers
#pragma unroll
    for (int i = 0; i < VECS; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(post[i][j]), "+v"(pre[i][j]));
    const u32x4* xp = (const u32x4*)((const unsigned short*)a.x + row * a.ldx);
    const u32x4* yp = (const u32x4*)((const unsigned short*)a.y + row * a.ldy);
    const u32x4* gp = (const u32x4*)((const unsigned short*)a.gate + row * a.ldg);
    u32x4 xv[VECS], yv[VECS], gv[VECS];
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int v = i * THREADS + tid;
      xv[i] = yv[i] = gv[i] = u32x4{0, 0, 0, 0};
      if (v < vecs) {
        xv[i] = xp[v];
        if (a.y) yv[i] = yp[v];
        if (a.gate) gv[i] = gp[v];
      }
    }
    float z[VECS][8];
    if (a.y) {
      Root r = {1.0f, 1.0f};
      if (a.post) {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < VECS; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float lo, hi;
            unpack2<T>(yv[i][j], lo, hi);
            s = __builtin_fma((double)lo, (double)lo, s);
            s = __builtin_fma((double)hi, (double)hi, s);
          }
        r = inverse_root(row_sum(s) * per_channel + (double)a.eps);
      }
#pragma unroll
      for (int i = 0; i < VECS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float b[2], x[2], w[2], g[2];
          unpack2<T>(yv[i][j], b[0], b[1]);
          unpack2<T>(xv[i][j], x[0], x[1]);
          unpack2<T>(post[i][j], w[0], w[1]);
          unpack2<T>(gv[i][j], g[0], g[1]);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            if (a.post) b[k] = b[k] * r.power * r.factor * w[k];
            if (a.gate) b[k] *= g[k];
            z[i][2 * j + k] = __builtin_fmaf(a.scale, b[k], x[k]);
          }
        }
    } else {
#pragma unroll
      for (int i = 0; i < VECS; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) unpack2<T>(xv[i][j], z[i][2 * j], z[i][2 * j + 1]);
    }
    if (a.x_out) {
      u32x4* p = (u32x4*)((unsigned short*)a.x_out + row * a.ldxo);
#pragma unroll
      for (int i = 0; i < VECS; ++i) {
        const int v = i * THREADS + tid;
        u32x4 o;
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] = T::pack2(z[i][2 * j], z[i][2 * j + 1]);
        if (v < vecs) p[v] = o;
      }
    }
    if (!a.h) continue;
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < VECS; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) s = __builtin_fma((double)z[i][j], (double)z[i][j], s);
    const Root r = inverse_root(row_sum(s) * per_channel + (double)a.eps);
    u32x4* p = (u32x4*)((unsigned short*)a.h + row * a.ldh);
#pragma unroll
    for (int i = 0; i < VECS; ++i) {
      const int v = i * THREADS + tid;
      u32x4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float w[2] = {1.0f, 1.0f};
        if (a.pre) unpack2<T>(pre[i][j], w[0], w[1]);
        o[j] = T::pack2(z[i][2 * j] * r.power * r.factor * w[0], z[i][2 * j + 1] * r.power * r.factor * w[1]);
      }
      if (v < vecs) p[v] = o;
    }
  }
}

template <class T, int THREADS, int VECS>
hipError_t launch(const NormArgs& a, hipStream_t stream) {
  const int most = 256 * (2048 / THREADS);
  add_norm_kernel<T, THREADS, VECS><<<a.rows < most ? a.rows : most, THREADS, 0, stream>>>(a, 1.0 / a.d);
  return hipGetLastError();
}

// The least form that holds a row: one vector a thread up to 256 threads, then up to four of 256 threads, and more threads beyond.
template <class T>
hipError_t launch_typed(const NormArgs& a, hipStream_t stream) {
  const int vecs = a.d / 8;
  if (vecs <= 64) return launch<T, 64, 1>(a, stream);
  if (vecs <= 256) return launch<T, 256, 1>(a, stream);
  if (vecs <= 512) return launch<T, 256, 2>(a, stream);
  if (vecs <= 1024) return launch<T, 256, 4>(a, stream);
  if (vecs <= 2048) return launch<T, 512, 4>(a, stream);
  return launch<T, 1024, 4>(a, stream);
}

}  // namespace

hipError_t launch_add_norm(int dtype, const NormArgs& a, hipStream_t stream) {
  return dtype == FSW_BF16 ? launch_typed<Bf16>(a, stream) : launch_typed<Fp16>(a, stream);
}

}  // namespace fsw
