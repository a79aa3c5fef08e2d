// Keys and values of some sequences out of their pages, packed one behind the other as rows of the element type: what a prompt's later part
// attends to together with itself (attn_prompt). From a cache of 16-bit elements, or of e4m3 elements with a power of two per row.
//
// Memory traffic bounds it: every cell is read and every row written once. A workgroup owns some rows in a row; its first wave finds the sequence and the
// page of all of them at once, a lane each, then its threads move 8 channels at a time, so that a wave's stores are one piece (16 channels of 8 bits a thread, two
// stores with gaps: 75 us for 70). Measured: 24 sequences of 100 .. 8192 tokens, 8 heads of 128 channels, from 8 bits 68 us a call (4.5 TB/s, two thirds of it written;
// workgroups of twice the rows 70, of half 79), from 16 bits 65 us (6.0 TB/s); pages of 9 tokens no slower. Two heads of 64 channels 12.3 us (a wave that looks up its
// rows one after the other 18.3). Four vectors of a thread under way at a time, and stores past the caches, change nothing.
#include <limits.h>

#include "attn.h"
#include "attn_device.h"
#include "fsw_device.h"
#include "fsw_internal.h"

namespace fsw {
namespace {

constexpr int MOST_ROWS = 64;  // of a workgroup, a lane each while they are looked up

// cells of a cache as 16-byte vectors, and what they stand for
template <class T>
struct Cells16 {
  static constexpr int VEC = 8;  // channels
  PagedKv c;
  __device__ __forceinline__ void move(bool value, long long page, int place, int head, int ch, unsigned short* to) const {
    const unsigned short* p = (const unsigned short*)(value ? c.v : c.k) + page * c.page + head * c.head + place * c.token + ch;
    *(u32x4*)to = __builtin_nontemporal_load((const u32x4*)p);
  }
};
template <class T>
struct Cells8 {
  static constexpr int VEC = 8;
  PagedKv8 c;
  __device__ __forceinline__ void move(bool value, long long page, int place, int head, int ch, unsigned short* to) const {
    const u32x2 x = __builtin_nontemporal_load((const u32x2*)((value ? c.v : c.k) + page * c.page + head * c.head + place * c.token + ch));
    const float up = scale_value((value ? c.v_scale : c.k_scale)[page * c.scale_page + head * c.scale_head + place * c.scale_token]);
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const f32x2 lo = unpack_e4m3<false>(x[i]), hi = unpack_e4m3<true>(x[i]);
      o[2 * i] = T::pack2(lo[0] * up, lo[1] * up);
      o[2 * i + 1] = T::pack2(hi[0] * up, hi[1] * up);
    }
    *(u32x4*)to = o;
  }
};

template <class T, class CELLS>
__global__ __launch_bounds__(256) void kv_read_kernel(ReadArgs a, CELLS cells, Divisor units, Divisor per_row, int rows) {
  // page of each row (-1: behind the last sequence, -2: no page of the cache) and its place there
  __shared__ int pages[MOST_ROWS], places[MOST_ROWS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, first = (int)blockIdx.x * rows;
  if (wave == 0) {
    // the last s <= seqs whose sequence does not begin behind the first row
    int seq = 0;
    for (int n = a.seqs + 1; n > 1;) {
      const int step = (n + 63) / 64, idx = lane * step;
      const int below = __popcll(__ballot(idx < n && a.cu[seq + (idx < n ? idx : 0)] <= first));
      const int skip = (below > 0 ? below - 1 : 0) * step;
      seq += skip;
      n = n - skip < step ? n - skip : step;
    }
    // and from there on those that begin up to each row, a lane's: 64 offsets at a time, as long as the last row is behind all of them
    int start = a.cu[seq], more = 64;
    for (int from = seq + 1; more == 64; from += 64) {
      const int offset = from + lane <= a.seqs ? a.cu[from + lane] : INT_MAX;
      int mine = 0;
      for (int r = 0; r < rows; ++r) {
        more = __popcll(__ballot(offset <= first + r));
        if (lane == r) mine = more;
      }
      const int last = __shfl(offset, mine > 0 ? mine - 1 : 0);
      if (mine > 0) start = last;
      seq += mine;
    }
    int page = -1, place = 0;
    const int row = first + lane;
    if (lane < rows && row < a.rows) {
      if (seq < a.seqs) {
        const int at = start < 0 || start > row ? 0 : row - start;
        const int idx = cells.c.per_page.quotient(at);
        page = idx < a.width ? a.block_table[seq * a.table_ld + idx] : -2;
        if ((unsigned)page >= (unsigned)cells.c.pages) page = -2;
        place = at - idx * cells.c.page_size;
      }
      pages[lane] = page, places[lane] = place;
    }
  }
  __syncthreads();
  const int left = a.rows - first < rows ? a.rows - first : rows;
  for (int i = threadIdx.x; i < left * (int)per_row.d; i += 256) {
    const int r = per_row.quotient(i), item = i - r * (int)per_row.d;
    const int h = units.quotient(item), ch = (item - h * (int)units.d) * CELLS::VEC;
    const bool value = h >= a.heads;
    const int head = value ? h - a.heads : h;
    const RowsOut dst = value ? a.v_out : a.k_out;
    unsigned short* to = (unsigned short*)dst.p + (first + r) * dst.token + head * dst.head + ch;
    if (pages[r] >= 0) {
      cells.move(value, pages[r], places[r], head, ch, to);
    } else {
      const unsigned fill = pages[r] == -1 ? 0u : T::pack2(__builtin_nanf(""), __builtin_nanf(""));
#pragma unroll
      for (int j = 0; j < CELLS::VEC; j += 8) *(u32x4*)(to + j) = u32x4{fill, fill, fill, fill};
    }
  }
}

template <class T, class CELLS>
hipError_t launch(const ReadArgs& a, const CELLS& cells, hipStream_t stream) {
  const int units = a.d / CELLS::VEC, per_row = 2 * a.heads * units;
  int rows = 1024 / per_row;
  rows = rows < 1 ? 1 : rows > MOST_ROWS ? MOST_ROWS : rows;
  while (rows > 1 && (a.rows + rows - 1) / rows < 512) rows /= 2;
  kv_read_kernel<T, CELLS><<<(a.rows + rows - 1) / rows, 256, 0, stream>>>(a, cells, Divisor(units), Divisor(per_row), rows);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv_read(int dtype, const ReadArgs& a, const PagedKv& cache, hipStream_t stream) {
  return dtype == FSW_BF16 ? launch<Bf16>(a, Cells16<Bf16>{cache}, stream) : launch<Fp16>(a, Cells16<Fp16>{cache}, stream);
}
hipError_t launch_kv_read8(int dtype, const ReadArgs& a, const PagedKv8& cache, hipStream_t stream) {
  return dtype == FSW_BF16 ? launch<Bf16>(a, Cells8<Bf16>{cache}, stream) : launch<Fp16>(a, Cells8<Fp16>{cache}, stream);
}

}  // namespace fsw
