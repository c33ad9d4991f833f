// Tiles of the dense products: which one a workgroup takes, and copies to LDS.
#pragma once
#include "gemm.h"

namespace lo {

// Workgroups are dealt round-robin to the 8 XCDs: each takes a range of tiles of its own, in groups of G token tiles by all columns, so that
// tiles at work at one time share rows and columns in its L2.
__device__ __forceinline__ bool dense_tile(int bid, int m_tiles, int n_tiles, int G, int &mt, int &nt) {
  const int total = m_tiles * n_tiles, per = (total + 7) / 8, id = (bid & 7) * per + (bid >> 3);
  if ((bid >> 3) >= per || id >= total) return false;
  const int first = id / (G * n_tiles) * G, in = id - first * n_tiles;
  const int size = m_tiles - first < G ? m_tiles - first : G;
  nt = in / size;
  mt = first + in - nt * size;
  return true;
}

__device__ __forceinline__ void copy16(brsrc r, int8_t *lds, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, lds, 16, voff, soff, 0, 0);
}
// All but this wave's newest N copies have landed and what it has read from LDS is there, and the workgroup meets.
template <int N> __device__ __forceinline__ void wait_barrier() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

} // namespace lo
