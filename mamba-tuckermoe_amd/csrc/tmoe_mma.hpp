// Primitives that the matrix kernels share: accumulators, LDS stages of 128-byte rows filled by
// direct loads, waits, and the order of tiles.
#pragma once

#include "tmoe_elem.hpp"

namespace tmoe {
namespace dev {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Accumulator element e of lane l holds row acc_row(l, e), column (l & 31).
__device__ __forceinline__ int acc_row(int lane, int e) {
  return 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3);
}
__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int e = 0; e < 16; ++e) z[e] = 0.f;
  return z;
}

typedef __attribute__((address_space(3))) void* lds_vptr;
typedef const __attribute__((address_space(1))) void* gbl_cvptr;

// s_waitcnt with vmcnt <= VM and lgkmcnt == 0 (gfx9 encoding: vmcnt in bits 3:0 and
// 15:14, expcnt 6:4, lgkmcnt 11:8).
template <int VM>
__device__ __forceinline__ void wait_vm_lds() {
  static_assert(VM >= 0 && VM < 64, "vmcnt range");
  __builtin_amdgcn_s_waitcnt((VM & 15) | ((VM >> 4) << 14) | (7 << 4));
}

// 24 wait states: more than the longest MFMA result latency a following VALU,
// LDS or memory instruction must respect (16-pass fp32 MFMAs need 18 or 19).
// Issued at the end of every main-loop K tile: the last MFMAs may sit in a
// conditional block, and the compiler's own padding before the copies it makes
// of the accumulators at the loop exit was found one wait state short there.
__device__ __forceinline__ void mfma_drain() { asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 7" ::: "memory"); }

// Work-group barrier that orders LDS traffic only; loads still in flight stay in
// flight. The empty asm statements keep the compiler from moving memory
// accesses across it.
__device__ __forceinline__ void lds_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);   // no instruction is scheduled across it
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// Chunk ch of tile row r lives at slot ch ^ ((r >> 1) & 7) of the row. A 32x32
// fragment read touches rows r0 .. r0 + 31 at one chunk; with this swizzle any 16
// consecutive of them fall on 16 distinct 16-byte bank groups (measured: no LDS
// bank conflicts, against half the LDS cycles lost with a (r & 7) swizzle).
__device__ __forceinline__ int lds_slot(int row, int ch) { return row * 8 + (ch ^ ((row >> 1) & 7)); }
// For a DMA of 8-row block blk, lane l writes slot 64 blk + l: row 8 blk + (l >> 3),
// physical chunk l & 7, which holds this logical chunk.
__device__ __forceinline__ int dma_chunk(int lane, int blk) {
  return (lane & 7) ^ ((lane >> 4) | ((blk & 1) << 2));
}

__device__ __forceinline__ int cmin_dev(int a, int b) { return a < b ? a : b; }

// Work-group -> tile order for 2-D grids launched as 1-D. Consecutive
// work-groups land on different XCDs (round robin over 8); this hands each XCD a
// contiguous run of tiles, row-major over (m, n), so the A rows of an m tile are
// fetched into one XCD's L2 and reused for all its n tiles.
__device__ __forceinline__ void tile_coords_of(int b, int n_tiles_n, int n_tiles, int& tm,
                                               int& tn) {
  const int per = n_tiles / 8;
  const int t = b < per * 8 ? (b % 8) * per + b / 8 : b;
  tm = t / n_tiles_n;
  tn = t - tm * n_tiles_n;
}

}  // namespace dev
}  // namespace tmoe
