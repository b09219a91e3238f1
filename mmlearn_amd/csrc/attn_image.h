// LDS images of 64-column tiles of 2-byte values, shared by the attention kernels: rows of 128 bytes whose 16-byte chunks are XOR-swizzled
// so that row reads (ds_read_b128) and transposed reads (ds_read_b64_tr_b16) are both free of bank conflicts, filled by LDS-DMA.
#pragma once
#include "common.h"

namespace mmk {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16_t bf16x8 __attribute__((ext_vector_type(8)));
typedef bf16_t bf16x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float att_exp2(float x) { return __builtin_amdgcn_exp2f(x); }


// ---- LDS image of a [rows][64] bf16 tile: 128-byte rows, the 16-byte chunk index XORed with img_swz(row).
// img_swz = bit-reversed (row>>1)&7: rows 2t, 2t+1 keep their 128-B bank offset from the row parity, the 8 row pairs of
// a ds_read_b128 lane group land in 8 different chunks (row reads conflict-free), and rows i, i+2 of an aligned 4-row
// block sit in opposite 64-B halves (transposed reads conflict-free).
__device__ __forceinline__ int img_swz(int row) {
  const int t = row >> 1;
  return ((t & 1) << 2) | (t & 2) | ((t >> 2) & 1);
}

// One LDS-DMA piece: 64 lanes x 16 B from per-lane global addresses to 1 KiB of LDS at the wave-uniform byte address
// `lds_addr`.  Written as inline asm (what the __builtin_amdgcn_global_load_lds builtin emits) so that the compiler does
// not track it: with the builtin, every later LDS read that might alias the destination gets a compiler-inserted
// s_waitcnt vmcnt(0), which would stall the compute of item n on the prefetch of item n+1.  The kernels order these
// writes themselves (s_waitcnt vmcnt(0) + barrier before the first read of an image); pieces are issued BEFORE any
// compiler-visible load of the same phase so the compiler's own vmcnt counts stay conservative.
__device__ __forceinline__ void lds_dma16(const void* sbase, uint32_t voff, uint32_t lds_addr) {
  // scalar 64-bit base + 32-bit per-lane byte offset: one VGPR of addressing per image instead of a pointer per piece
  const uint64_t pb = reinterpret_cast<uint64_t>(sbase);
  const uint64_t ps = ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(pb >> 32)) << 32) |
                      (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)pb);
  sbase = reinterpret_cast<const void*>(ps);
  lds_addr = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds_addr);
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" : : "v"(voff), "s"(sbase), "s"(lds_addr) : "memory");
}
__device__ __forceinline__ uint32_t lds_addr_of(const char* p) {
  return (uint32_t)(uintptr_t)((const __attribute__((address_space(3))) char*)p);
}

// s_waitcnt vmcnt(0) as the BUILTIN (expcnt / lgkmcnt fields left at their maxima): unlike an asm statement the
// compiler's wait-count bookkeeping sees it, so it knows every earlier load has landed and inserts no vmcnt of its own
// in the compute phase -- vmcnt is in-order, and any such wait would also wait for the prefetch issued after it.
__device__ __forceinline__ void wait_vmem_all() { __builtin_amdgcn_s_waitcnt(0x0F70); }

// MFMA operands out of an image.  k along the 64 COLUMNS: lane (r, h) takes row `row`, elements 16kk + 8h .. +7, one
// ds_read_b128 at  row * 128 + (((2 kk + h) ^ img_swz(row)) << 4).  k along the ROWS (transposed use of the same image):
// for the 32x32x16 A operand X^T[c][k] with c = 32 ct + (lane & 31) and the accumulator-as-operand k order, the lane
// needs column c of rows r0 .. r0+3 and r0+8 .. r0+11 (r0 = 16 s + 4 h + tile base): two ds_read_b64_tr_b16, for which
// lane 4q + p of each 16-lane group supplies the address of row r0 + q, columns 4p .. 4p+3 of the group's 4 x 16 block
// (chunk 4 ct + 2 (lane>>4 & 1) + (p >> 1), byte 8 (p & 1)) and receives column (lane & 15) of the four rows.
// Per-lane byte offsets into an image that do not depend on the 32-row tile: a tile adds 4096 B, the second k-step of
// a transposed fragment (rows +16) adds 2048 B, because img_swz only looks at (row >> 1) & 7.  Computing them once
// keeps the integer address arithmetic out of the MFMA loops (the loops were VALU-issue bound without this).
struct ImgLane {
  int row[4];    // row fragment kk of row 32t + (lane & 31)             = img + 4096 t + row[kk]
  int tr[2][2];  // transposed half u of k-step s, column tile ct        = img + 4096 t + 2048 s + tr[u][ct]
};
__device__ __forceinline__ ImgLane img_lane(int lane) {
  ImgLane o;
  const int r = lane & 31, h = lane >> 5;
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) o.row[kk] = r * 128 + (((2 * kk + h) ^ img_swz(r)) << 4);
  const int li = lane & 15, q = li >> 2, p = li & 3;
#pragma unroll
  for (int u = 0; u < 2; ++u)
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
      const int row = 4 * h + 8 * u + q;
      const int ch = 4 * ct + 2 * ((lane >> 4) & 1) + (p >> 1);
      o.tr[u][ct] = row * 128 + ((ch ^ img_swz(row)) << 4) + 8 * (p & 1);
    }
  return o;
}
__device__ __forceinline__ bf16x8 lds_row_frag(const char* p) { return *reinterpret_cast<const bf16x8*>(p); }
__device__ __forceinline__ bf16x8 lds_tr_frag(const char* img, const ImgLane& il, int tile_s_off, int ct) {
  typedef short s4 __attribute__((ext_vector_type(4)));
  const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(img + tile_s_off + il.tr[0][ct]));
  const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(img + tile_s_off + il.tr[1][ct]));
  typedef short s8 __attribute__((ext_vector_type(8)));
  s8 f;
  f[0] = lo[0]; f[1] = lo[1]; f[2] = lo[2]; f[3] = lo[3];
  f[4] = hi[0]; f[5] = hi[1]; f[6] = hi[2]; f[7] = hi[3];
  return __builtin_bit_cast(bf16x8, f);
}

}  // namespace mmk
