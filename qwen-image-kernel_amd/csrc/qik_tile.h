// What the tiled products share: copies from global memory straight into LDS,
// the buffer resources that bound them, and the wait for them.
#ifndef QIK_TILE_H
#define QIK_TILE_H

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace qik_tile {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

typedef __attribute__((address_space(3))) void* lds_ptr_t;

#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
// 64 lanes x 16 B global -> LDS (buffer_load_dwordx4 ... lds): lane l's 16
// bytes land at LDS byte lds_addr + 16*l.  Asm, so the compiler neither moves
// the fragment reads around it nor waits for it; the main loop waits for the
// copies itself (vmcnt) before the barrier that publishes a stage.
__device__ __forceinline__ void dma16(u32x4 rsrc, uint32_t lds_addr, uint32_t voff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :: "s"(lds_addr), "v"(voff), "s"(rsrc) : "m0");
}
// the same with 4 bytes a lane: 256 contiguous bytes of LDS
__device__ __forceinline__ void dma4(u32x4 rsrc, uint32_t lds_addr, uint32_t voff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
               :: "s"(lds_addr), "v"(voff), "s"(rsrc) : "m0");
}
#pragma clang diagnostic pop

// Wave-uniform buffer resource over [base, base + bytes): loads at or past
// `bytes` return zeros.
__device__ __forceinline__ u32x4 rsrc_words(const unsigned char* base, uint32_t bytes) {
  const uint64_t a = (uint64_t)(uintptr_t)base;
  return u32x4{(uint32_t)a, (uint32_t)(a >> 32) & 0xffffu, bytes, 0x00020000u};
}

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  static_assert(N >= 0 && N < 64, "vmcnt field");
  // vmcnt in bits 3:0 and 15:14, expcnt (7) and lgkmcnt (63) left alone
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (0x7 << 4) | (0x3f << 8));
}

}  // namespace qik_tile

#endif  // QIK_TILE_H
