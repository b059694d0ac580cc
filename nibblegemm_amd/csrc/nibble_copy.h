// Copies from memory straight into LDS, and the 16-bit type of a kernel.
#pragma once

#include "nibble_decode.h"

namespace nibble {

// One LDS-DMA copy of 16 bytes a lane: lane l's bytes, at byte voff + soff of
// [base, base + bytes) (beyond it: zeros), land at LDS byte address dst + 16 l;
// dst and soff are the same in every lane.  (The range check takes soff in
// without wrapping.)  Written as assembly because the compiler, knowing a
// pending copy, waits for it before every LDS read that it cannot tell apart;
// the kernel's own waits (vmcnt) order the copies.  No register is written; the
// addresses are read at issue.
__device__ __forceinline__ void lds_copy16(const void* base, uint32_t bytes, uint32_t dst,
                                           uint32_t voff, uint32_t soff = 0) {
  const uint64_t b = reinterpret_cast<uint64_t>(base);
  const u4_t rsrc = {static_cast<uint32_t>(b), static_cast<uint32_t>(b >> 32) & 0xffffu, bytes,
                     0x00020000u};
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               :
               : "s"(dst), "v"(voff), "s"(rsrc), "s"(soff)
               : "memory", "m0");
}
// The same for bytes that are read once (nt): a streaming read of 272 MB 6.9 TB/s, 6.0
// without.
__device__ __forceinline__ void lds_stream16(const void* base, uint32_t bytes, uint32_t dst,
                                             uint32_t voff) {
  const uint64_t b = reinterpret_cast<uint64_t>(base);
  const u4_t rsrc = {static_cast<uint32_t>(b), static_cast<uint32_t>(b >> 32) & 0xffffu, bytes,
                     0x00020000u};
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds"
               :
               : "s"(dst), "v"(voff), "s"(rsrc)
               : "memory", "m0");
}
// The same with 4 bytes a lane, landing at dst + 4 l.
__device__ __forceinline__ void lds_copy4(const void* base, uint32_t bytes, uint32_t dst,
                                          uint32_t voff, uint32_t soff = 0) {
  const uint64_t b = reinterpret_cast<uint64_t>(base);
  const u4_t rsrc = {static_cast<uint32_t>(b), static_cast<uint32_t>(b >> 32) & 0xffffu, bytes,
                     0x00020000u};
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, %3 offen lds"
               :
               : "s"(dst), "v"(voff), "s"(rsrc), "s"(soff)
               : "memory", "m0");
}

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (__attribute__((address_space(3))) void*)const_cast<void*>(p)));
}

// A 16-bit floating type: its 8-vectors and its 16x16x32 matrix product.
typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
struct Half {
  using type = _Float16;
  using vec8 = h8_t;
  static constexpr unsigned short kExponent = 0x7c00;  // of infinities and NaN
  static __device__ __forceinline__ f4_t mfma(vec8 a, vec8 b, f4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
struct Bfloat {
  using type = __bf16;
  using vec8 = b8_t;
  static constexpr unsigned short kExponent = 0x7f80;
  static __device__ __forceinline__ f4_t mfma(vec8 a, vec8 b, f4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

}  // namespace nibble
