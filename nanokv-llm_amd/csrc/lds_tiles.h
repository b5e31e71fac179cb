// K/V tiles in LDS for the kernels that attend with many query rows (prefill.hip,
// diff_prefill.hip): rows fetched straight into LDS, their 16-byte chunks permuted so that the K
// row reads and the V transpose reads are free of bank conflicts.
#pragma once

#include "nkv_common.h"

// Asm that writes m0 says so, lest the compiler take a value of its own in it for kept; clang warns of
// every reserved register in such a list.
#pragma clang diagnostic ignored "-Winline-asm"

namespace nkv {

// XOR applied to the 16-byte chunk index of LDS row r (even: chunk pairs stay together).
// Keeps the K row reads and the V transpose reads free of bank conflicts: 2*(r & 7) for
// 256- and 512-byte rows, 2*((r >> 1) & 3) for 128-byte rows (two rows per bank line).
template <int D>
__device__ __forceinline__ int chunk_swz(int r) {
  if constexpr (D == 64) return 2 * ((r >> 1) & 3);
  else return 2 * (r & 7);
}

typedef __attribute__((address_space(3))) u32x4_t lds_u32x4_t;
typedef int32_t i32x4_t __attribute__((ext_vector_type(4)));

// Raw buffer descriptor over [base, base + bytes): loads past `bytes` return 0.
__device__ __forceinline__ i32x4_t buffer_desc(const void* base, uint32_t bytes) {
  const uint64_t a = (uint64_t)(uintptr_t)base;
  return i32x4_t{__builtin_amdgcn_readfirstlane((int32_t)(uint32_t)a),
                 __builtin_amdgcn_readfirstlane((int32_t)((a >> 32) & 0xffffu)),
                 __builtin_amdgcn_readfirstlane((int32_t)bytes), kBufferFlags};
}
// The start of asm that loads into LDS: m0, which the load takes its LDS address from, and the wait states
// that the compiler puts before a load of its own but not into asm: one after m0 is written, five after a
// vector instruction (readfirstlane above, or the reload of a spilled register) wrote a word of the
// descriptor. Prompts of 1500 and 2900 (bf16, Hq 32, Hk 8, D 128) take 33.4 and 77.8 us with the five, 33.1
// and 77.2 with the one alone, 33.2 and 78.6 with four loads in a block behind one wait of five.
#define NKV_LDS_AT "s_mov_b32 m0, %0\n\ts_nop 4\n\t"
// 16 bytes per lane from desc+voff into LDS at lds_addr + 16 * lane. Written as
// asm so that the compiler does not add a wait for it before every barrier;
// the ring's own s_waitcnt (vmcnt) orders it.
__device__ __forceinline__ void load_to_lds(i32x4_t desc, uint32_t lds_addr, uint32_t voff) {
  asm volatile(NKV_LDS_AT "buffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"(lds_addr), "v"(voff), "s"(desc)
               : "memory", "m0");
}

}  // namespace nkv
