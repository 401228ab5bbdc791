// Loads from a buffer straight into LDS, and their waits.
#pragma once
#include "common.h"

#define LDS_AS __attribute__((address_space(3)))

namespace psgdk {

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));

// make_rsrc's words, in scalar registers
__device__ __forceinline__ i32x4_t rsrc_words(const void* p, long long bytes) {
  const uint64_t at = (uint64_t)(uintptr_t)p;
  const int n = bytes > 0x7fffffffLL ? 0x7fffffff : bytes < 0 ? 0 : (int)bytes;
  return i32x4_t{__builtin_amdgcn_readfirstlane((int)at), __builtin_amdgcn_readfirstlane((int)(at >> 32) & 0xffff),
                 __builtin_amdgcn_readfirstlane(n), 0x00020000};
}
// 16 bytes a lane from the buffer to LDS at `lds` (wave-uniform) + 16 lane; lanes beyond the buffer write zeros. Not the
// builtin: with it the compiler waits for every such load before any LDS read. The waits are load_wait's.
__device__ __forceinline__ void load_lds(i32x4_t rs, int voff, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(voff), "s"(rs), "s"(lds)
               : "memory");
}
// the same with 4 bytes a lane
__device__ __forceinline__ void load_lds4(i32x4_t rs, int voff, unsigned lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dword %0, %1, 0 offen lds" ::"v"(voff), "s"(rs), "s"(lds)
               : "memory");
}
// all but the newest N loads into LDS of this wave have arrived, its LDS reads are done, and so for the whole workgroup
template <int N>
__device__ __forceinline__ void load_wait() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

}  // namespace psgdk
