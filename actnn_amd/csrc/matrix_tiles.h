// What the matrix kernels over 8-bit tokens share: loads from memory straight into LDS, LDS by its addresses, waits and loops
// that are counted at compile time.
#pragma once

#include "device_utils.h"

namespace actnn {

// f(Const<0>{}) .. f(Const<N - 1>{})
template <int N> struct Const { static constexpr int value = N; };
template <int N, typename F> ACTNN_DEV void for_each(F&& f) {
  if constexpr (N > 0) {
    for_each<N - 1>(f);
    f(Const<N - 1>{});
  }
}

typedef __attribute__((address_space(3))) uint8_t* lds_ptr_t;
ACTNN_DEV uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const uint8_t*)p;
}
template <typename V> ACTNN_DEV V lds_load(uint32_t address) {
  return *reinterpret_cast<const __attribute__((address_space(3))) V*>((lds_ptr_t)(uintptr_t)address);
}
template <typename V> ACTNN_DEV void lds_store(uint32_t address, V v) {
  *reinterpret_cast<__attribute__((address_space(3))) V*>((lds_ptr_t)(uintptr_t)address) = v;
}

// 16 (4) bytes a lane from a base that the wave shares, plus the lane's offset, to LDS: lane l's at lds + 16 l (4 l).  They are
// asynchronous: the kernel counts them itself and waits for all but the last n.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
ACTNN_DEV void load_rows(const void* base, uint32_t lane_bytes, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               : : "s"(lds), "v"(lane_bytes), "s"(base) : "memory", "m0");
}
ACTNN_DEV void load_words(const void* base, uint32_t lane_bytes, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
               : : "s"(lds), "v"(lane_bytes), "s"(base) : "memory", "m0");
}
#pragma clang diagnostic pop
// what s_waitcnt takes to wait for LDS and for all but the last n loads
constexpr int waitcnt_all_but(int n) { return (n & 15) | 7 << 4 | (n >> 4) << 14; }

// between writes and reads of the same wave: LDS operations of a wave complete in order
ACTNN_DEV void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// A launch counts its work items in 32 bits: blocks of 256 threads that one takes.
constexpr int64_t kMostBlocks = 0xffffff;

}  // namespace actnn
