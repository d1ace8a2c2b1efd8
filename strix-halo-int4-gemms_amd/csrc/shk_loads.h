// Loads from a uniform address, kept in scalar registers, plus a lane's 32-bit
// offset: left to itself the compiler keeps one 64-bit vector address for every
// load of a piece.  The address space is spelled out, since the empty asm hides
// where the pointer comes from and flat loads cannot be waited for one by one.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace shk {

typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef uint32_t any_u32 __attribute__((aligned(1)));  // of any alignment
typedef u2 any_u2 __attribute__((aligned(1)));
typedef u4 any_u4 __attribute__((aligned(1)));

// `offset` goes into the instruction: loads near each other share an address.
template <typename T>
__device__ __forceinline__ T load_at(const void* p, uint32_t mine, int offset = 0) {
  typedef __attribute__((address_space(1))) const uint8_t* global_bytes;
  global_bytes q = (global_bytes)p;
  asm("" : "+s"(q));
  return *(__attribute__((address_space(1))) const T*)(q + mine + offset);
}

}  // namespace shk
