// Loads from device memory straight to LDS.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace dz {

// 16 bytes a lane to LDS, 1,024 consecutive bytes from address `lds` on (the same for the whole wave), from
// base + offset or from p. In assembly, so that the compiler, which cannot tell the slabs' places apart
// from one round of the loop to the next, does not wait for every load before it reads LDS; the caller waits.
// (M0 cannot be reserved by a statement. Nothing else here uses it: tests/test_head_asm.py looks for it in
// the generated code.)
template <bool ONCE>
__device__ __forceinline__ void to_lds(const void* base, uint32_t offset, uint32_t lds) {
  if (ONCE) asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"s"(lds), "v"(offset), "s"(base) : "memory");
  else asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}
__device__ __forceinline__ void to_lds(const void* p, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory");
}

}  // namespace dz
