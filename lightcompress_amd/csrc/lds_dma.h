// LDS-DMA and LDS reads of kernels that wait for their loads themselves (mla.hip, int4.hip).
#pragma once

#include "lcq_common.h"

namespace lcq {

typedef short v8s_t __attribute__((ext_vector_type(8)));
typedef short v4s_t __attribute__((ext_vector_type(4)));

// The DMA is inline asm, so the compiler neither orders LDS reads behind it (it cannot tell the
// stage being read from the one being filled, and puts a vmcnt(0) before every read) nor counts
// it; it has no result register. The kernel waits with s_waitcnt vmcnt before a stage is read,
// and with lgkmcnt(0) for its reads of a stage before that is filled again.
__device__ __forceinline__ uint32_t lds_addr(const void* p) {
  return (uint32_t)reinterpret_cast<uintptr_t>(p);
}
// 16 bytes per lane from base + off (base wave-uniform) to lds + 16 lane (lds wave-uniform)
__device__ __forceinline__ void dma16(uint32_t lds, const void* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
               :
               : "s"(lds), "v"(off), "s"(base)
               : "memory");
}
// the same from a 64-bit address of each lane's own
__device__ __forceinline__ void dma16_at(uint32_t lds, uint64_t addr) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
               :
               : "s"(lds), "v"(addr)
               : "memory");
}
// 4 bytes per lane from base + off (base wave-uniform) to lds + 4 lane
__device__ __forceinline__ void dma4(uint32_t lds, const void* base, uint32_t off) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2"
               :
               : "s"(lds), "v"(off), "s"(base)
               : "memory");
}
typedef __attribute__((address_space(3))) const v8s_t lds_v8s_t;
typedef __attribute__((address_space(3))) v4s_t lds_v4s_t;
__device__ __forceinline__ v8s_t lds_read16(uint32_t at) {
  return *reinterpret_cast<lds_v8s_t*>(at);
}
__device__ __forceinline__ v4s_t lds_read_tr(uint32_t at) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(reinterpret_cast<lds_v4s_t*>(at));
}

}  // namespace lcq
