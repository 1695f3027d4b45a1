// Pieces shared by the flash-attention kernels (attention.hip, mla.hip): MFMA and LDS images.
#pragma once

#include "lds_dma.h"

namespace lcq {

typedef __bf16 v8bf_t __attribute__((ext_vector_type(8)));
typedef _Float16 v8hf_t __attribute__((ext_vector_type(8)));
typedef float v16f_t __attribute__((ext_vector_type(16)));

// byte offset of 16-byte chunk ch (0..15) of row `row` in a [rows][128 x bf16] LDS image
__device__ __forceinline__ int img_off(int row, int ch) {
  return 256 * row + 16 * (ch ^ (((row & 3) << 2) | ((row >> 2) & 3)));
}

// Transposed 8-byte LDS read as inline asm: the builtin form makes the compiler put a
// vmcnt(0) before it (it cannot tell the read from the K / V stage being filled by LDS-DMA for
// the next tile), which serialised every tile behind the next tile's loads. The asm reads are
// invisible to the compiler's lgkmcnt tracking: tr_wait() below waits for them explicitly and
// ties their results, so no consumer is scheduled above the wait.
__device__ __forceinline__ v4s_t tr_read(const char* lds, int byte_off) {
  v4s_t r;
  const uint32_t addr = (uint32_t)reinterpret_cast<uintptr_t>(lds + byte_off);
  asm volatile("ds_read_b64_tr_b16 %0, %1" : "=v"(r) : "v"(addr) : "memory");
  return r;
}

__device__ __forceinline__ void tr_wait(v4s_t (&lo)[4], v4s_t (&hi)[4]) {
  asm volatile("s_waitcnt lgkmcnt(0)"
               : "+v"(lo[0]), "+v"(lo[1]), "+v"(lo[2]), "+v"(lo[3]), "+v"(hi[0]), "+v"(hi[1]),
                 "+v"(hi[2]), "+v"(hi[3])
               :
               : "memory");
}

template <int DT = LCQ_BF16>
__device__ __forceinline__ v16f_t mfma32(v8s_t a, v8s_t b, v16f_t c) {
  if constexpr (DT == LCQ_BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8bf_t, a),
                                                   __builtin_bit_cast(v8bf_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8hf_t, a),
                                                  __builtin_bit_cast(v8hf_t, b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
  typedef __bf16 v2bf_t __attribute__((ext_vector_type(2)));
  typedef float v2f_t __attribute__((ext_vector_type(2)));
  const v2bf_t hv = __builtin_convertvector((v2f_t){a, b}, v2bf_t);
  return __builtin_bit_cast(uint32_t, hv);
}

// two floats rounded to DT (nearest even), packed
template <int DT>
__device__ __forceinline__ uint32_t pack_dt(float a, float b) {
  if constexpr (DT == LCQ_BF16) return pack_bf16(a, b);
  typedef _Float16 v2hf_t __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, (v2hf_t){(_Float16)a, (_Float16)b});
}

// value of lane ^ 32 (the other half of a 32-lane query block): v_permlane32_swap, a VALU op,
// where __shfl_xor lowers to ds_bpermute (an LDS round trip and an lgkmcnt wait per call)
__device__ __forceinline__ float other_half(float v, int h) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                  false);
  return __uint_as_float(h ? r[0] : r[1]);
}

typedef __attribute__((address_space(3))) void lds_void_t;

// buffer descriptor of the 2 GB behind a wave-uniform pointer
__device__ __forceinline__ __amdgpu_buffer_rsrc_t head_rsrc(const uint16_t* p) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  void* q = reinterpret_cast<void*>(((uint64_t)hi << 32) | lo);
  return __builtin_amdgcn_make_buffer_rsrc(q, (short)0, 0x7fffffff, 0x00020000);
}

}  // namespace lcq
