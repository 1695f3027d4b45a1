// Fragments of the 4-bit weight kernels (int4.hip): packed words -> MFMA operands.
//
// A code c (0..15) becomes the float 16 + c by placing its four bits at the top of the mantissa of
// 16.0 (bf16 0x4180 | c << 3, fp16 0x4c00 | c << 6): exact, one shift and one and-or for two
// codes. With u = 16 + c the product with the weight (c - z) s of one group is
//   s * ( sum_k x_k u_k  -  (16 + z) sum_k x_k ),
// so a group costs its MFMAs, the sum of its x (one more MFMA against ones, shared by all the
// columns of a wave) and one fp32 multiply-add per output. The codes stay exact; the offset of
// 16 costs at most 2 more bits of the fp32 sum than a signed code would.
#pragma once

#include "lds_dma.h"

namespace lcq {

typedef short i4_v8s __attribute__((ext_vector_type(8)));
typedef __bf16 i4_v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 i4_v8h __attribute__((ext_vector_type(8)));
typedef float i4_v4f __attribute__((ext_vector_type(4)));
typedef uint32_t i4_v4u __attribute__((ext_vector_type(4)));

template <int DT>
__device__ __forceinline__ i4_v4f i4_mfma(i4_v4u a, i4_v4u b, i4_v4f c) {
  if constexpr (DT == LCQ_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(i4_v8bf, a),
                                                   __builtin_bit_cast(i4_v8bf, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(i4_v8h, a),
                                                  __builtin_bit_cast(i4_v8h, b), c, 0, 0, 0);
}

// 1.0 in both halves
template <int DT>
constexpr uint32_t i4_ones = DT == LCQ_BF16 ? 0x3f803f80u : 0x3c003c00u;

// The mask and the base of a pair of codes, in a vector and a scalar register: as literals the and
// and the or would be two instructions (one instruction takes no literal and one scalar)
template <int DT>
struct I4Const {
  uint32_t mask = DT == LCQ_BF16 ? 0x00780078u : 0x03c003c0u;
  uint32_t base = DT == LCQ_BF16 ? 0x41804180u : 0x4c004c00u;
  __device__ __forceinline__ I4Const() {
    asm volatile("" : "+v"(mask));
    asm volatile("" : "+s"(base));
  }
};

// nibbles P and P + 4 of w as 16 + code in the low and high half (P = 0..3)
template <int DT, int P>
__device__ __forceinline__ uint32_t i4_pair(uint32_t w, const I4Const<DT>& k) {
  constexpr int sh = (DT == LCQ_BF16 ? 3 : 6) - 4 * P;  // to the top of the mantissa
  if constexpr (sh >= 0) return ((w << sh) & k.mask) | k.base;
  else return ((w >> -sh) & k.mask) | k.base;
}

// one word of 8 codes along k as a B fragment, elements in the order 0 4 1 5 2 6 3 7
template <int DT>
__device__ __forceinline__ i4_v4u i4_word(uint32_t w, const I4Const<DT>& k) {
  return i4_v4u{i4_pair<DT, 0>(w, k), i4_pair<DT, 1>(w, k), i4_pair<DT, 2>(w, k),
                i4_pair<DT, 3>(w, k)};
}

// nibble t of every half of four packed pairs
template <int DT>
__device__ __forceinline__ i4_v4u i4_nibble(i4_v4u v, int t, const I4Const<DT>& k) {
  auto f = [&](uint32_t w) {
    return t == 0   ? i4_pair<DT, 0>(w, k)
           : t == 1 ? i4_pair<DT, 1>(w, k)
           : t == 2 ? i4_pair<DT, 2>(w, k)
                    : i4_pair<DT, 3>(w, k);
  };
  return i4_v4u{f(v.x), f(v.y), f(v.z), f(v.w)};
}

// load from a wave-uniform base + a lane's 32-bit offset, as a global (not a flat) load: flat loads
// count against the LDS waits too
template <typename T>
__device__ __forceinline__ T gload(const void* base, uint32_t off) {
  typedef const __attribute__((address_space(1))) char gchar;
  typedef const __attribute__((address_space(1))) T gT;
  return *reinterpret_cast<gT*>(reinterpret_cast<gchar*>(reinterpret_cast<uint64_t>(base)) + off);
}
template <typename T>
__device__ __forceinline__ T gload_at(const void* p) {
  typedef const __attribute__((address_space(1))) T gT;
  return *reinterpret_cast<gT*>(reinterpret_cast<uint64_t>(p));
}

// 8 consecutive x values as an A fragment in that order
__device__ __forceinline__ i4_v4u i4_xorder(i4_v4u d) {
  return i4_v4u{__builtin_amdgcn_perm(d.z, d.x, 0x05040100u),
                __builtin_amdgcn_perm(d.z, d.x, 0x07060302u),
                __builtin_amdgcn_perm(d.w, d.y, 0x05040100u),
                __builtin_amdgcn_perm(d.w, d.y, 0x07060302u)};
}

// AutoAWQ words hold 8 columns of one k: 16 bits of a word are 4 columns. Four B fragments (4
// tiles, 64 columns) come from two transposed LDS reads (ds_read_b64_tr_b16) of the words as they
// lie: lane c of a 16-lane group gets 16-bit column c of 4 rows (k) each, in packed pairs. Its
// tile t is nibble t of them: column 8 (c / 2) + 2 t + c % 2.
__device__ __forceinline__ int i4_awq_column(int c, int t) { return 8 * (c >> 1) + 2 * t + (c & 1); }

// XOR of the 16-byte chunks of 256-byte LDS rows: conflict-free for 16 rows at one chunk
__device__ __forceinline__ int i4_swz(int row) { return ((row & 3) << 2) | ((row >> 2) & 3); }

// 4 x 4 transpose of words between the lanes q = 0..3 of a row (lane = 16 q + row)
__device__ __forceinline__ i4_v4u i4_transpose(i4_v4u v) {
  auto p = __builtin_amdgcn_permlane32_swap(v.x, v.z, false, false);
  v.x = p[0]; v.z = p[1];
  p = __builtin_amdgcn_permlane32_swap(v.y, v.w, false, false);
  v.y = p[0]; v.w = p[1];
  p = __builtin_amdgcn_permlane16_swap(v.x, v.y, false, false);
  v.x = p[0]; v.y = p[1];
  p = __builtin_amdgcn_permlane16_swap(v.z, v.w, false, false);
  v.z = p[0]; v.w = p[1];
  return v;
}

}  // namespace lcq
