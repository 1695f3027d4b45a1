// Products with 4-bit packed weights and group scales (gfx950, bf16 / fp16 MFMA): the forward of
// the deployed linears (VllmRealQuantLinear / AutoawqRealQuantLinear buffers) for one matrix and
// for an MoE layer's routed experts.
//
//   y[m, n] = sum_k x[m, k] (c[n, k] - z[n, k / g]) s[n, k / g]  (+ bias[n])
//
// vLLM layout: words [N, K/8] of 8 codes along k (nibble i = code of k + i), z = 8, s [N, K/g].
// AutoAWQ layout: words [K, N/8] of 8 codes along n (nibble i = column {0,2,4,6,1,3,5,7}[i]),
// z packed the same [K/g, N/8], s [K/g, N]. Codes and zero points are exact in the products
// (int4_common.h), sums are fp32, the result is rounded once.
//
// Both layouts are read as they were deployed: no second copy of the weights is made or kept.
#define LCQ_BF16_HW 1
#include <type_traits>

#include "int4_common.h"

namespace lcq {
namespace {

constexpr int LV = 0, LA = 1;  // vLLM, AutoAWQ

struct I4Args {
  const uint16_t* x;
  int64_t ldx;              // row stride of x (elements)
  int64_t m, n, k, group;
  const uint32_t* qw;       // one matrix (grouped: from the table)
  const uint16_t* sc;
  const uint32_t* qz;
  const uint16_t* bias;     // nullable [n]
  uint16_t* y;
  int64_t ldy;
  // grouped
  const int64_t* row_off;   // [G + 1], null = one matrix
  const int64_t* a_rows;    // nullable gather [m]
  const int64_t* wtab;      // [sets][G][3]
  int64_t x_rows;
  int G;
  bool wide_y;              // rows of y are 16-byte aligned
  float* part;              // [nsplit][m][n] partial sums, nsplit > 1
  int nsplit;               // one matrix: workgroups a column block's k is split over
  uint32_t gmul;            // floor(2^32 / (group / 32)) + 1: exact division of k / 32 by group / 32
};

// scale group of k (a multiple of 32, below 2^21): k / group
__device__ __forceinline__ uint32_t i4_group(const I4Args& a, uint32_t k) {
  return a.gmul == 0 ? k >> 5 : __umulhi(k >> 5, a.gmul);
}

template <typename P>
__device__ __forceinline__ const P* uni(const P* p) {  // a wave-uniform pointer in scalar registers
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  return reinterpret_cast<const P*>(((uint64_t)hi << 32) | lo);
}
__device__ __forceinline__ int64_t uni(int64_t v) {
  return (int64_t)reinterpret_cast<uint64_t>(uni(reinterpret_cast<const char*>(v)));
}

__device__ __forceinline__ float h2f(uint16_t h) {
  return (float)__builtin_bit_cast(_Float16, h);
}

// The rows [r0, r1) and the group of row tile `slot` when every group's rows are cut into tiles of
// bm rows; false past the last tile. Offsets are clamped to [0, m] and made monotone.
__device__ __forceinline__ bool i4_find(const I4Args& a, int slot, int bm, int64_t& r0,
                                        int64_t& r1, int& grp) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int g0 = 0; g0 < a.G; g0 += 64) {
    const int g = g0 + lane;
    int64_t lo = 0, hi = 0;
    if (g < a.G) {
      lo = min(max(a.row_off[g], (int64_t)0), a.m);
      hi = min(max(a.row_off[g + 1], lo), a.m);
    }
    const int t = (int)((hi - lo + bm - 1) / bm);
    int inc = t;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(inc, d);
      if (lane >= d) inc += o;
    }
    const int total = __shfl(inc, 63);
    if (slot < base + total) {
      const uint64_t hit = __ballot(slot < base + inc);
      const int l = __builtin_ctzll(hit);
      const int first = base + __shfl(inc - t, l);
      const int64_t glo = __shfl(lo, l), ghi = __shfl(hi, l);
      grp = __builtin_amdgcn_readfirstlane(g0 + l);
      r0 = uni(glo + (int64_t)(slot - first) * bm);
      r1 = uni(min(r0 + bm, ghi));
      return true;
    }
    base += total;
  }
  return false;
}

// one output: bias, or the SiLU product of the two sets; a row gathered from outside x is zero
template <int DT, int SETS>
__device__ __forceinline__ void i4_store(const I4Args& a, int64_t row, int64_t col, float v0,
                                         float v1) {
  float o = v0;
  if constexpr (SETS == 2) o = v0 / (1.f + expf(-v0)) * v1;
  if (a.bias) o += ld1<DT>(a.bias, col);
  if (a.a_rows && (a.a_rows[row] < 0 || a.a_rows[row] >= a.x_rows)) o = 0.f;
  st1<DT>(a.y + (a.row_off && SETS == 1 ? blockIdx.z * a.m * a.ldy : 0), row * a.ldy + col, o);
}

// column tiles of 16 per workgroup of the 16-row kernel: as many as leave about 200 workgroups (a
// tile more shares x's fragments and their order changes; measured at 8 x 14336 x 4096: 4 tiles
// 10.9 us, 2 13.5, 1 19.1; at 1 x 4096 x 4096: 1 tile 5.2 us, 2 6.1, 4 8.1). Of groups n is all
// their columns (16 experts of 2048: 4 tiles 22 us, 1 38)
inline int i4_few_tiles(int layout, int64_t n) {
  return layout == LA || n >= 12288 ? 4 : n >= 6144 ? 2 : 1;
}

// this wave's weight pointers: one matrix, or the group's entry of the table
template <int SETS>
__device__ __forceinline__ void i4_weights(const I4Args& a, int grp, const uint32_t* (&qw)[SETS],
                                           const uint16_t* (&sc)[SETS],
                                           const uint32_t* (&qz)[SETS]) {
#pragma unroll
  for (int s = 0; s < SETS; ++s) {
    if (a.row_off) {
      const int64_t* t = a.wtab + ((int64_t)(SETS == 1 ? blockIdx.z : s) * a.G + grp) * 3;
      qw[s] = uni(reinterpret_cast<const uint32_t*>(t[0]));
      sc[s] = uni(reinterpret_cast<const uint16_t*>(t[1]));
      qz[s] = uni(reinterpret_cast<const uint32_t*>(t[2]));
    } else {
      qw[s] = a.qw;
      sc[s] = a.sc;
      qz[s] = a.qz;
    }
  }
}

// Column block of a workgroup: the dispatcher places workgroup p on XCD p % 8; neighbouring blocks
// go to one XCD, so the cache lines they share (AutoAWQ: 16 NT columns are 8 NT bytes of a row of
// words) are fetched into one L2.
__device__ __forceinline__ int i4_block(int p, int n) {
  const int xcd = p & 7, q8 = n >> 3, r8 = n & 7;
  return (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (p >> 3);
}

// Byte offsets of this lane's columns in the (wave-uniform) weight, scale and zero arrays: 32 bits,
// the entry points refuse a weight past 4 GB. NT column tiles of 16 per set; AutoAWQ: NT 4.
template <int LAYOUT, int NT>
struct I4Cols {
  uint32_t wo[LAYOUT == LV ? NT : 1];  // vLLM: the tiles' rows; AutoAWQ: this lane's DMA source
  uint32_t so, zo, ldw, lds;
  bool wide;                           // AutoAWQ: 16-byte DMA (rows of words 16-byte aligned)

  __device__ __forceinline__ void init(const I4Args& a, int64_t n0, int lane) {
    const int c = lane & 15, q = lane >> 4;
    if constexpr (LAYOUT == LV) {
      ldw = (uint32_t)(a.k / 2);
      lds = (uint32_t)(a.k / a.group * 2);
#pragma unroll
      for (int t = 0; t < NT; ++t) wo[t] = (uint32_t)min(n0 + 16 * t + c, a.n - 1) * ldw;
      so = (uint32_t)min(n0 + 16 * min(q, NT - 1) + c, a.n - 1) * lds;  // lane q: tile q's scale
      zo = 0;
      wide = true;
    } else {
      ldw = (uint32_t)(a.n / 2);
      lds = (uint32_t)(a.n * 2);
      wide = a.n % 32 == 0;
      // a stage row is 32 bytes: two lanes of 16, or eight of 4
      wo[0] = wide ? (uint32_t)min(n0 / 2 + 16 * (lane & 1), a.n / 2 - 16) + (lane >> 1) * ldw
                   : (uint32_t)min(n0 / 2 + 4 * (lane & 7), a.n / 2 - 4) + (lane >> 3) * ldw;
      const uint32_t wc = (uint32_t)min(n0 / 8 + (c >> 1), a.n / 8 - 1);
      so = 16 * wc;
      zo = 4 * wc;
    }
  }
};

// A unit is 128 k; F scale groups to the unit (1: the group is a multiple of 128, 2: of 64, 4: of
// 32). Its scales and zero points as loaded:
// vLLM: lane (c, q) holds the scale of column tile q; AutoAWQ: the 8 scales of the lane's word
// column and its word of zero points.
template <int LAYOUT, int F>
struct I4Scales {
  uint32_t s[F][LAYOUT == LV ? 1 : 4];
  uint32_t z[LAYOUT == LV ? 1 : F];

  template <int NT>
  __device__ __forceinline__ void load(const I4Args& a, const I4Cols<LAYOUT, NT>& cols,
                                       const uint16_t* sc, const uint32_t* qz, int k0) {
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const uint32_t gi = i4_group(a, (uint32_t)min(k0 + 128 / F * f, (int)a.k - 32));
      if constexpr (LAYOUT == LV) {
        s[f][0] = gload<uint16_t>(sc, cols.so + 2 * gi);
      } else {
        const i4_v4u v = gload<i4_v4u>(sc, cols.so + gi * cols.lds);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[f][j] = v[j];
        z[f] = gload<uint32_t>(qz, cols.zo + gi * cols.ldw);
      }
    }
  }
  // scale and 16 + zero point of the lane's column of tile t
  __device__ __forceinline__ void get(int f, int t, int c, float& sv, float& zv) const {
    if constexpr (LAYOUT == LV) {
      sv = h2f((uint16_t)__shfl(s[f][0], 16 * t + c));
      zv = 24.f;
    } else {
      sv = h2f((uint16_t)(s[f][t] >> (c & 1 ? 16 : 0)));
      zv = 16.f + (float)((z[f] >> (4 * t + 16 * (c & 1))) & 15u);
    }
  }
};

// AutoAWQ: one unit's words of 64 columns into LDS, 128 rows of 32 bytes (rows past k re-read the
// last one)
__device__ __forceinline__ void i4_stage(const I4Args& a, const I4Cols<LA, 4>& cols,
                                         const uint32_t* qw, uint32_t lds, int k0, int lane) {
  const int k = (int)a.k;
  if (cols.wide) {
    const int r = lane >> 1;
#pragma unroll
    for (int j = 0; j < 4; ++j)
      dma16(lds + 1024 * j, qw,
            cols.wo[0] + (uint32_t)(min(k0 + 32 * j + r, k - 1) - r) * cols.ldw);
  } else {
    const int r = lane >> 3;
#pragma unroll
    for (int j = 0; j < 16; ++j)
      dma4(lds + 256 * j, qw,
           cols.wo[0] + (uint32_t)(min(k0 + 8 * j + r, k - 1) - r) * cols.ldw);
  }
}

// Few rows: 16 MT rows of x and NT column tiles of 16 (of each set) per workgroup, the units of 128
// k split over its W waves (and, one matrix only, over a.nsplit workgroups), every word used by
// one wave. vLLM words go straight from memory to the MFMA operands; AutoAWQ words through a
// wave's own LDS stage, whose transposed reads form the fragments. The waves' partial tiles are
// summed through LDS in a fixed order. What bounds it: one row, the latency of a wave's few units
// (1 x 4096 x 4096 5.5 us); many words, memory (64 experts' gate and up, 2048 x 7168: 4.2 TB/s);
// more rows, x's fragments, which every wave loads, and for AutoAWQ a unit's words, which nothing
// runs under (no PRE): 37 x 14336 x 4096 in 21-22 us, 1.5 TB/s, waves waiting 51 % of their cycles.
// AutoAWQ with PRE or groups of 64: the compiler does not see the waits of the word copies and adds
// one right behind them, before a unit's scales and x are requested.
template <int DT, int LAYOUT, int F, int MT, int NT, int SETS, int W>
struct I4Few {
  static constexpr int T = NT * SETS;
  static constexpr bool HALVE = W * MT * T > 64;  // partial tiles of all waves past 64 KB
  static constexpr int WR = HALVE ? W / 2 : W;
  // the next unit is loaded meanwhile, where its registers cost no occupancy that hides more (one
  // matrix of vLLM words, MT 1: 5.5 us without, 5.8 with; 64 experts' gate and up: 223 with, 228
  // without; AutoAWQ, MT 4, 8 waves: 25.5 without, 37.9 with)
  static constexpr bool PRE = MT == 1 ? LAYOUT == LA || SETS == 2 : LAYOUT == LV && W == 4;
  static constexpr int STAGE = LAYOUT == LA ? 4096 * SETS : 0;
  static constexpr int RED = WR * MT * T * 1024, STAGES = W * (PRE ? 2 : 1) * STAGE;
  static constexpr int LDS = RED > STAGES ? RED : STAGES;
};

template <int DT, int LAYOUT, int F, int MT, int NT, int SETS, int W>
__global__ __launch_bounds__(64 * W) void k_int4_few(I4Args a) {
  using C = I4Few<DT, LAYOUT, F, MT, NT, SETS, W>;
  constexpr int T = C::T, WR = C::WR, NB = C::PRE ? 2 : 1;
  extern __shared__ __attribute__((aligned(1024))) char i4_lds[];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & 15, q = lane >> 4;
  int64_t r0, r1;
  int grp = 0;
  if (a.row_off) {
    if (!i4_find(a, blockIdx.y, 16 * MT, r0, r1, grp)) return;
  } else {
    r0 = (int64_t)blockIdx.y * 16 * MT;
    r1 = min(r0 + 16 * MT, a.m);
  }
  const uint32_t* qw[SETS];
  const uint16_t* sc[SETS];
  const uint32_t* qz[SETS];
  i4_weights<SETS>(a, grp, qw, sc, qz);
  // this lane's rows of x (as the A operand: row lane & 15 of each tile); a row past the last one
  // or gathered from outside x reads some other row, and its sums are not stored as they are
  const uint16_t* xr[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    int64_t row = min(r0 + 16 * i + c, r1 - 1);
    if (a.a_rows) row = min(max(a.a_rows[row], (int64_t)0), a.x_rows - 1);
    xr[i] = a.x + row * a.ldx;
  }
  const int64_t n0 = (int64_t)i4_block(blockIdx.x, gridDim.x) * 16 * NT;
  I4Cols<LAYOUT, NT> cols;
  cols.init(a, n0, lane);
  const uint32_t stage = lds_addr(i4_lds) + w * NB * C::STAGE;
  // transposed reads: rows 8 q + (0..3) of the step, 8 bytes a lane
  const uint32_t tr = stage + 32 * (8 * q + (c >> 2)) + 8 * (c & 3);

  i4_v4f acc[MT][T];
  const i4_v4f zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int t = 0; t < T; ++t) acc[i][t] = zero;
  const i4_v4u ones = {i4_ones<DT>, i4_ones<DT>, i4_ones<DT>, i4_ones<DT>};
  const I4Const<DT> kc;

  const int nb = (int)((a.k + 127) / 128);
  const int sp = a.row_off ? 0 : blockIdx.z;
  const int u0 = nb * sp / a.nsplit, un = nb * (sp + 1) / a.nsplit - u0;
  const int b0 = u0 + un * w / W, b1 = u0 + un * (w + 1) / W;
  i4_v4u xf[NB][MT][4], wv[NB][SETS][LAYOUT == LV ? NT : 1];
  I4Scales<LAYOUT, F> scl[NB][SETS];
  auto load = [&](int slot, int b) {
    const int k0 = b * 128;
    if constexpr (LAYOUT == LA) {
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the stage's last reads are done
#pragma unroll
      for (int s = 0; s < SETS; ++s)
        i4_stage(a, cols, qw[s], stage + slot * C::STAGE + s * 4096, k0, lane);
    } else {
      // 16 bytes of a row: the words of k0 + 32 q .. + 31 (rows end on a multiple of 32 k)
      const uint32_t kw = F == 1 ? (uint32_t)(k0 / 2 + 16 * q)
                                 : (uint32_t)min(k0 + 32 * q, (int)a.k - 32) / 2;
#pragma unroll
      for (int s = 0; s < SETS; ++s)
#pragma unroll
        for (int t = 0; t < NT; ++t)
          wv[slot][s][t] = gload<i4_v4u>(qw[s], cols.wo[t] + kw);
    }
#pragma unroll
    for (int s = 0; s < SETS; ++s) scl[slot][s].load(a, cols, sc[s], qz[s], k0);
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      if constexpr (F == 1) {
        const uint16_t* p = xr[i] + (k0 + (LAYOUT == LA ? 8 * q : 32 * q));
#pragma unroll
        for (int j = 0; j < 4; ++j)
          xf[slot][i][j] = gload_at<i4_v4u>(p + (LAYOUT == LA ? 32 * j : 8 * j));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)  // steps past k are not computed
          xf[slot][i][j] = gload_at<i4_v4u>(xr[i] + (min(k0 + 32 * j, (int)a.k - 32) + 8 * q));
      }
    }
  };
  auto compute = [&](int slot, int b) {
    const int k0 = b * 128;
    if constexpr (LAYOUT == LV) {
      // natural k order where a scale group ends inside the unit, else the words as loaded: word
      // j of lane q holds k = 32 q + 8 j, and x follows
      if constexpr (F > 1) {
#pragma unroll
        for (int s = 0; s < SETS; ++s)
#pragma unroll
          for (int t = 0; t < NT; ++t) wv[slot][s][t] = i4_transpose(wv[slot][s][t]);
      }
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) xf[slot][i][j] = i4_xorder(xf[slot][i][j]);
    }
#pragma unroll
    for (int f = 0; f < F; ++f) {
      if (F > 1 && k0 + 128 / F * f >= a.k) break;
      i4_v4f xs[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        xs[i] = zero;
#pragma unroll
        for (int j = 4 / F * f; j < 4 / F * (f + 1); ++j)
          xs[i] = i4_mfma<DT>(xf[slot][i][j], ones, xs[i]);
      }
#pragma unroll
      for (int s = 0; s < SETS; ++s) {
        i4_v4u pk[LAYOUT == LA ? 4 / F : 1];
        if constexpr (LAYOUT == LA) {
          typedef uint32_t v2u_t __attribute__((ext_vector_type(2)));
#pragma unroll
          for (int j = 0; j < 4 / F; ++j) {
            const uint32_t at = tr + slot * C::STAGE + s * 4096 + 1024 * (4 / F * f + j);
            const v2u_t l = __builtin_bit_cast(v2u_t, lds_read_tr(at));
            const v2u_t h = __builtin_bit_cast(v2u_t, lds_read_tr(at + 128));
            pk[j] = i4_v4u{l.x, l.y, h.x, h.y};
          }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          i4_v4f g[MT];
#pragma unroll
          for (int i = 0; i < MT; ++i) g[i] = zero;
#pragma unroll
          for (int j = 0; j < 4 / F; ++j) {
            const i4_v4u bf = LAYOUT == LV
                                  ? i4_word<DT>(wv[slot][s][LAYOUT == LV ? t : 0][4 / F * f + j], kc)
                                  : i4_nibble<DT>(pk[LAYOUT == LA ? j : 0], t, kc);
#pragma unroll
            for (int i = 0; i < MT; ++i) g[i] = i4_mfma<DT>(xf[slot][i][4 / F * f + j], bf, g[i]);
          }
          float sv, zv;
          scl[slot][s].get(f, t, c, sv, zv);
#pragma unroll
          for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              acc[i][s * NT + t][r] = __fmaf_rn(sv, __fmaf_rn(-zv, xs[i][r], g[i][r]),
                                                acc[i][s * NT + t][r]);
        }
      }
    }
  };
  if constexpr (C::PRE) {
    if (b0 < b1) {
      load(0, b0);
      int b = b0;
      for (; b + 2 < b1; b += 2) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        load(1, b + 1);
        compute(0, b);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        load(0, b + 2);
        compute(1, b + 1);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (b + 1 < b1) load(1, b + 1);
      compute(0, b);
      if (b + 1 < b1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        compute(1, b + 1);
      }
    }
  } else {
    for (int b = b0; b < b1; ++b) {
      load(0, b);
      if constexpr (LAYOUT == LA) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      compute(0, b);
    }
  }
  typedef i4_v4f red_t[MT * T][64];
  red_t* red = reinterpret_cast<red_t*>(i4_lds);
  if constexpr (LAYOUT == LA) __syncthreads();  // the stages become the partial tiles
  if constexpr (C::HALVE) {
    if (w >= WR) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < T; ++t) red[w - WR][i * T + t][lane] = acc[i][t];
    }
    __syncthreads();
    if (w < WR) {
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int t = 0; t < T; ++t) {
          acc[i][t] += red[w][i * T + t][lane];
          red[w][i * T + t][lane] = acc[i][t];
        }
    }
  } else {
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int t = 0; t < T; ++t) red[w][i * T + t][lane] = acc[i][t];
  }
  __syncthreads();
  // outputs: element r of (tile, lane) is row r0 + 16 i + 4 q + r; the waves share the tiles
  for (int e = w; e < MT * NT; e += W) {
    const int i = e / NT, t = e - i * NT;
    const int64_t cc = n0 + (LAYOUT == LV ? 16 * t + c : i4_awq_column(c, t));
    if (cc >= a.n) continue;
    i4_v4f v[SETS];
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      v[s] = red[0][i * T + s * NT + t][lane];
#pragma unroll
      for (int x = 1; x < WR; ++x) v[s] += red[x][i * T + s * NT + t][lane];
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t row = r0 + 16 * i + 4 * q + r;
      if (row >= r1) continue;
      if (a.nsplit > 1) a.part[(sp * a.m + row) * a.n + cc] = v[0][r];
      else i4_store<DT, SETS>(a, row, cc, v[0][r], v[SETS - 1][r]);
    }
  }
}

// Many rows: 128 rows x 256 columns (of one set, or 128 of each of two) per workgroup, 8 waves. x
// goes through LDS in units of 128 k (three buffers, one barrier a unit); a wave unpacks its
// columns' words once per unit and walks its row tiles, reading x fragments one tile ahead and
// scaling a tile's products while the next one's run. vLLM: 128 x 32 a wave, words straight to
// registers, x put into the words' element order on its way to LDS. AutoAWQ: 64 x 64 a wave, words
// through LDS too (a transposed read gives 64 columns). The sums of x of the next unit's groups are
// formed one unit ahead, one row tile by each wave. What bounds it: of the time its CU is busy MFMA
// works 46 % and LDS 38 %, beside 3.0 other vector instructions to a product (half of those unpack
// and scale); waves wait 33 % of their cycles. 2048 x 14336 x 4096 in 274-290 us, 830-880 TF/s, 0.55
// of a plain bf16 product's rate of that width.
constexpr int TM = 128, TX = TM * 256, TW = 128 * 128;  // rows; bytes of an x, a word buffer

template <int LAYOUT>
constexpr int i4_tile_lds = 3 * TX + (LAYOUT == LA ? 3 * TW : 0) + 2 * 4 * TM * 4;

template <int DT, int LAYOUT, int F, int SETS>
__global__ __launch_bounds__(512, 2) void k_int4_tile(I4Args a) {
  extern __shared__ __attribute__((aligned(1024))) char i4_lds[];
  constexpr int MI = LAYOUT == LV ? 8 : 4, NI = LAYOUT == LV ? 2 : 4;  // 16 x 16 tiles of a wave
  constexpr int NC = 16 * NI / SETS, WC = 256 / SETS;  // columns of a set per wave, workgroup
  constexpr int NX = LAYOUT == LA ? 3 * TW : 0;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, q = lane >> 4;
  const int mh = LAYOUT == LV ? 0 : w >> 2, nw = LAYOUT == LV ? w : w & 3;
  const int nblk = (int)((a.n + WC - 1) / WC);
  // neighbouring workgroups share their weights (one matrix) or their rows (grouped)
  const int id = i4_block(blockIdx.x, gridDim.x);
  int64_t r0, r1;
  int grp = 0, nbk;
  if (a.row_off) {
    nbk = id % nblk;
    if (!i4_find(a, id / nblk, TM, r0, r1, grp)) return;
  } else {
    const int slots = gridDim.x / nblk;
    nbk = id / slots;
    r0 = (int64_t)(id % slots) * TM;
    r1 = min(r0 + TM, a.m);
  }
  const uint32_t* qw[SETS];
  const uint16_t* sc[SETS];
  const uint32_t* qz[SETS];
  i4_weights<SETS>(a, grp, qw, sc, qz);
  const int64_t n0 = (int64_t)nbk * WC + nw * NC;  // this wave's first column of a set
  const int k = (int)a.k, nb = (k + 127) / 128;
  const uint32_t lds0 = lds_addr(i4_lds), xs0 = lds0 + 3 * TX + NX;

  // ---- staging: this thread's 16-byte chunk of 4 rows of x (rows tid / 16 + 32 i; rows past the
  // last, or gathered from outside x, read another one and are not stored as they come)
  const uint16_t* xr[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    // LDS-DMA: a wave's instruction i fills rows 16 w + 4 i .. + 3
    int64_t row = min(r0 + (LAYOUT == LA ? 16 * w + 4 * i + q : (tid >> 4) + 32 * i), r1 - 1);
    if (a.a_rows) row = min(max(a.a_rows[row], (int64_t)0), a.x_rows - 1);
    xr[i] = a.x + row * a.ldx;
  }
  i4_v4u xg[4];
  auto x_load = [&](int u) {  // vLLM: to registers
#pragma unroll
    for (int i = 0; i < 4; ++i)
      xg[i] = gload_at<i4_v4u>(xr[i] + min(128 * u + 8 * c, k - 8));
  };
  auto x_store = [&](uint32_t buf) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = (tid >> 4) + 32 * i;
      *reinterpret_cast<i4_v4u*>(i4_lds + (buf - lds0) + 256 * row + 16 * (c ^ i4_swz(row))) =
          i4_xorder(xg[i]);
    }
  };
  // AutoAWQ: a word row of the buffer is 128 bytes: the 64 columns of wave 0, 1, 2, 3 (two sets: 32
  // columns of each), 16-byte chunks ch at ch ^ 2 ((row / 2) % 4)
  uint64_t wsrc = 0;
  uint32_t ldw = (uint32_t)(a.n / 2);
  if constexpr (LAYOUT == LA) {
    // a wave's instruction i fills rows 16 w + 8 i .. + 7; this lane's chunk of row lane / 8
    const int r = lane >> 3, ch = (lane & 7) ^ (((r >> 1) & 3) << 1);
    const int64_t at = (int64_t)nbk * (WC / 2);
    const int64_t byte = SETS == 2 ? at + 16 * (ch >> 1) : at + 16 * ch;
    wsrc = reinterpret_cast<uint64_t>(qw[SETS == 2 ? ch & 1 : 0]) + min(byte, a.n / 2 - 16);
  }
  auto dma = [&](int u, uint32_t xbuf, uint32_t wbuf) {  // AutoAWQ: x and words by LDS-DMA
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 16 * w + 4 * i + q;
      dma16_at(xbuf + 1024 * (4 * w + i),
               reinterpret_cast<uint64_t>(xr[i] + min(128 * u + 8 * (c ^ i4_swz(row)), k - 8)));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      dma16_at(wbuf + 1024 * (2 * w + i),
               wsrc + (uint64_t)min(128 * u + 16 * w + 8 * i + (lane >> 3), k - 1) * ldw);
  };
  // vLLM words and the scales of a unit; column tile t of vLLM is set t / (2 / SETS)
  uint32_t wo[NI], so[LAYOUT == LV ? NI : 1], zo = 0;
  const char* sp = nullptr;
  const char* zp = nullptr;
  const uint32_t lds_s = LAYOUT == LV ? (uint32_t)(a.k / a.group * 2) : (uint32_t)(a.n * 2);
  if constexpr (LAYOUT == LV) {
#pragma unroll
    for (int t = 0; t < NI; ++t) {
      const uint32_t row = (uint32_t)min(n0 + 16 * (SETS == 2 ? 0 : t) + c, a.n - 1);
      wo[t] = row * (uint32_t)(k / 2);
      so[t] = row * lds_s;
    }
  } else {
    const int s = SETS == 2 ? c >> 3 : 0;
    const uint32_t wc = (uint32_t)min(n0 / 8 + ((SETS == 2 ? c & 7 : c) >> 1), a.n / 8 - 1);
    so[0] = 16 * wc;
    zo = 4 * wc;
    sp = reinterpret_cast<const char*>(sc[s]);
    zp = reinterpret_cast<const char*>(qz[s]);
  }
  i4_v4u wv[LAYOUT == LV ? NI : 1];
  uint32_t sv4[F][LAYOUT == LV ? NI : 4], zv1[LAYOUT == LV ? 1 : F];
  auto w_load = [&](int u) {
    const int k0 = 128 * u;
    if constexpr (LAYOUT == LV) {
      const uint32_t kw = (uint32_t)min(k0 + 32 * q, k - 32) / 2;
#pragma unroll
      for (int t = 0; t < NI; ++t) wv[t] = gload<i4_v4u>(qw[SETS == 2 ? t : 0], wo[t] + kw);
    }
#pragma unroll
    for (int f = 0; f < F; ++f) {
      const uint32_t gi = i4_group(a, (uint32_t)min(k0 + 128 / F * f, k - 32));
      if constexpr (LAYOUT == LV) {
#pragma unroll
        for (int t = 0; t < NI; ++t)
          sv4[f][t] = gload<uint16_t>(sc[SETS == 2 ? t : 0], so[t] + 2 * gi);
      } else {
        const i4_v4u v = gload<i4_v4u>(sp, so[0] + gi * lds_s);
#pragma unroll
        for (int j = 0; j < 4; ++j) sv4[f][j] = v[j];
        zv1[f] = gload<uint32_t>(zp, zo + gi * ldw);
      }
    }
  };
  // x fragment of row tile i, k-step j. vLLM with F 1: word j of lane q holds k = 32 q + 8 j
  uint32_t xo[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    xo[j] = 256 * c + 16 * ((LAYOUT == LV && F == 1 ? 4 * q + j : 4 * j + q) ^ i4_swz(c));
  const i4_v4f zero = {0.f, 0.f, 0.f, 0.f};
  const i4_v4u ones = {i4_ones<DT>, i4_ones<DT>, i4_ones<DT>, i4_ones<DT>};
  const I4Const<DT> kc;
  // sums of row tile w, to the unit's sum buffer (vLLM: times -(16 + z), z = 8)
  auto x_sums = [&](int u, uint32_t buf) {
#pragma unroll
    for (int f = 0; f < F; ++f) {
      i4_v4f xs = zero;
#pragma unroll
      for (int j = 4 / F * f; j < 4 / F * (f + 1); ++j)
        if (F == 1 || 128 * u + 32 * j < k)
          xs = i4_mfma<DT>(__builtin_bit_cast(i4_v4u, lds_read16(buf + 4096 * w + xo[j])), ones, xs);
      if constexpr (LAYOUT == LV) xs *= -24.f;
      if (c == 0)
        *reinterpret_cast<i4_v4f*>(i4_lds + (xs0 - lds0) + ((u & 1) * 4 + f) * TM * 4 +
                                   (16 * w + 4 * q) * 4) = xs;
    }
  };

  i4_v4f acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int t = 0; t < NI; ++t) acc[i][t] = zero;

  uint32_t xb[3] = {lds0, lds0 + TX, lds0 + 2 * TX};
  uint32_t wb[3] = {lds0 + 3 * TX, lds0 + 3 * TX + TW, lds0 + 3 * TX + 2 * TW};
  if constexpr (LAYOUT == LA) {
    dma(0, xb[0], wb[0]);
    if (nb > 1) dma(1, xb[1], wb[1]);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  } else {
    x_load(0);
    x_store(xb[0]);
    x_load(min(1, nb - 1));
    x_store(xb[1]);
    x_load(min(2, nb - 1));
  }
  w_load(0);
  __syncthreads();
  x_sums(0, xb[0]);
  const uint32_t trl = 1024 * q + 128 * (c >> 2) +
                       16 * ((2 * nw + ((c & 3) >> 1)) ^ ((c >> 3) << 1)) + 8 * (c & 1);
  const uint32_t trh = (trl ^ 64) + 512;

  for (int u = 0; u < nb; ++u) {
    // the next unit's x (and words) and this one's sums are in LDS; the oldest buffer is free
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    i4_v4u wc4[LAYOUT == LV ? NI : 1];
    uint32_t sc4[F][LAYOUT == LV ? NI : 4], zc1[LAYOUT == LV ? 1 : F];
#pragma unroll
    for (int t = 0; t < (LAYOUT == LV ? NI : 0); ++t) wc4[t] = F == 1 ? wv[t] : i4_transpose(wv[t]);
#pragma unroll
    for (int f = 0; f < F; ++f) {
#pragma unroll
      for (int j = 0; j < NI; ++j) sc4[f][j] = sv4[f][j];
      if constexpr (LAYOUT == LA) zc1[f] = zv1[f];
    }
    if constexpr (LAYOUT == LA) {
      if (u + 1 < nb) w_load(u + 1);
      if (u + 2 < nb) dma(u + 2, xb[2], wb[2]);
    } else {
      if (u + 2 < nb) {
        x_store(xb[2]);
        x_load(min(u + 3, nb - 1));
      }
      if (u + 1 < nb) w_load(u + 1);
    }
    if (u + 1 < nb) x_sums(u + 1, xb[1]);
    constexpr int J = 4 / F;
    i4_v4u xf[2][J];
    i4_v4f xs[2], g[2][NI];
    // (the empty asm keeps a lane's addresses whole, so that tiles and groups are read at constant
    // offsets: the compiler would add up each address instead)
    uint32_t xa[4], sa = xs0 + (u & 1) * 4 * TM * 4 + 256 * mh + 16 * q;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      xa[j] = xb[0] + 16384 * mh + xo[j];
      asm volatile("" : "+v"(xa[j]));
    }
    asm volatile("" : "+v"(sa));
    auto fetch = [&](int f, int i) {
#pragma unroll
      for (int j = 0; j < J; ++j)
        xf[i & 1][j] = __builtin_bit_cast(i4_v4u, lds_read16(xa[J * f + j] + 4096 * i));
      xs[i & 1] = __builtin_bit_cast(i4_v4f, lds_read16(sa + f * TM * 4 + 64 * i));
    };
#pragma unroll
    for (int f = 0; f < F; ++f) {
      if (F > 1 && 128 * u + 128 / F * f >= k) break;
      fetch(f, 0);
      i4_v4u bf[NI][J];
      float s[NI], z[NI];
      if constexpr (LAYOUT == LA) {
        typedef uint32_t v2u_t __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const uint32_t at = wb[0] + 4096 * (J * f + j);
          const v2u_t l = __builtin_bit_cast(v2u_t, lds_read_tr(at + trl));
          const v2u_t h = __builtin_bit_cast(v2u_t, lds_read_tr(at + trh));
          const i4_v4u pk = {l.x, l.y, h.x, h.y};
#pragma unroll
          for (int t = 0; t < NI; ++t) bf[t][j] = i4_nibble<DT>(pk, t, kc);
        }
      }
#pragma unroll
      for (int t = 0; t < NI; ++t) {
        if constexpr (LAYOUT == LV) {
          s[t] = h2f((uint16_t)sc4[f][t]);
          z[t] = 0.f;
#pragma unroll
          for (int j = 0; j < J; ++j) bf[t][j] = i4_word<DT>(wc4[LAYOUT == LV ? t : 0][J * f + j], kc);
        } else {
          s[t] = h2f((uint16_t)(sc4[f][t] >> (c & 1 ? 16 : 0)));
          z[t] = -16.f - (float)((zc1[f] >> (4 * t + 16 * (c & 1))) & 15u);
        }
      }
#pragma unroll
      for (int i = 0; i <= MI; ++i) {
        if (i + 1 < MI) fetch(f, i + 1);
        if (i < MI) {
#pragma unroll
          for (int t = 0; t < NI; ++t)
            g[i & 1][t] = LAYOUT == LV ? xs[i & 1] : z[t] * xs[i & 1];
#pragma unroll
          for (int j = 0; j < J; ++j)
#pragma unroll
            for (int t = 0; t < NI; ++t)
              g[i & 1][t] = i4_mfma<DT>(xf[i & 1][j], bf[t][j], g[i & 1][t]);
        }
        if (i > 0) {
#pragma unroll
          for (int t = 0; t < NI; ++t)
#pragma unroll
            for (int r = 0; r < 4; ++r)
              acc[i - 1][t][r] = __fmaf_rn(s[t], g[(i - 1) & 1][t][r], acc[i - 1][t][r]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if constexpr (LAYOUT == LA) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const uint32_t x0 = xb[0], w0 = wb[0];
    xb[0] = xb[1]; xb[1] = xb[2]; xb[2] = x0;
    wb[0] = wb[1]; wb[1] = wb[2]; wb[2] = w0;
  }
  __syncthreads();
  // the wave's tile through LDS (its own 8 KB) to row-wise stores; chunks of 8 columns swizzled by
  // the row: 16 rows of a column spread over the banks
  constexpr int RB = 32 * NI, SW = RB / 16 - 1;  // bytes of a row, chunks - 1
  char* out = i4_lds + 8192 * w;
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 16 * i + 4 * q + r;
#pragma unroll
      for (int t = 0; t < (LAYOUT == LV ? NI / SETS : NI); ++t) {
        float o = acc[i][t][r];
        const int col = LAYOUT == LV ? 16 * t + c : i4_awq_column(c, t);
        if constexpr (SETS == 2) {
          const float up = LAYOUT == LV ? acc[i][1][r] : __shfl_xor(o, 8);
          o = o / (1.f + expf(-o)) * up;
        }
        if (a.bias) o += ld1<DT>(a.bias, min(n0 + col, a.n - 1));
        if (SETS == 1 || LAYOUT == LV || c < 8)
          st1<DT>(out + RB * row + 16 * ((col >> 3) ^ (row & SW)), col & 7, o);
      }
    }
  __syncthreads();
  constexpr int CPR = NC / 8;  // 16-byte chunks of a row
#pragma unroll
  for (int e = 0; e < MI * CPR / 4; ++e) {
    const int row = e * (64 / CPR) + lane / CPR, ch = lane % CPR;
    const int64_t gr = r0 + 64 * mh + row, col = n0 + 8 * ch;
    if (gr >= r1) continue;
    i4_v4u v = *reinterpret_cast<const i4_v4u*>(out + RB * row + 16 * (ch ^ (row & SW)));
    if (a.a_rows && (a.a_rows[gr] < 0 || a.a_rows[gr] >= a.x_rows)) v = i4_v4u{0, 0, 0, 0};
    uint16_t* yp = a.y + (a.row_off && SETS == 1 ? blockIdx.z * a.m * a.ldy : 0) + gr * a.ldy + col;
    if (a.wide_y && col + 8 <= a.n) {
      *reinterpret_cast<i4_v4u*>(yp) = v;
      continue;
    }
#pragma unroll
    for (int x = 0; x < 8; ++x)
      if (col + x < a.n) yp[x] = (uint16_t)(v[x >> 1] >> (16 * (x & 1)));
  }
}

// sum of the splits in split order, 4 columns a thread
template <int DT>
__global__ __launch_bounds__(256) void k_int4_join(I4Args a) {
  const int64_t n = a.m * a.n, at = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  for (int64_t e = at; e < min(at + 4, n); ++e) {
    float v = 0.f;
    for (int s = 0; s < a.nsplit; ++s) v += a.part[s * n + e];
    i4_store<DT, 1>(a, e / a.n, e % a.n, v, 0.f);
  }
}

// The 128-row kernel runs where its tiles cost less than k_int4_few's passes over the words. One
// matrix, k 4096: a round of 128 x 256 tiles over the chip takes 63 us however few rows they hold,
// k_int4_few about 25 us per 64 rows of 14336 columns (128 rows 51 us, 256 rows 95; of 4096
// columns 400 rows 49). Groups (2048 x 2048 each, sets 1 / 2): vLLM 48 rows each, 64 groups: 111 /
// 233 us against 140 / 252, but 16 groups leave CUs idle: 67 / 135 against 55 / 107, from 64 rows on
// 68 / 137 against 85 / 132; AutoAWQ, whose small kernel costs less: one set 64 rows 130 against
// 159, 48 rows 128 against 121; two sets 100 rows 394 against 346, 128 rows 394 against 412. Not
// for AutoAWQ weights whose rows of words are not 16-byte aligned (LDS-DMA).
bool i4_tile_one(int64_t m, int64_t n, int layout) {
  return !(layout == LA && n % 32) && m > 64 && (m + TM - 1) / TM * ((n + 255) / 256) >= 96;
}
bool i4_use_tile(const I4Args& a, int layout, int sets) {
  if (!a.row_off) return i4_tile_one(a.m, a.n, layout);
  if (layout == LA && a.n % 32) return false;
  const int64_t cols = sets == 2 ? 128 : 256, nblk = (a.n + cols - 1) / cols;
  const int64_t least = layout == LA ? (sets == 2 ? 120 : 56) : a.G * nblk >= 512 ? 40 : 64;
  return a.m >= least * a.G;
}

// How one matrix's k is split over workgroups (a function of the shape alone): where the blocks of
// rows and columns leave CUs without a workgroup, and up to 16 rows only where the waves have units
// enough to pay for the join. 1 x 4096 x 14336 AutoAWQ, 64 blocks: 16.5 us with 4 splits, 28.9
// without, 17.6 with 8; at k 4096 8.9 with 2, 7.7 without. 37 x 4096 x 14336: 25 us with 4, 54
// without, 31 with 8. 128 x 1024 x 4096: 14.5 us with 8, 23.6 without.
int i4_nsplit(int64_t m, int64_t n, int64_t k, int layout) {
  if (i4_tile_one(m, n, layout)) return 1;
  const int64_t nt = m > 16 ? 4 : i4_few_tiles(layout, n);
  const int64_t blocks = (n + 16 * nt - 1) / (16 * nt) * ((m + 63) / 64);
  const int64_t upw = ((k + 127) / 128 + 7) / 8;  // units per wave of a workgroup
  if (m <= 16 && upw <= (layout == LA ? 6 : 8)) return 1;
  const int64_t most = m > 16 ? upw : upw / 2, fit = 256 / blocks;
  const int64_t s = most < fit ? most : fit;
  return s < 2 ? 1 : (int)(s > 8 ? 8 : s);
}

template <int DT, int LAYOUT, int F, int MT, int NT, int SETS, int W>
int i4_go(const I4Args& a, int slots, int nsets, hipStream_t st) {
  constexpr int lds = I4Few<DT, LAYOUT, F, MT, NT, SETS, W>::LDS;
  const dim3 grid((unsigned)((a.n + 16 * NT - 1) / (16 * NT)), (unsigned)slots,
                  (unsigned)(a.row_off ? (SETS == 1 ? nsets : 1) : a.nsplit));
  if constexpr (lds > 65536)
    (void)hipFuncSetAttribute((const void*)k_int4_few<DT, LAYOUT, F, MT, NT, SETS, W>,
                              hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  hipLaunchKernelGGL((k_int4_few<DT, LAYOUT, F, MT, NT, SETS, W>), grid, 64 * W, lds, st, a);
  if (int rc = check_launch("lcq_int4_gemm")) return rc;
  if (a.nsplit > 1) {
    hipLaunchKernelGGL(k_int4_join<DT>, dim3((unsigned)((a.m * a.n + 1023) / 1024)), 256, 0, st, a);
    return check_launch("lcq_int4_gemm");
  }
  return LCQ_OK;
}

template <int DT, int LAYOUT, int F, int SETS>
int i4_launch(const I4Args& a, int nsets, hipStream_t st) {
  if (i4_use_tile(a, LAYOUT, SETS)) {
    constexpr int lds = i4_tile_lds<LAYOUT>;
    constexpr int cols = SETS == 2 ? 128 : 256;
    const int64_t slots = a.row_off ? a.m / TM + (a.G < a.m ? a.G : a.m) : (a.m + TM - 1) / TM;
    const int64_t wgs = (a.n + cols - 1) / cols * slots;
    if (wgs >= (int64_t(1) << 31)) return fail(LCQ_EINVAL, "lcq_int4_gemm: too many rows");
    (void)hipFuncSetAttribute((const void*)k_int4_tile<DT, LAYOUT, F, SETS>,
                              hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    hipLaunchKernelGGL((k_int4_tile<DT, LAYOUT, F, SETS>),
                       dim3((unsigned)wgs, 1, (unsigned)(SETS == 1 ? nsets : 1)), 512, lds, st, a);
    return check_launch("lcq_int4_gemm");
  }
  // As many row tiles as the rows need. Groups: half as many again as their mean, or most of the
  // fuller ones would read their weights twice (16 experts of 16 rows, 2048 x 4096: 28 us, 61 with
  // tiles of 16), and 4 waves instead of 8 (experts of 30 rows, AutoAWQ gate and up: 82 us, 109)
  const int64_t per = a.row_off ? (a.m + a.G - 1) / a.G : a.m;
  constexpr int MB = SETS == 2 ? 2 : 4;
  const int64_t most = a.row_off ? per + per / 2 : per, tiles = (most + 15) / 16;
  const int mt = per <= (a.row_off ? 12 : 16) ? 1 : (int)(tiles < MB ? tiles : MB);
  const int bm = 16 * mt;
  const int64_t slots = a.row_off ? a.m / bm + (a.G < a.m ? a.G : a.m) : (a.m + bm - 1) / bm;
  if (slots > 65535) return fail(LCQ_EINVAL, "lcq_int4_gemm: too many rows");
  if (mt > 1) {
    constexpr int NT = LAYOUT == LA || SETS == 1 ? 4 : 2;
    auto go = [&](auto w) {
      constexpr int W = decltype(w)::value;
      if constexpr (MB == 4) {
        if (mt == 4) return i4_go<DT, LAYOUT, F, 4, NT, SETS, W>(a, (int)slots, nsets, st);
        if (mt == 3) return i4_go<DT, LAYOUT, F, 3, NT, SETS, W>(a, (int)slots, nsets, st);
      }
      return i4_go<DT, LAYOUT, F, 2, NT, SETS, W>(a, (int)slots, nsets, st);
    };
    if constexpr (SETS == 1)
      if (!a.row_off) return go(std::integral_constant<int, 8>{});
    return go(std::integral_constant<int, 4>{});
  }
  if constexpr (LAYOUT == LA || SETS == 2) {
    return i4_go<DT, LAYOUT, F, 1, LAYOUT == LA ? 4 : 2, SETS, 8>(a, (int)slots, nsets, st);
  } else {
    switch (i4_few_tiles(LAYOUT, a.row_off ? a.n * (a.G < a.m ? a.G : a.m) : a.n)) {
      case 1: return i4_go<DT, LAYOUT, F, 1, 1, SETS, 8>(a, (int)slots, nsets, st);
      case 2: return i4_go<DT, LAYOUT, F, 1, 2, SETS, 8>(a, (int)slots, nsets, st);
      default: return i4_go<DT, LAYOUT, F, 1, 4, SETS, 8>(a, (int)slots, nsets, st);
    }
  }
}

template <int DT, int LAYOUT>
int i4_dispatch(const I4Args& a, int nsets, bool silu, hipStream_t st) {
  const int f = a.group % 128 == 0 ? 1 : a.group % 64 == 0 ? 2 : 4;
  if (silu)
    return f == 1   ? i4_launch<DT, LAYOUT, 1, 2>(a, nsets, st)
           : f == 2 ? i4_launch<DT, LAYOUT, 2, 2>(a, nsets, st)
                    : i4_launch<DT, LAYOUT, 4, 2>(a, nsets, st);
  return f == 1   ? i4_launch<DT, LAYOUT, 1, 1>(a, nsets, st)
         : f == 2 ? i4_launch<DT, LAYOUT, 2, 1>(a, nsets, st)
                  : i4_launch<DT, LAYOUT, 4, 1>(a, nsets, st);
}

int i4_dispatch(const I4Args& a, int dtype, int layout, int nsets, bool silu, hipStream_t st) {
  if (dtype == LCQ_BF16)
    return layout == LV ? i4_dispatch<LCQ_BF16, LV>(a, nsets, silu, st)
                        : i4_dispatch<LCQ_BF16, LA>(a, nsets, silu, st);
  return layout == LV ? i4_dispatch<LCQ_F16, LV>(a, nsets, silu, st)
                      : i4_dispatch<LCQ_F16, LA>(a, nsets, silu, st);
}

int i4_check(const char* who, int dtype, int64_t m, int64_t n, int64_t k, int layout,
             int64_t group) {
  auto bad = [&](const char* msg) { return fail(LCQ_EINVAL, std::string(who) + ": " + msg); };
  if (dtype != LCQ_BF16 && dtype != LCQ_F16) return bad("bf16 / fp16 activations only");
  if (layout != LV && layout != LA) return bad("layout must be 0 (vllm) or 1 (autoawq)");
  if (m < 0 || n <= 0 || k <= 0) return bad("bad shape");
  if (k % 32) return bad("k must be a multiple of 32");
  if (group <= 0 || group % 32 || k % group) return bad("group must be a multiple of 32 and divide k");
  if (layout == LA && n % 8) return bad("autoawq layout: n must be a multiple of 8");
  if (n >= (int64_t(1) << 31) || k >= (1 << 21) || m >= (int64_t(1) << 31) ||
      n * k >= (int64_t(1) << 32))
    return bad("shape too large");
  return LCQ_OK;
}

uint32_t group_mul(int64_t group) {  // 0: group 32
  return group == 32 ? 0 : (uint32_t)((int64_t(1) << 32) / (group / 32) + 1);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace lcq

using namespace lcq;

extern "C" int64_t lcq_int4_gemm_workspace_bytes(int64_t m, int64_t n, int64_t k, int layout) {
  constexpr int64_t big = int64_t(1) << 31;
  if (m <= 0 || n <= 0 || k <= 0 || m >= big || n >= big || k >= big) return 0;
  const int s = i4_nsplit(m, n, k, layout);
  return s > 1 ? 4 * s * m * n : 0;
}

extern "C" int lcq_int4_gemm(const void* x, int dtype, int64_t ldx, int64_t m, int64_t k,
                             const void* qweight, const void* scales, const void* qzeros,
                             int layout, int64_t group, int64_t n, const void* bias, void* y,
                             int64_t ldy, void* workspace, int64_t ws_bytes, void* stream) {
  if (int rc = i4_check("lcq_int4_gemm", dtype, m, n, k, layout, group)) return rc;
  if (m == 0) return LCQ_OK;
  LCQ_REQUIRE(x && qweight && scales && y, "null pointer");
  LCQ_REQUIRE((layout == 1) == (qzeros != nullptr), "qzeros belong to the autoawq layout");
  LCQ_REQUIRE(ldx >= k && ldx % 8 == 0 && ldy >= n, "bad row stride");
  LCQ_REQUIRE(aligned16(x) && aligned16(qweight) && aligned16(scales),
              "x, qweight and scales must be 16-byte aligned");
  I4Args a{};
  a.x = static_cast<const uint16_t*>(x);
  a.ldx = ldx; a.m = m; a.n = n; a.k = k; a.group = group;
  a.qw = static_cast<const uint32_t*>(qweight);
  a.sc = static_cast<const uint16_t*>(scales);
  a.qz = static_cast<const uint32_t*>(qzeros);
  a.bias = static_cast<const uint16_t*>(bias);
  a.gmul = group_mul(group);
  a.y = static_cast<uint16_t*>(y);
  a.ldy = ldy;
  a.wide_y = aligned16(y) && ldy % 8 == 0;
  a.nsplit = i4_nsplit(m, n, k, layout);
  a.part = static_cast<float*>(workspace);
  LCQ_REQUIRE(a.nsplit == 1 || (workspace && ws_bytes >= 4 * a.nsplit * m * n),
              "workspace too small (lcq_int4_gemm_workspace_bytes)");
  return i4_dispatch(a, dtype, layout, 1, false, as_stream(stream));
}

extern "C" int lcq_int4_gemm_grouped(const void* x, int dtype, int64_t ldx, int64_t x_rows,
                                     const int64_t* a_rows, int64_t rows, const int64_t* row_off,
                                     const int64_t* wtab, int64_t G, int nsets, int silu_mul,
                                     int layout, int64_t group, int64_t n, int64_t k, void* y,
                                     void* stream) {
  if (int rc = i4_check("lcq_int4_gemm_grouped", dtype, rows, n, k, layout, group)) return rc;
  LCQ_REQUIRE(G > 0 && G < (1 << 20), "bad group count");
  LCQ_REQUIRE(nsets == 1 || nsets == 2, "one or two weight sets");
  LCQ_REQUIRE(!silu_mul || nsets == 2, "silu_mul takes the gate and up sets");
  if (rows == 0) return LCQ_OK;
  LCQ_REQUIRE(x && row_off && wtab && y, "null pointer");
  LCQ_REQUIRE(ldx >= k && ldx % 8 == 0 && aligned16(x), "x rows must be 16-byte aligned");
  LCQ_REQUIRE(x_rows > 0 && (a_rows || x_rows >= rows), "x has fewer rows than the groups");
  I4Args a{};
  a.x = static_cast<const uint16_t*>(x);
  a.ldx = ldx; a.m = rows; a.n = n; a.k = k; a.group = group;
  a.y = static_cast<uint16_t*>(y);
  a.ldy = n;
  a.gmul = group_mul(group);
  a.wide_y = aligned16(y) && n % 8 == 0;
  a.nsplit = 1;
  a.row_off = row_off;
  a.a_rows = a_rows;
  a.wtab = wtab;
  a.x_rows = x_rows;
  a.G = (int)G;
  return i4_dispatch(a, dtype, layout, nsets, silu_mul != 0, as_stream(stream));
}
