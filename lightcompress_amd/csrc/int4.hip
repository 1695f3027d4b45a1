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
};

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
      grp = g0 + l;
      r0 = glo + (int64_t)(slot - first) * bm;
      r1 = min(r0 + bm, ghi);
      return true;
    }
    base += total;
  }
  return false;
}

// Decode kernel: 16 rows of x per workgroup, NT column tiles of 16 per set, the K blocks of 128
// split over the workgroup's waves, their partial tiles summed through LDS in wave order.
// NAT: x and the words are taken in natural k order, 32 k per MFMA, so that a scale group may end
// after any multiple of 32; else (group a multiple of 128) a lane's 16-byte load of a row is used
// as it comes: word j of the 4 lanes of a row holds k = 32 q + 8 j, one permutation of the
// block's k that x follows.
template <int DT, int LAYOUT, bool NAT, int NT, int SETS, int W>
__global__ __launch_bounds__(64 * W) void k_int4_dec(I4Args a) {
  constexpr int T = NT * SETS;
  __shared__ float red[W][T * 4][64];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = lane & 15, q = lane >> 4;
  int64_t r0, r1;
  int grp = 0;
  if (a.row_off) {
    if (!i4_find(a, blockIdx.y, 16, r0, r1, grp)) return;
  } else {
    r0 = (int64_t)blockIdx.y * 16;
    r1 = min(r0 + 16, a.m);
  }
  const uint32_t* qw[SETS];
  const uint16_t* sc[SETS];
  const uint32_t* qz[SETS];
#pragma unroll
  for (int s = 0; s < SETS; ++s) {
    if (a.row_off) {
      const int64_t* t = a.wtab + ((int64_t)(SETS == 1 ? blockIdx.z : s) * a.G + grp) * 3;
      qw[s] = reinterpret_cast<const uint32_t*>(t[0]);
      sc[s] = reinterpret_cast<const uint16_t*>(t[1]);
      qz[s] = reinterpret_cast<const uint32_t*>(t[2]);
    } else {
      qw[s] = a.qw;
      sc[s] = a.sc;
      qz[s] = a.qz;
    }
  }
  // this lane's row of x (as the A operand: row lane & 15)
  const uint16_t* xr = nullptr;
  if (r0 + c < r1) {
    int64_t row = r0 + c;
    if (a.a_rows) row = a.a_rows[row];
    if (!a.a_rows || (row >= 0 && row < a.x_rows)) xr = a.x + row * a.ldx;
  }
  const int64_t n0 = (int64_t)blockIdx.x * 16 * NT;
  const int64_t ng = a.k / a.group;
  // column of tile t for this lane (clamped for the loads; the stores check)
  int64_t col[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t cc = LAYOUT == LV ? n0 + 16 * t + c : n0 + 8 * c + t;
    col[t] = min(cc, a.n - 1);
  }
  const int64_t wc = min(n0 / 8 + c, a.n / 8 - 1);  // AutoAWQ word column

  i4_v4f acc[T], g[T], xs = {0.f, 0.f, 0.f, 0.f};
  const i4_v4f zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int t = 0; t < T; ++t) acc[t] = g[t] = zero;
  const i4_v4u ones = {i4_ones<DT>, i4_ones<DT>, i4_ones<DT>, i4_ones<DT>};

  const int nb = (int)((a.k + 127) / 128);
  const int b0 = (int)((int64_t)nb * w / W), b1 = (int)((int64_t)nb * (w + 1) / W);
  // acc += s (g - (16 + z) xs) for the group that ends here; g, xs = 0
  auto flush = [&](int64_t gi) {
#pragma unroll
    for (int s = 0; s < SETS; ++s) {
      uint32_t zw = 0;
      if constexpr (LAYOUT == LA) zw = qz[s][gi * (a.n / 8) + wc];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float sv, zv;
        if constexpr (LAYOUT == LV) {
          sv = h2f(sc[s][col[t] * ng + gi]);
          zv = 24.f;
        } else {
          sv = h2f(sc[s][gi * a.n + col[t]]);
          constexpr int inv[8] = {0, 4, 1, 5, 2, 6, 3, 7};
          zv = 16.f + (float)((zw >> (4 * inv[t & 7])) & 15u);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
          acc[s * NT + t][r] = __fmaf_rn(sv, __fmaf_rn(-zv, xs[r], g[s * NT + t][r]),
                                         acc[s * NT + t][r]);
        g[s * NT + t] = zero;
      }
    }
    xs = zero;
  };
  for (int b = b0; b < b1; ++b) {
    const int64_t k0 = (int64_t)b * 128;
    i4_v4u xf[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t kk = (LAYOUT == LA || NAT) ? k0 + 32 * j + 8 * q : k0 + 32 * q + 8 * j;
      xf[j] = i4_v4u{0, 0, 0, 0};
      if (xr && kk < a.k) xf[j] = *reinterpret_cast<const i4_v4u*>(xr + kk);
      if constexpr (LAYOUT == LV) xf[j] = i4_xorder(xf[j]);
    }
    i4_v4u wv[LAYOUT == LV ? T : 1];
    if constexpr (LAYOUT == LV) {
      // 16 bytes of row col[t]: the words of k0 + 32 q .. + 31 (rows end on a multiple of 32 k)
      const int64_t kw = min(k0 + 32 * q, a.k - 32) / 8;
#pragma unroll
      for (int s = 0; s < SETS; ++s)
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          i4_v4u v = *reinterpret_cast<const i4_v4u*>(qw[s] + col[t] * (a.k / 8) + kw);
          if constexpr (NAT) {
            // 4 x 4 transpose of words between the lanes q = 0..3 of a row: word j then holds
            // k = 32 j + 8 q
            auto p = __builtin_amdgcn_permlane32_swap(v.x, v.z, false, false);
            v.x = p[0]; v.z = p[1];
            p = __builtin_amdgcn_permlane32_swap(v.y, v.w, false, false);
            v.y = p[0]; v.w = p[1];
            p = __builtin_amdgcn_permlane16_swap(v.x, v.y, false, false);
            v.x = p[0]; v.y = p[1];
            p = __builtin_amdgcn_permlane16_swap(v.z, v.w, false, false);
            v.z = p[0]; v.w = p[1];
          }
          wv[s * NT + t] = v;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t ks = k0 + 32 * j;
      if ((LAYOUT == LA || NAT) && ks >= a.k) break;
      xs = i4_mfma<DT>(xf[j], ones, xs);
      if constexpr (LAYOUT == LV) {
#pragma unroll
        for (int t = 0; t < T; ++t) g[t] = i4_mfma<DT>(xf[j], i4_word<DT>(wv[t][j]), g[t]);
      } else {
#pragma unroll
        for (int s = 0; s < SETS; ++s) {
          uint32_t u[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) u[i] = qw[s][(ks + 8 * q + i) * (a.n / 8) + wc];
          uint32_t lo[4], hi[4];  // nibbles 0..3 / 4..7 of word 2 p and 2 p + 1
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            lo[p] = __builtin_amdgcn_perm(u[2 * p + 1], u[2 * p], 0x05040100u);
            hi[p] = __builtin_amdgcn_perm(u[2 * p + 1], u[2 * p], 0x07060302u);
          }
          // column 2 i is nibble i, column 2 i + 1 nibble i + 4
          auto tile = [&](int t, i4_v4u f) {
            g[s * NT + t] = i4_mfma<DT>(xf[j], f, g[s * NT + t]);
          };
#define LCQ_I4_COL(i)                                                                       \
  tile(2 * i, i4_v4u{i4_pair<DT, i>(lo[0]), i4_pair<DT, i>(lo[1]), i4_pair<DT, i>(lo[2]),  \
                     i4_pair<DT, i>(lo[3])});                                               \
  tile(2 * i + 1, i4_v4u{i4_pair<DT, i>(hi[0]), i4_pair<DT, i>(hi[1]),                      \
                         i4_pair<DT, i>(hi[2]), i4_pair<DT, i>(hi[3])});
          LCQ_I4_COL(0) LCQ_I4_COL(1) LCQ_I4_COL(2) LCQ_I4_COL(3)
#undef LCQ_I4_COL
        }
      }
      if constexpr (LAYOUT == LA || NAT)
        if ((ks + 32) % a.group == 0) flush(ks / a.group);
    }
    if constexpr (!(LAYOUT == LA || NAT))
      if ((k0 + 128) % a.group == 0) flush(k0 / a.group);
  }
  // a group cut by the wave's range: its part is linear in s
  if (b1 > b0) {
    const int64_t kend = min((int64_t)b1 * 128, a.k);
    if (kend % a.group != 0) flush((kend - 1) / a.group);
  }
#pragma unroll
  for (int t = 0; t < T; ++t)
#pragma unroll
    for (int r = 0; r < 4; ++r) red[w][4 * t + r][lane] = acc[t][r];
  __syncthreads();
  // outputs (tile t, lane, r): row r0 + 4 q + r; the waves share the NT tiles
  for (int t = w; t < NT; t += W) {
    const int64_t cc = LAYOUT == LV ? n0 + 16 * t + c : n0 + 8 * c + t;
    if (cc >= a.n) continue;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t row = r0 + 4 * q + r;
      float v[SETS];
#pragma unroll
      for (int s = 0; s < SETS; ++s) {
        v[s] = 0.f;
        for (int i = 0; i < W; ++i) v[s] += red[i][4 * (s * NT + t) + r][lane];
      }
      float o = v[0];
      if constexpr (SETS == 2) o = v[0] / (1.f + expf(-v[0])) * v[1];
      if (a.bias) o += ld1<DT>(a.bias, cc);
      if (row < r1) st1<DT>(a.y + (SETS == 1 ? blockIdx.z * a.m * a.ldy : 0), row * a.ldy + cc, o);
    }
  }
}

template <int DT, int LAYOUT, bool NAT, int SETS>
int i4_launch_dec(const I4Args& a, int slots, int nsets, hipStream_t st) {
  constexpr int NT = LAYOUT == LV ? 2 : 8;
  constexpr int W = LAYOUT == LA && SETS == 2 ? 4 : 8;
  const dim3 grid((unsigned)((a.n + 16 * NT - 1) / (16 * NT)), (unsigned)slots,
                  (unsigned)(SETS == 1 ? nsets : 1));
  hipLaunchKernelGGL((k_int4_dec<DT, LAYOUT, NAT, NT, SETS, W>), grid, 64 * W, 0, st, a);
  return check_launch("lcq_int4_gemm");
}

template <int DT>
int i4_dispatch(const I4Args& a, int layout, int slots, int nsets, bool silu, hipStream_t st) {
  if (layout == LV) {
    const bool nat = a.group % 128 != 0;
    if (silu) return nat ? i4_launch_dec<DT, LV, true, 2>(a, slots, nsets, st)
                         : i4_launch_dec<DT, LV, false, 2>(a, slots, nsets, st);
    return nat ? i4_launch_dec<DT, LV, true, 1>(a, slots, nsets, st)
               : i4_launch_dec<DT, LV, false, 1>(a, slots, nsets, st);
  }
  return silu ? i4_launch_dec<DT, LA, true, 2>(a, slots, nsets, st)
              : i4_launch_dec<DT, LA, true, 1>(a, slots, nsets, st);
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
  if (n >= (int64_t(1) << 31) || k >= (int64_t(1) << 31) || m >= (int64_t(1) << 31))
    return bad("shape too large");
  return LCQ_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace lcq

using namespace lcq;

extern "C" int lcq_int4_gemm(const void* x, int dtype, int64_t ldx, int64_t m, int64_t k,
                             const void* qweight, const void* scales, const void* qzeros,
                             int layout, int64_t group, int64_t n, const void* bias, void* y,
                             int64_t ldy, void* stream) {
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
  a.y = static_cast<uint16_t*>(y);
  a.ldy = ldy;
  LCQ_REQUIRE((m + 15) / 16 <= 65535, "too many rows");
  const int slots = (int)((m + 15) / 16);
  return dtype == LCQ_BF16 ? i4_dispatch<LCQ_BF16>(a, layout, slots, 1, false, as_stream(stream))
                           : i4_dispatch<LCQ_F16>(a, layout, slots, 1, false, as_stream(stream));
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
  LCQ_REQUIRE(a_rows || x_rows >= rows, "x has fewer rows than the groups");
  I4Args a{};
  a.x = static_cast<const uint16_t*>(x);
  a.ldx = ldx; a.m = rows; a.n = n; a.k = k; a.group = group;
  a.y = static_cast<uint16_t*>(y);
  a.ldy = n;
  a.row_off = row_off;
  a.a_rows = a_rows;
  a.wtab = wtab;
  a.x_rows = x_rows;
  a.G = (int)G;
  const int64_t slots = rows / 16 + (G < rows ? G : rows);
  LCQ_REQUIRE(slots <= 65535, "too many rows");
  return dtype == LCQ_BF16
             ? i4_dispatch<LCQ_BF16>(a, layout, (int)slots, nsets, silu_mul != 0, as_stream(stream))
             : i4_dispatch<LCQ_F16>(a, layout, (int)slots, nsets, silu_mul != 0, as_stream(stream));
}
