// Latent attention (keys and values of every head from one shared latent vector per token) on
// bf16 / fp16 MFMA, gfx950. Two forms of the same attention:
//
// Expanded (prompts, chunks, calibration): per head a key of 128 "nope" dims from the latent's
// up-projection and 64 rotary dims shared by all heads, a value of 128 dims:
//   out_i = sum_j softmax_j( (qn_i . kn_j + qr_i . kr_j) scale ) v_j,   j <= q_start + i, j < len.
// The kernel reads the up-projection's output and the shared rotary key as they are: neither the
// concatenated keys nor a copy of the rotary key per head is ever written.
//
// Absorbed (decode): with the up-projections folded into the query and the output, a head's key
// and value are the latent itself: scores q_latent . c_j + q_rope . kr_j, output sum_j p_j c_j
// (512 dims). All heads read the one cache row of 576 values, so a token's attention is a
// matrix product of (tokens x heads) rows with the cache.
//
// Both are flash kernels: fp32 scores and sums, online softmax in the exp2 domain, P rounded to
// the input type for the P V product (fp32 accumulation; its rounding is relative 2^-9 / 2^-12 per
// weight, averaged over the row), the output rounded once.
#include <type_traits>

#include "attn_common.h"

namespace lcq {
namespace {

constexpr int DN = 128, DR = 64, DV = 128, DL = 512;  // nope, rope, value, latent dims

// XOR of the 16 low chunks of a row in the 256- and 1024-byte-row images (the rotary image, two
// rows to the 256 bytes of the 64 banks, takes (row >> 1) & 7): conflict-free for the row reads and
// the transposed reads
__device__ __forceinline__ int swz16(int row) { return ((row & 3) << 2) | ((row >> 2) & 3); }

// a wave-uniform pointer kept in scalar registers
__device__ __forceinline__ const uint16_t* uni(const uint16_t* p) {
  const uint64_t u = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)u);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(u >> 32));
  return reinterpret_cast<const uint16_t*>(((uint64_t)hi << 32) | lo);
}

__device__ __forceinline__ int64_t uni(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)((uint64_t)v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// ---------------------------------------------------------------------------------------
// Expanded form
// ---------------------------------------------------------------------------------------
constexpr int FQT = 128;  // query rows per workgroup (4 waves of 32)
constexpr int FKT = 64;   // keys per tile
constexpr int F_STAGE = FKT * (DN + DR + DV) * 2;  // 40 KB
constexpr int F_AHEAD = 4;                         // LDS fragments read ahead of their product
constexpr int F_MIN = 8;                           // least tiles of a share of the keys
constexpr int F_PART = FQT * DV;                   // floats of a query tile's partial output

struct MlaFwdArgs {
  const uint16_t *qn, *qr, *kn, *kr, *v;
  uint16_t* out;            // [B, Sq, H, 128]
  int64_t qnb, qnh, qns, qrb, qrh, qrs, knb, knh, kns, krb, krs, vb, vh, vs;  // elements
  const int32_t* q_start;   // nullable [B]: position of query 0 (default Skv - Sq)
  const int32_t* kv_lens;   // nullable [B]: valid keys (default Skv)
  int Sq, Skv, H, nqt, ns;  // ns shares of the keys per query tile
  float* part;              // ns > 1: [query tiles][ns] partial outputs, then their max / sum
  float2* ml;
  float sl2;                // scale * log2(e)
};

// The three images of one 64-key tile by LDS-DMA, 10 instructions per wave. The base moves with the
// tile (64-bit), so only a tile's own span has to fit 32 bits; a lane's offsets are formed once
// (`lim` 63) and again for a last tile, whose keys past `lim` re-read it: what lies behind a
// sequence is never loaded.
struct FwdStage {
  uint32_t kn[4], v[4], kr[2];
  __device__ __forceinline__ void init_keys(const MlaFwdArgs& a, int lim, int w, int lane) {
#pragma unroll
    for (int j = 0; j < 4; ++j) kn[j] = at(4 * (4 * w + j) + (lane >> 4), lim, a.kns, lane);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int row = 8 * (2 * w + j) + (lane >> 3);
      kr[j] = (uint32_t)min(row, lim) * (uint32_t)a.krs * 2 + 16 * ((lane & 7) ^ ((row >> 1) & 7));
    }
  }
  __device__ __forceinline__ void init_values(const MlaFwdArgs& a, int lim, int w, int lane) {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = at(4 * (4 * w + j) + (lane >> 4), lim, a.vs, lane);
  }
  static __device__ __forceinline__ uint32_t at(int row, int lim, int64_t stride, int lane) {
    return (uint32_t)min(row, lim) * (uint32_t)stride * 2 + 16 * ((lane & 15) ^ swz16(row));
  }
  __device__ __forceinline__ void keys(uint32_t st, const uint16_t* pn, const uint16_t* pr,
                                       int w) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) dma16(st + 1024 * (4 * w + j), pn, kn[j]);
#pragma unroll
    for (int j = 0; j < 2; ++j) dma16(st + 32768 + 1024 * (2 * w + j), pr, kr[j]);
  }
  __device__ __forceinline__ void values(uint32_t st, const uint16_t* pv, int w) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) dma16(st + 16384 + 1024 * (4 * w + j), pv, v[j]);
  }
};

// Four waves of 32 query rows share 64-key tiles: scores transposed (a lane holds 32 keys of one
// row), so that the weights turn into the second product's operand in place. Keys and values stand
// in two buffers each (80 KB, two workgroups per CU). What bounds it: no unit alone (of the time its
// CU is busy MFMA works 41 %, LDS 22 %) but the chain of phases in a wave, two waves to a SIMD, which
// stand at a wait 37 % of their cycles: 2048 tokens of 128 heads in 226-237 us, 725-760 TF/s; four
// padded sequences of 301, 16 heads, 12-13 us, waiting 53 %.
// SPLIT: the workgroup takes its share of the query tile's key tiles and leaves the unnormalised
// output (lane order) with the rows' max and sum for k_mla_fwd_join
template <int DT, bool SPLIT>
__global__ void __launch_bounds__(256, 2) k_mla_fwd(MlaFwdArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char mla_lds[];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 31, h = lane >> 5;
  const uint32_t lds0 = lds_addr(mla_lds);
  // the query tiles of one (batch, head) run together on one XCD and share its keys in L2
  int L;
  {
    const int nwg = (int)gridDim.x, p = (int)blockIdx.x;
    const int xcd = p & 7, q8 = nwg >> 3, r8 = nwg & 7;
    L = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (p >> 3);
  }
  const int qt = a.nqt - 1 - L % a.nqt;  // longest tiles first
  const int sp = SPLIT ? (L / a.nqt) % a.ns : 0;
  if (SPLIT) L /= a.ns * a.nqt;
  else L /= a.nqt;
  const int hq = L % a.H, b = L / a.H;
  const int q0 = qt * FQT;
  const int klen = a.kv_lens ? min(max(a.kv_lens[b], 0), a.Skv) : a.Skv;
  const int qs = a.q_start ? min(max(a.q_start[b], -(1 << 29)), 1 << 29) : a.Skv - a.Sq;
  int kbeg = 0, kend = min(klen, qs + min(q0 + FQT, a.Sq));
  const int64_t pt = SPLIT ? ((int64_t)(b * a.H + hq) * a.nqt + qt) * a.ns + sp : 0;
  if constexpr (SPLIT) {
    const int n = kend > 0 ? (kend + FKT - 1) / FKT : 0, each = (n + a.ns - 1) / a.ns;
    kbeg = min(sp * each * FKT, max(kend, 0));
    kend = min(kbeg + each * FKT, kend);
    if (kbeg >= kend) {  // nothing to add: the join skips rows of sum 0
      if (tid < FQT) a.ml[pt * FQT + tid] = make_float2(-INFINITY, 0.f);
      return;
    }
  }
  if (kend <= 0) {  // no row of the tile sees a key
    for (int i = tid; i < FQT * 16; i += 256) {
      const int qr = q0 + (i >> 4);
      if (qr < a.Sq)
        *reinterpret_cast<uint4*>(a.out + (((int64_t)b * a.Sq + qr) * a.H + hq) * DV +
                                  (i & 15) * 8) = make_uint4(0, 0, 0, 0);
    }
    return;
  }
  const uint16_t* qnp = a.qn + b * a.qnb + hq * a.qnh;
  const uint16_t* qrp = a.qr + b * a.qrb + hq * a.qrh;
  const uint16_t* knp = uni(a.kn + b * a.knb + hq * a.knh);
  const uint16_t* krp = uni(a.kr + b * a.krb);
  const uint16_t* vp = uni(a.v + b * a.vb + hq * a.vh);
  FwdStage fs;
  const int lim0 = min(FKT - 1, klen - 1 - kbeg);
  fs.init_keys(a, lim0, w, lane);
  fs.init_values(a, lim0, w, lane);
  const int ntile = (kend - kbeg + FKT - 1) / FKT;
  // called for tile after tile; keys and values have two buffers each
  auto stage_keys = [&](int t) {
    const int k0 = kbeg + t * FKT;
    if (t > 0 && klen - 1 - k0 < FKT - 1) fs.init_keys(a, klen - 1 - k0, w, lane);
    fs.keys(lds0 + (t & 1) * F_STAGE, uni(knp + k0 * a.kns), uni(krp + k0 * a.krs), w);
  };
  auto stage_values = [&](int t) {
    const int k0 = kbeg + t * FKT;
    if (t > 0 && klen - 1 - k0 < FKT - 1) fs.init_values(a, klen - 1 - k0, w, lane);
    fs.values(lds0 + (t & 1) * F_STAGE, uni(vp + k0 * a.vs), w);
  };
  stage_keys(0);

  const int qrow = q0 + 32 * w + c;  // this lane's query row (both halves)
  // Q^T as the B operand of mfma(K, Q^T): lane holds Q[qrow][16 kk + 8 h + j]
  v8s_t qf[12];
#pragma unroll
  for (int kk = 0; kk < 12; ++kk) {
    qf[kk] = (v8s_t){0, 0, 0, 0, 0, 0, 0, 0};
    if (qrow < a.Sq)
      qf[kk] = *reinterpret_cast<const v8s_t*>(
          kk < 8 ? qnp + qrow * a.qns + 16 * kk + 8 * h
                 : qrp + qrow * a.qrs + 16 * (kk - 8) + 8 * h);
  }
  const int pos = min(qs + qrow, klen - 1);       // last key this lane's row sees
  // the least and the greatest of the wave's rows (a wave without rows: none)
  const int wmin = min(qs + q0 + 32 * w, klen - 1);
  const int wmax = q0 + 32 * w < a.Sq ? min(qs + q0 + 32 * w + 31, klen - 1) : -1;
  float m = -INFINITY, l = 0.f;
  v16f_t o[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[dt][r] = 0.f;
  const int g = lane >> 4, i16 = lane & 15, qq = i16 >> 2, pp = i16 & 3;
  // LDS offsets in a stage; a constant XOR walks the swizzled chunks of a row
  const uint32_t ka = 256 * c + 16 * (h ^ swz16(c));              // K chunk 2 kk + h: ^ 32 kk
  const uint32_t ra = 32768 + 128 * c + 16 * (h ^ ((c >> 1) & 7));  // rope chunk: ^ 32 kk
  const uint32_t va = 16384 + 256 * (4 * (g >> 1) + qq) +
                      16 * ((2 * (g & 1) + (pp >> 1)) ^ (qq << 2 | (g >> 1))) + 8 * (pp & 1);

  // one product of S^T = K Q^T (two tiles of 32 keys in turn, so that a product does not wait for
  // the one before it): product f is k-step f / 2 of tile f & 1. Register r of tile t holds key
  // 32 t + (r & 3) + 8 (r >> 2) + 4 h of the lane's row
  auto kfrag = [&](uint32_t st, int f) {
    const int kk = f >> 1, t = f & 1;
    return kk < 8 ? lds_read16(((st + ka) ^ (32 * kk)) + 8192 * t)
                  : lds_read16(((st + ra) ^ (32 * (kk - 8))) + 4096 * t);
  };
  v16f_t s[2];
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  if (ntile > 1) stage_keys(1);
  stage_values(0);
#pragma unroll
  for (int r = 0; r < 16; ++r) s[0][r] = s[1][r] = 0.f;
  if (kbeg <= wmax) {
#pragma unroll
    for (int f = 0; f < 24; ++f) s[f & 1] = mfma32<DT>(kfrag(lds0, f), qf[f >> 1], s[f & 1]);
  }

  // Iteration t: the softmax of tile t's scores stands between the products of tile t + 1's (the
  // matrix pipe and the vector pipe work at once), then O^T += V^T P^T. K fragments are read
  // F_AHEAD products ahead (the scheduling barriers keep the compiler to that order: left alone
  // it waits for each read right before its product). The copies of the tiles after stand behind
  // the softmax only: the compiler does not see the waits below, holds the queries' loads for
  // outstanding, and puts a vmcnt(0) of its own before an iteration's first product.
  for (int it = 0; it < ntile; ++it) {
    const int k0 = kbeg + it * FKT;
    const uint32_t cur = lds0 + (it & 1) * F_STAGE, nxt = lds0 + ((it & 1) ^ 1) * F_STAGE;
    // this wave's part of K(t + 1) and V(t) has arrived; behind the barrier every wave's has, and
    // every wave is done with K(t) and V(t - 1), whose buffers are filled next
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    if (it + 2 < ntile) stage_keys(it + 2);
    if (it + 1 < ntile) stage_values(it + 1);
    if (k0 > wmax) continue;  // no row of this wave sees the tile, nor a later one

    if (k0 + FKT - 1 > wmin) {  // wave-uniform: some key is hidden from some row
      const int lim = pos - k0 - 4 * h;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (32 * t + (r & 3) + 8 * (r >> 2) > lim) s[t][r] = -INFINITY;
    }
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[t][r]);
    mx = fmaxf(mx, other_half(mx, h)) * a.sl2;  // sl2 > 0: max commutes with the scale
    // the output is rescaled only when a row's maximum has grown by more than 2^8 since it last
    // was: weights stay below 2^8, in range of fp16
    if (__any(mx > m + 8.f)) {
      const float mn = mx > m + 8.f ? mx : m;
      const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      l *= alpha;
      m = mn;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
    }
    const float msub = m == -INFINITY ? 0.f : m;
    float rs = 0.f;
    v8s_t pf[4];  // k-step ts = (t, s2) of P^T: score registers 8 s2 .. 8 s2 + 7 of tile t
    auto soft = [&](int e, float msub) {  // weights 2 e, 2 e + 1 of 32
      const int t = e >> 3, r = 2 * (e & 7);
      const float p0 = __builtin_amdgcn_exp2f(__fmaf_rn(s[t][r], a.sl2, -msub));
      const float p1 = __builtin_amdgcn_exp2f(__fmaf_rn(s[t][r + 1], a.sl2, -msub));
      rs += p0;
      rs += p1;
      reinterpret_cast<uint32_t*>(&pf[2 * t + (r >> 3)])[(r & 7) >> 1] = pack_dt<DT>(p0, p1);
    };
    v16f_t n[2];
#pragma unroll
    for (int r = 0; r < 16; ++r) n[0][r] = n[1][r] = 0.f;
    if (it + 1 < ntile) {
      float ms = msub;  // its own value, or the compiler would lift the weights above the branch
      asm volatile("" : "+v"(ms));
      v8s_t kf[F_AHEAD];
#pragma unroll
      for (int f = 0; f < F_AHEAD; ++f) kf[f] = kfrag(nxt, f);
#pragma unroll
      for (int f = 0; f < 24; ++f) {
        n[f & 1] = mfma32<DT>(kf[f % F_AHEAD], qf[f >> 1], n[f & 1]);
        if (f + F_AHEAD < 24) kf[f % F_AHEAD] = kfrag(nxt, f + F_AHEAD);
        if (f >= 3 && f < 19) soft(f - 3, ms);
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) soft(e, msub);
    }
    l += rs + other_half(rs, h);
    {  // V^T fragments by transposed reads of the keys' rows
      const uint32_t vb = cur + va;
      auto vfrag = [&](int f) {  // product f: k-step f / 4, dims 32 (f & 3) ..
        const uint32_t at = (vb ^ (64 * (f & 3))) + 4096 * (f >> 2);
        const v4s_t lo = lds_read_tr(at), hi = lds_read_tr((at ^ 32) + 2048);
        return (v8s_t){lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      };
      v8s_t vf[F_AHEAD];
#pragma unroll
      for (int f = 0; f < F_AHEAD; ++f) vf[f] = vfrag(f);
#pragma unroll
      for (int f = 0; f < 16; ++f) {
        o[f & 3] = mfma32<DT>(vf[f % F_AHEAD], pf[f >> 2], o[f & 3]);
        if (f + F_AHEAD < 16) vf[f % F_AHEAD] = vfrag(f + F_AHEAD);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    s[0] = n[0];
    s[1] = n[1];
  }
  if constexpr (SPLIT) {
    float4* dst = reinterpret_cast<float4*>(a.part + pt * F_PART) + tid;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        dst[(4 * dt + i) * 256] = make_float4(o[dt][4 * i], o[dt][4 * i + 1], o[dt][4 * i + 2],
                                              o[dt][4 * i + 3]);
    if (h == 0) a.ml[pt * FQT + 32 * w + c] = make_float2(m, l);
    return;
  }
  __syncthreads();
  // a row that saw no key has l = 0: zeros (a NaN l stays one)
  const float il = l == 0.f ? 0.f : 1.f / l;
  {
    const int row = 32 * w + c;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint2 pk;
        pk.x = pack_dt<DT>(o[dt][4 * i] * il, o[dt][4 * i + 1] * il);
        pk.y = pack_dt<DT>(o[dt][4 * i + 2] * il, o[dt][4 * i + 3] * il);
        *reinterpret_cast<uint2*>(mla_lds + img_off(row, 4 * dt + i) + 8 * h) = pk;
      }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) {  // 128 rows x 16 chunks
    const int idx = i * 256 + tid, row = idx >> 4, ch = idx & 15;
    const int qr = q0 + row;
    if (qr < a.Sq)
      *reinterpret_cast<uint4*>(a.out + (((int64_t)b * a.Sq + qr) * a.H + hq) * DV + ch * 8) =
          *reinterpret_cast<const uint4*>(mla_lds + img_off(row, ch));
  }
}

// Joins the shares of a query tile, 32 dims (one dt of k_mla_fwd) per workgroup, in share order.
template <int DT>
__global__ void __launch_bounds__(256) k_mla_fwd_join(MlaFwdArgs a) {
  __shared__ __attribute__((aligned(16))) char img[FQT * 64];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, c = lane & 31, h = lane >> 5;
  const int dt = blockIdx.x & 3, tile = blockIdx.x >> 2;
  const int qt = tile % a.nqt, hq = (tile / a.nqt) % a.H, b = tile / (a.nqt * a.H);
  const float2* ml = a.ml + (int64_t)tile * a.ns * FQT + 32 * w + c;
  float M = -INFINITY;
  for (int i = 0; i < a.ns; ++i) M = fmaxf(M, ml[i * FQT].x);
  const float msub = M == -INFINITY ? 0.f : M;
  float l = 0.f, acc[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.f;
  const float4* pt =
      reinterpret_cast<const float4*>(a.part + (int64_t)tile * a.ns * F_PART) + 4 * dt * 256 + tid;
  for (int i = 0; i < a.ns; ++i, pt += F_PART / 4) {
    const float2 p = ml[i * FQT];
    if (p.y == 0.f) continue;  // the row saw no key there, and the share may not be written
    const float f = __builtin_amdgcn_exp2f(p.x - msub);
    l += f * p.y;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float4 v = pt[j * 256];
      acc[4 * j] += f * v.x;
      acc[4 * j + 1] += f * v.y;
      acc[4 * j + 2] += f * v.z;
      acc[4 * j + 3] += f * v.w;
    }
  }
  const float il = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int j = 0; j < 4; ++j) {  // dims 8 j + 4 h ..
    uint2 pk;
    pk.x = pack_dt<DT>(acc[4 * j] * il, acc[4 * j + 1] * il);
    pk.y = pack_dt<DT>(acc[4 * j + 2] * il, acc[4 * j + 3] * il);
    *reinterpret_cast<uint2*>(img + 64 * (32 * w + c) + 16 * j + 8 * h) = pk;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int idx = i * 256 + tid, row = idx >> 2, ch = idx & 3, qr = qt * FQT + row;
    if (qr < a.Sq)
      *reinterpret_cast<uint4*>(a.out + (((int64_t)b * a.Sq + qr) * a.H + hq) * DV + 32 * dt +
                                8 * ch) = *reinterpret_cast<const uint4*>(img + 64 * row + 16 * ch);
  }
}

// Shares of the keys per query tile. Two workgroups fit a CU; when the query tiles fill at most
// half of those 512 places, their keys are split, F_MIN tiles at least to a share: a chunk of 77
// rows of 128 heads over 4 Ki keys takes 79 us, 145 without shares (96 with one per CU).
int fwd_shares(int64_t B, int64_t H, int64_t Sq, int64_t Skv) {
  const int64_t tiles = B * H * ((Sq + FQT - 1) / FQT);
  const int64_t most = (Skv + FKT - 1) / FKT / F_MIN, fit = 512 / tiles;
  const int64_t n = most < fit ? most : fit;
  return n < 1 ? 1 : (int)n;
}

template <int DT>
int launch_fwd(const MlaFwdArgs& a, int64_t tiles, hipStream_t st) {
  constexpr int lds = 2 * F_STAGE;
  auto go = [&](auto split) {
    constexpr bool SP = decltype(split)::value;
    (void)hipFuncSetAttribute((const void*)k_mla_fwd<DT, SP>,
                              hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    hipLaunchKernelGGL((k_mla_fwd<DT, SP>), dim3((unsigned)(tiles * a.ns)), 256, lds, st, a);
  };
  if (a.ns == 1) {
    go(std::false_type{});
    return check_launch("lcq_mla_fwd_causal");
  }
  go(std::true_type{});
  if (int rc = check_launch("lcq_mla_fwd_causal")) return rc;
  hipLaunchKernelGGL(k_mla_fwd_join<DT>, dim3((unsigned)(tiles * 4)), 256, 0, st, a);
  return check_launch("lcq_mla_fwd_causal");
}

// ---------------------------------------------------------------------------------------
// Absorbed form over a paged latent cache
// ---------------------------------------------------------------------------------------
constexpr int DKT = 32;                          // keys per tile
constexpr int D_STAGE = DKT * (DL + DR) * 2;     // 36 KB: latent rows of 1 KB, rotary rows of 128 B
constexpr int D_RING = 8;                        // tiles whose key addresses are held in LDS
// tiles whose page numbers are held in LDS at a time: what the stages leave of 160 / 80 KB
constexpr int dec_tab(int nst) { return nst == 4 ? 64 : 16; }
constexpr int D_ROWS = 16;                       // query rows (token x head) per wave
constexpr int D_PART = D_ROWS * DL;              // floats of one row block's partial output
constexpr int D_CUTS = 48;                       // most partial outputs of a line of tiles, on average
constexpr int D_AHEAD = 4;                       // LDS fragments read ahead of their product

typedef float v4f_t __attribute__((ext_vector_type(4)));

// XOR of the 16 low chunks of a latent row: 16 rows differ (the row reads), and of the rows 4 q + i
// that 32 lanes read transposed, those of q = 0, 1 (2, 3) differ in chunk bit 1, which those reads
// leave free (with swz16, whose rows 4 apart differ in bit 0, every transposed read met a conflict)
__device__ __forceinline__ int dec_swz(int row) {
  return ((row & 3) << 2) | ((row >> 1) & 2) | ((row >> 3) & 1);
}

template <int DT>
__device__ __forceinline__ v4f_t mfma16(v8s_t a, v8s_t b, v4f_t c) {
  if constexpr (DT == LCQ_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf_t, a),
                                                   __builtin_bit_cast(v8bf_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8hf_t, a),
                                                  __builtin_bit_cast(v8hf_t, b), c, 0, 0, 0);
}

// max / sum over the four lanes of a row (lane & 15), left in all four
__device__ __forceinline__ float row_max(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float row_sum(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

struct MlaDecArgs {
  const uint16_t *ql, *qr;  // [B, Sq, H, 512], [B, Sq, H, 64]
  int64_t qlb, qls, qlh, qrb, qrs, qrh;
  const uint16_t *ckv, *kr; // [P, ps, 512], [P, ps, 64]
  int64_t cp, cs, rp, rs;   // page and slot strides
  const int32_t* table;     // [B, nb]
  const int32_t* lens;      // [B]
  uint16_t* out;            // [B, Sq, H, 512]
  float* part;              // [2 * wgs][RB][D_PART]
  float* ml;                // [2 * wgs][RB][16][2]
  int64_t P;
  int B, Sq, H, ps, nb, nrb, ny, wgs;  // nrb row blocks, ny = ceil(nrb / RB) of a workgroup
  float sl2;
};

// ---- how the work is divided -----------------------------------------------------------
// A sequence b takes n_b = max(1, ceil(len / 32)) key tiles, once for each of its ny groups of RB row
// blocks. The tiles of all (b, group) stand in one line, b major, and the line is cut into wgs
// equal ranges, one workgroup each: whatever
// the lengths, the workgroups do the same work. A (b, group) inside one range is finished by its
// workgroup; one that a cut divides leaves partial outputs in its workgroups' slots, 2 i for the
// segment that workgroup i begins with, 2 i + 1 for another one, and k_mla_join adds them in order.
__device__ __forceinline__ int dec_len(const MlaDecArgs& a, int b) {
  return (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.nb * a.ps);
}
__device__ __forceinline__ int dec_tiles(const MlaDecArgs& a, int b) {
  return max(1, (dec_len(a, b) + DKT - 1) / DKT);
}
// total tiles over all (b, group)
__device__ __forceinline__ int dec_total(const MlaDecArgs& a) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int b = lane; b < a.B; b += 64) n += dec_tiles(a, b);
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) n += __shfl_xor(n, d);
  return __builtin_amdgcn_readfirstlane(n) * a.ny;
}
// the sequence that holds tile `at`, and its first tile
__device__ __forceinline__ int dec_find(const MlaDecArgs& a, int at, int& first) {
  const int lane = threadIdx.x & 63;
  int base = 0;
  for (int b0 = 0; b0 < a.B; b0 += 64) {
    const int b = b0 + lane;
    const int t = b < a.B ? dec_tiles(a, b) * a.ny : 0;
    int inc = t;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(inc, d);
      if (lane >= d) inc += o;
    }
    const int total = __builtin_amdgcn_readfirstlane(__shfl(inc, 63));
    if (at < base + total) {
      const int l = __builtin_ctzll(__ballot(at < base + inc));
      first = __builtin_amdgcn_readfirstlane(base + __shfl(inc - t, l));
      return __builtin_amdgcn_readfirstlane(b0 + l);
    }
    base += total;
  }
  return a.B;
}
// tiles of a range
__device__ __forceinline__ int dec_step(const MlaDecArgs& a, int total) {
  return (total + a.wgs - 1) / a.wgs;
}

// One wave per 16 query rows, RB waves per workgroup sharing the key tiles. Scores are held
// transposed (mfma(K, Q^T): a lane has 8 keys of one row), so they turn into the B operand of
// O^T += C^T P^T in place; lane (c, q), register j of output block dt = dim 16 dt + 4 q + j of row
// c. Element j of a k-step's operands is key 16 (j >> 2) + 4 q + (j & 3).
// What bounds it: LDS reads, since every wave reads the whole tile for its 16 rows (32 rows a wave
// would halve that, but queries and outputs would take 512 registers; as it is 21 of the 256 are
// spilled with 8 waves, 7 with fewer, outside the loop over the tiles): 32 sequences of up to 8192
// tokens, 2 x 128 heads, 161-172 us with the join, 520-560 TF/s, LDS at work 49 % of the time (a
// third of it bank conflicts) and MFMA 32 %; one sequence of 777, 16 heads, 12 us. Up to 16 rows
// (RB 1) the compiler, which does not see the waits below, waits for the queries' loads all through
// a tile's score products, and so for the copies of the next tile that were just issued.
template <int DT, int RB, int NST>
__global__ void __launch_bounds__(64 * RB, 2) k_mla_dec(MlaDecArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char mla_lds[];
  // addresses of the keys of D_RING tiles: [tile][32] {latent row, rotary row}, and their masks
  typedef uint64_t addr_t[DKT][2];
  addr_t* addrs = reinterpret_cast<addr_t*>(mla_lds + NST * D_STAGE);
  uint32_t* mask_of = reinterpret_cast<uint32_t*>(mla_lds + NST * D_STAGE +
                                                  D_RING * sizeof(addr_t));
  int32_t* tab = reinterpret_cast<int32_t*>(mask_of + D_RING);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, q = lane >> 4;
  const int rows = a.Sq * a.H;
  const uint32_t lds0 = lds_addr(mla_lds);
  const int total = dec_total(a), step = dec_step(a, total);
  // neighbouring ranges (a sequence's) on one XCD
  int wg;
  {
    const int p = (int)blockIdx.x, nwg = (int)gridDim.x;
    const int xcd = p & 7, q8 = nwg >> 3, r8 = nwg & 7;
    wg = (xcd < r8 ? xcd * (q8 + 1) : r8 * (q8 + 1) + (xcd - r8) * q8) + (p >> 3);
  }
  int at = wg * step;
  if (at >= total) return;
  const int end = min(total, at + step), begin = at;
  // LDS offsets in a stage; a constant XOR walks the swizzled chunks of a row
  const int q4 = c >> 2, pp = c & 3;
  const uint32_t ka = 1024 * c + 16 * (q ^ dec_swz(c));                    // chunk 4 kk + q
  const uint32_t ra = DKT * 1024 + 128 * c + 16 * (q ^ ((c >> 1) & 7));     // rotary chunk
  const uint32_t va = 1024 * (4 * q + q4) + 16 * ((pp >> 1) ^ dec_swz(4 * q + q4)) + 8 * (pp & 1);
  const v4f_t zero = {0.f, 0.f, 0.f, 0.f};

  int first;
  int b = dec_find(a, at, first);
  while (at < end) {
    const int len = __builtin_amdgcn_readfirstlane(dec_len(a, b));
    const int nt = max(1, (len + DKT - 1) / DKT);
    const int y = __builtin_amdgcn_readfirstlane((at - first) / nt);
    const int t0 = at - first - y * nt, t1 = min(nt, t0 + (end - at));
    const int rb = y * RB + w;  // this wave's row block

    int p0 = 0;  // page that tab begins with
    // Addresses of tile t's keys, by 32 lanes of one wave (page numbers from LDS: a load from memory
    // here would wait for every tile in flight). A key past the length or on a page
    // outside the pool takes the tile's first existing key (or the pool's first row): nothing
    // behind a sequence is read.
    auto locate = [&](int t) {
      const int key = DKT * t + (lane & 31);
      const int pg = key / a.ps, slot = key - pg * a.ps;
      const int page = key < len ? tab[pg - p0] : -1;
      const bool ok = page >= 0 && page < a.P;
      const uint32_t mask = (uint32_t)__ballot(ok);
      const int src = mask ? __builtin_ctz(mask) : 0;
      uint64_t cb = reinterpret_cast<uint64_t>(a.ckv), rbs = reinterpret_cast<uint64_t>(a.kr);
      if (ok) {
        cb += 2 * (page * a.cp + slot * a.cs);
        rbs += 2 * (page * a.rp + slot * a.rs);
      }
      const uint64_t cb0 = __shfl(cb, src), rb0 = __shfl(rbs, src);
      if (!ok) { cb = cb0; rbs = rb0; }
      if (lane < 32) {
        addrs[t % D_RING][lane][0] = cb;
        addrs[t % D_RING][lane][1] = rbs;
      }
      if (lane == 0) mask_of[t % D_RING] = mask;
    };
    auto stage = [&](int t) {  // tile t's rows: DKT / RB + (w < 4) LDS-DMA instructions a wave
      const uint32_t st = lds0 + (t % NST) * D_STAGE;
      const addr_t& ad = addrs[t % D_RING];
#pragma unroll 4
      for (int j = 0; j < DKT / RB; ++j) {
        const int r = w * (DKT / RB) + j;
        dma16_at(st + 1024 * r, ad[r][0] + (lane ^ dec_swz(r)) * 16);
      }
#pragma unroll 1
      for (int g8 = w; g8 < DKT / 8; g8 += RB) {  // rotary rows, 8 keys an instruction
        const int r = 8 * g8 + (lane >> 3);
        dma16_at(st + DKT * 1024 + 1024 * g8, ad[r][1] + ((lane & 7) ^ ((r >> 1) & 7)) * 16);
      }
    };

    // a lane past the last row computes it again and stores nothing
    const int qrow = min(D_ROWS * rb + c, rows - 1), qi = qrow / a.H, qh = qrow - qi * a.H;
    v8s_t qf[18];  // Q^T as the B operand: Q[row][32 kk + 8 q + j]
    {
      const uint16_t* ql = a.ql + b * a.qlb + qi * a.qls + qh * a.qlh + 8 * q;
      const uint16_t* qr = a.qr + b * a.qrb + qi * a.qrs + qh * a.qrh + 8 * q;
#pragma unroll
      for (int kk = 0; kk < 18; ++kk)
        qf[kk] = *reinterpret_cast<const v8s_t*>(kk < 16 ? ql + 32 * kk : qr + 32 * (kk - 16));
    }
    const int pos = len - a.Sq + qi;  // last key this lane's row sees
    float m = -INFINITY, l = 0.f;
    v4f_t o[32];
#pragma unroll
    for (int dt = 0; dt < 32; ++dt) o[dt] = zero;

    for (int tb = t0; tb < t1; tb += dec_tab(NST)) {
    const int te = min(t1, tb + dec_tab(NST));
    p0 = DKT * tb / a.ps;
    const int np = (min(len, DKT * te) - 1) / a.ps - p0 + 1;  // an empty sequence: 0 or 1, unused
    __syncthreads();  // the tiles before are done with the stages and the addresses
    for (int i = tid; i < np; i += 64 * RB) tab[i] = a.table[(int64_t)b * a.nb + p0 + i];
    __syncthreads();
    for (int i = w; i < NST + 1; i += RB)
      if (tb + i < te) locate(tb + i);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NST - 1; ++i)
      if (tb + i < te) stage(tb + i);
    for (int t = tb; t < te; ++t) {
      const uint32_t cur = lds0 + (t % NST) * D_STAGE;
      // this wave's part of the tile has arrived (the NST - 2 tiles behind it may be in flight);
      // behind the barrier every wave's has, and every wave is done with the tile before, whose
      // stage is filled next
      if (NST > 2 && t + NST - 2 < te) {
        constexpr int n = (NST - 2) * (DKT / RB);
        if (w < DKT / 8) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(n + NST - 2) : "memory");
        else asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(n) : "memory");
      } else {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      }
      __builtin_amdgcn_s_barrier();
      if (t + NST - 1 < te) stage(t + NST - 1);
      const uint32_t vm = __builtin_amdgcn_readfirstlane(mask_of[t % D_RING]);
      if (vm != 0) {
        // S^T: register j of tile u = key 16 u + 4 q + j of the lane's row
        // (the two tiles in turn, so that a product does not wait for the one before it). K fragments
        // are read D_AHEAD products ahead; the scheduling barriers keep the compiler to that order
        // (left alone it waits for each read right before its product)
        v4f_t s[2] = {zero, zero};
        const uint32_t kb = cur + ka, rp = cur + ra;
        auto kfrag = [&](int f) {  // product f: k-step f / 2 of tile f & 1
          const int kk = f >> 1, u = f & 1;
          return kk < 16 ? lds_read16((kb ^ (64 * (kk & 3))) + 256 * (kk >> 2) + 16384 * u)
                         : lds_read16((rp ^ (64 * (kk - 16))) + 2048 * u);
        };
        v8s_t kf[D_AHEAD];
#pragma unroll
        for (int f = 0; f < D_AHEAD; ++f) kf[f] = kfrag(f);
#pragma unroll
        for (int f = 0; f < 36; ++f) {
          s[f & 1] = mfma16<DT>(kf[f % D_AHEAD], qf[f >> 1], s[f & 1]);
          if (f + D_AHEAD < 36) kf[f % D_AHEAD] = kfrag(f + D_AHEAD);
          __builtin_amdgcn_sched_barrier(0);
        }
        // keys this lane's row sees: bit = key offset in the tile
        const int d = pos - DKT * t;
        const uint32_t see = vm & (d >= 31 ? ~0u : d < 0 ? 0u : (2u << d) - 1);
        if (!__all(see == ~0u)) {
          const uint32_t sh = see >> (4 * q);
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (!((sh >> (16 * u + j)) & 1)) s[u][j] = -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < 8; ++j) mx = fmaxf(mx, s[j >> 2][j & 3]);
        mx = row_max(mx) * a.sl2;
        if (__any(mx > m + 8.f)) {  // as in k_mla_fwd
          const float mn = mx > m + 8.f ? mx : m;
          const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
          l *= alpha;
          m = mn;
#pragma unroll
          for (int dt = 0; dt < 32; ++dt) o[dt] *= alpha;
        }
        const float msub = m == -INFINITY ? 0.f : m;
        float rsum = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float p = __builtin_amdgcn_exp2f(__fmaf_rn(s[j >> 2][j & 3], a.sl2, -msub));
          s[j >> 2][j & 3] = p;
          rsum += p;
        }
        l += row_sum(rsum);
        v8s_t pf;
        uint32_t* pw = reinterpret_cast<uint32_t*>(&pf);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          pw[j] = pack_dt<DT>(s[j >> 1][2 * (j & 1)], s[j >> 1][2 * (j & 1) + 1]);
        const uint32_t vb = cur + va;
        auto vfrag = [&](int dt) {
          const uint32_t ad = (vb ^ (32 * (dt & 7))) + 256 * (dt >> 3);
          const v4s_t lo = lds_read_tr(ad), hi = lds_read_tr(ad + 16384);
          return (v8s_t){lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        };
        v8s_t vf[D_AHEAD];
#pragma unroll
        for (int dt = 0; dt < D_AHEAD; ++dt) vf[dt] = vfrag(dt);
#pragma unroll
        for (int dt = 0; dt < 32; ++dt) {
          o[dt] = mfma16<DT>(vf[dt % D_AHEAD], pf, o[dt]);
          if (dt + D_AHEAD < 32) vf[dt % D_AHEAD] = vfrag(dt + D_AHEAD);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      // the addresses of the tile staged in the iteration after next (in the ring's slot of a
      // tile that every wave has finished), by the waves in turn
      if (t + NST + 1 < te && w == t % RB) locate(t + NST + 1);
    }
    }

    if (rb < a.nrb) {
      if (t0 == 0 && t1 == nt) {  // the whole line of keys: finished
        const float il = l == 0.f ? 0.f : 1.f / l;  // a row without a key: zeros
        const int row = D_ROWS * rb + (threadIdx.x & 15);
        if (row < rows) {
          uint16_t* op = a.out + ((int64_t)b * rows + row) * DL;
#pragma unroll
          for (int dt = 0; dt < 32; ++dt) {
            uint2 pk;
            pk.x = pack_dt<DT>(o[dt][0] * il, o[dt][1] * il);
            pk.y = pack_dt<DT>(o[dt][2] * il, o[dt][3] * il);
            *reinterpret_cast<uint2*>(op + 16 * dt + 4 * q) = pk;
          }
        }
      } else {
        const int64_t slot = (2 * (int64_t)wg + (at == begin ? 0 : 1)) * RB + w;
        if (q == 0) {
          a.ml[(slot * D_ROWS + c) * 2] = m;
          a.ml[(slot * D_ROWS + c) * 2 + 1] = l;
        }
        v4f_t* pt = reinterpret_cast<v4f_t*>(a.part + slot * D_PART);
#pragma unroll
        for (int dt = 0; dt < 32; ++dt) pt[dt * 64 + lane] = o[dt];
      }
    }
    at += t1 - t0;
    if (y == a.ny - 1 && t1 == nt) {
      first += nt * a.ny;
      ++b;
    }
  }
}

// Joins the partial outputs of one row block in key order. A thread takes one float4 (4 dims of a
// row) of every partial (W 1: 8 workgroups per block), or of a quarter of them, the workgroup's
// four waves one after the other in the end (W 4: 32 workgroups per block, for many partials).
template <int DT, int RB, int W>
__global__ void __launch_bounds__(256) k_mla_join(MlaDecArgs a) {
  __shared__ float red[W == 1 ? 1 : 3][64][6];
  const int b = blockIdx.y, rb = blockIdx.x / (8 * W), wave = threadIdx.x >> 6;
  const int y = rb / RB, w = rb - y * RB;
  const int total = dec_total(a), step = dec_step(a, total);
  int s = 0;
  {
    const int lane = threadIdx.x & 63;
    for (int i = lane; i < b; i += 64) s += dec_tiles(a, i);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
    s *= a.ny;
  }
  const int nt = dec_tiles(a, b);
  s = __builtin_amdgcn_readfirstlane(s) + y * nt;          // this block's first tile
  const int i0 = s / step, i1 = (s + nt - 1) / step;       // the workgroups that hold its tiles
  if (i0 == i1) return;                                    // finished by its workgroup
  const int at4 = W == 1 ? (blockIdx.x & 7) * 256 + threadIdx.x  // float4 of the block: dt * 64 + lane
                         : (blockIdx.x & 31) * 64 + (threadIdx.x & 63);
  const int lane = at4 & 63, c = lane & 15, q = lane >> 4, dt = at4 >> 6;
  const int row = D_ROWS * rb + c, rows = a.Sq * a.H;
  // slot of workgroup i's segment: its second only where its range began before this block
  auto slot = [&](int i) { return (2 * (int64_t)i + (i == i0 && i0 * step < s ? 1 : 0)) * RB + w; };
  float m = -INFINITY, l = 0.f;
  v4f_t acc = {0.f, 0.f, 0.f, 0.f};
  auto add = [&](float m1, float l1, v4f_t v1) {
    if (l1 == 0.f) return;  // the row saw no key there (a NaN sum goes on)
    const float mn = fmaxf(m, m1), ref = mn == -INFINITY ? 0.f : mn;
    const float f0 = __builtin_amdgcn_exp2f(m - ref), f1 = __builtin_amdgcn_exp2f(m1 - ref);
    l = l * f0 + l1 * f1;
    acc = acc * f0 + v1 * f1;
    m = mn;
  };
  // four partials in flight; the running maximum rescales
  const int cnt = i1 - i0 + 1;
  const int lo = i0 + (W == 1 ? 0 : cnt * wave / W), hi = i0 + (W == 1 ? cnt : cnt * (wave + 1) / W);
  for (int i = lo; i < hi; i += 4) {
    float ms[4], ls[4];
    v4f_t v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int64_t at = slot(min(i + j, hi - 1));
      ms[j] = a.ml[(at * D_ROWS + c) * 2];
      ls[j] = a.ml[(at * D_ROWS + c) * 2 + 1];
      v[j] = reinterpret_cast<const v4f_t*>(a.part + at * D_PART)[at4];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j < hi) add(ms[j], ls[j], v[j]);
  }
  if constexpr (W > 1) {
    if (wave > 0) {
      float* r = red[wave - 1][lane];
      r[0] = m; r[1] = l;
#pragma unroll
      for (int j = 0; j < 4; ++j) r[2 + j] = acc[j];
    }
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int x = 0; x < W - 1; ++x) {
      const float* r = red[x][lane];
      add(r[0], r[1], v4f_t{r[2], r[3], r[4], r[5]});
    }
  }
  if (row >= rows) return;
  const float il = l == 0.f ? 0.f : 1.f / l;
  uint2 pk;
  pk.x = pack_dt<DT>(acc[0] * il, acc[1] * il);
  pk.y = pack_dt<DT>(acc[2] * il, acc[3] * il);
  *reinterpret_cast<uint2*>(a.out + ((int64_t)b * rows + row) * DL + 16 * dt + 4 * q) = pk;
}

struct DecPlan {
  int rb, nrb, ny, wgs;
};
// RB row blocks per workgroup (all heads of a token share its key tiles); as many workgroups as the
// chip holds at once, one of 8 waves per CU (144 KB of stages), two of fewer; and no more than
// D_CUTS per line of tiles, since each leaves a partial output (one sequence of 4000 tokens, 128
// heads: 29 us, 35 with a workgroup for each of its 125 tiles, 32 with 24)
DecPlan dec_plan(int64_t B, int64_t rows, int64_t maxlen) {
  DecPlan p;
  p.nrb = (int)((rows + D_ROWS - 1) / D_ROWS);
  p.rb = p.nrb <= 1 ? 1 : p.nrb <= 2 ? 2 : p.nrb <= 4 ? 4 : 8;
  p.ny = (p.nrb + p.rb - 1) / p.rb;
  const int64_t lines = B * p.ny, tiles = (maxlen + DKT - 1) / DKT;
  const int64_t most = lines * (tiles < D_CUTS ? tiles : D_CUTS);
  const int64_t fit = p.rb == 8 ? 256 : 512;
  p.wgs = (int)(most < fit ? most : fit);
  return p;
}

bool dec_rows_ok(int64_t B, int64_t Sq, int64_t H) {
  return B <= 65535 && Sq <= (1 << 20) && H <= (1 << 20) && Sq * H <= (1 << 20);
}

template <int DT, int RB, int NST>
int launch_dec(const MlaDecArgs& a, hipStream_t st) {
  constexpr int lds = NST * D_STAGE + D_RING * (DKT * 16 + 4) + (dec_tab(NST) * DKT + 1) * 4;
  static_assert(lds <= (NST == 4 ? 163840 : 81920), "one / two workgroups per CU");
  static_assert(NST + 2 <= D_RING, "tiles whose addresses are live");
  (void)hipFuncSetAttribute((const void*)k_mla_dec<DT, RB, NST>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  hipLaunchKernelGGL((k_mla_dec<DT, RB, NST>), dim3((unsigned)a.wgs), 64 * RB, lds, st, a);
  if (int rc = check_launch("lcq_mla_decode")) return rc;
  if (a.wgs == 1) return LCQ_OK;
  // the mean number of partials of a row block decides (one sequence of 4000 tokens, 16 heads: 17
  // against 26 us for both kernels; 32 sequences of 8192, 3 partials each: 177 against 161)
  if (a.wgs >= 8 * a.B * a.ny)
    hipLaunchKernelGGL((k_mla_join<DT, RB, 4>), dim3((unsigned)a.nrb * 32, (unsigned)a.B), 256, 0, st,
                       a);
  else
    hipLaunchKernelGGL((k_mla_join<DT, RB, 1>), dim3((unsigned)a.nrb * 8, (unsigned)a.B), 256, 0, st,
                       a);
  return check_launch("lcq_mla_decode");
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace lcq

using namespace lcq;

extern "C" int64_t lcq_mla_fwd_causal_workspace_bytes(int64_t B, int64_t H, int64_t Sq,
                                                      int64_t Skv) {
  if (B <= 0 || H <= 0 || Sq <= 0 || Skv <= 0 || B >= (1 << 24) || H >= (1 << 24) ||
      B * H >= (int64_t(1) << 31) || Sq >= (1 << 28) || Skv >= (1 << 28))
    return 0;
  const int64_t ns = fwd_shares(B, H, Sq, Skv);
  return ns == 1 ? 0 : B * H * ((Sq + FQT - 1) / FQT) * ns * (F_PART + 2 * FQT) * 4;
}

extern "C" int lcq_mla_fwd_causal(const void* q_nope, const int64_t* q_nope_strides,
                                  const void* q_rope, const int64_t* q_rope_strides,
                                  const void* k_nope, const int64_t* k_nope_strides,
                                  const void* k_rope, const int64_t* k_rope_strides,
                                  const void* v, const int64_t* v_strides, int dtype, int64_t B,
                                  int64_t H, int64_t Sq, int64_t Skv, const int32_t* q_start,
                                  const int32_t* kv_lens, float scale, void* out, void* workspace,
                                  int64_t ws_bytes, void* stream) {
  LCQ_REQUIRE(dtype == LCQ_BF16 || dtype == LCQ_F16, "bf16 / fp16 only");
  LCQ_REQUIRE(B >= 0 && H > 0 && Sq >= 0 && Skv > 0, "bad shape");
  LCQ_REQUIRE(Sq < (1 << 28) && Skv < (1 << 28), "sequence too long");
  LCQ_REQUIRE(scale > 0.f && scale < 3.4e38f, "scale must be positive and finite");
  if (B == 0 || Sq == 0) return LCQ_OK;
  LCQ_REQUIRE(q_nope && q_rope && k_nope && k_rope && v && out && q_nope_strides &&
                  q_rope_strides && k_nope_strides && k_rope_strides && v_strides,
              "null pointer");
  LCQ_REQUIRE(q_start || Skv >= Sq, "more queries than keys needs q_start");
  const int64_t nqt = (Sq + FQT - 1) / FQT;
  LCQ_REQUIRE(B < (1 << 24) && H < (1 << 24) && B * H < (int64_t(1) << 31) &&
                  B * H * nqt < (int64_t(1) << 31),
              "shape too large");
  int64_t all = 0;
  for (int i = 0; i < 3; ++i)
    all |= q_nope_strides[i] | q_rope_strides[i] | k_nope_strides[i] | v_strides[i];
  all |= k_rope_strides[0] | k_rope_strides[1];
  LCQ_REQUIRE((all & 7) == 0, "row strides must be multiples of 8 elements");
  LCQ_REQUIRE(al16(q_nope) && al16(q_rope) && al16(k_nope) && al16(k_rope) && al16(v) && al16(out),
              "16-byte aligned tensors required");
  auto tile_ok = [](int64_t s) { return s >= 0 && s < (int64_t(1) << 24); };
  LCQ_REQUIRE(tile_ok(k_nope_strides[2]) && tile_ok(v_strides[2]) && tile_ok(k_rope_strides[1]),
              "key / value sequence strides must be in [0, 2^24)");
  MlaFwdArgs a{};
  a.qn = static_cast<const uint16_t*>(q_nope);
  a.qr = static_cast<const uint16_t*>(q_rope);
  a.kn = static_cast<const uint16_t*>(k_nope);
  a.kr = static_cast<const uint16_t*>(k_rope);
  a.v = static_cast<const uint16_t*>(v);
  a.out = static_cast<uint16_t*>(out);
  a.qnb = q_nope_strides[0]; a.qnh = q_nope_strides[1]; a.qns = q_nope_strides[2];
  a.qrb = q_rope_strides[0]; a.qrh = q_rope_strides[1]; a.qrs = q_rope_strides[2];
  a.knb = k_nope_strides[0]; a.knh = k_nope_strides[1]; a.kns = k_nope_strides[2];
  a.krb = k_rope_strides[0]; a.krs = k_rope_strides[1];
  a.vb = v_strides[0]; a.vh = v_strides[1]; a.vs = v_strides[2];
  a.q_start = q_start;
  a.kv_lens = kv_lens;
  a.Sq = (int)Sq; a.Skv = (int)Skv; a.H = (int)H; a.nqt = (int)nqt;
  a.sl2 = scale * 1.44269504088896340736f;
  a.ns = fwd_shares(B, H, Sq, Skv);
  const int64_t need = lcq_mla_fwd_causal_workspace_bytes(B, H, Sq, Skv);
  LCQ_REQUIRE(ws_bytes >= need && (need == 0 || (workspace && al16(workspace))),
              "workspace too small (lcq_mla_fwd_causal_workspace_bytes)");
  if (a.ns > 1) {
    a.part = static_cast<float*>(workspace);
    a.ml = reinterpret_cast<float2*>(a.part + B * H * nqt * a.ns * F_PART);
  }
  return dtype == LCQ_BF16 ? launch_fwd<LCQ_BF16>(a, B * H * nqt, as_stream(stream))
                           : launch_fwd<LCQ_F16>(a, B * H * nqt, as_stream(stream));
}

extern "C" int64_t lcq_mla_decode_workspace_bytes(int64_t B, int64_t Sq, int64_t H,
                                                  int64_t max_len) {
  if (B <= 0 || Sq <= 0 || H <= 0 || max_len <= 0 || !dec_rows_ok(B, Sq, H) ||
      max_len >= (int64_t(1) << 30))
    return 0;
  const DecPlan p = dec_plan(B, Sq * H, max_len);
  return p.wgs == 1 ? 0 : 2 * (int64_t)p.wgs * p.rb * (D_PART + 2 * D_ROWS) * 4;
}

extern "C" int lcq_mla_decode(const void* q_latent, const int64_t* q_latent_strides,
                              const void* q_rope, const int64_t* q_rope_strides, const void* ckv,
                              const int64_t* ckv_strides, const void* k_rope,
                              const int64_t* k_rope_strides, int64_t pages, int64_t page_size,
                              const int32_t* block_table, int64_t nb, const int32_t* kv_lens,
                              int dtype, int64_t B, int64_t Sq, int64_t H, float scale, void* out,
                              void* workspace, int64_t ws_bytes, void* stream) {
  LCQ_REQUIRE(dtype == LCQ_BF16 || dtype == LCQ_F16, "bf16 / fp16 only");
  LCQ_REQUIRE(B >= 0 && H > 0 && Sq >= 0 && pages > 0 && page_size > 0 && nb > 0, "bad shape");
  LCQ_REQUIRE(pages < (int64_t(1) << 31) && page_size < (1 << 28) && nb < (1 << 28) &&
                  nb * page_size < (1 << 30),
              "cache too long");
  LCQ_REQUIRE(dec_rows_ok(B, Sq, H), "too many query rows");
  LCQ_REQUIRE(scale > 0.f && scale < 3.4e38f, "scale must be positive and finite");
  if (B == 0 || Sq == 0) return LCQ_OK;
  LCQ_REQUIRE(q_latent && q_rope && ckv && k_rope && block_table && kv_lens && out &&
                  q_latent_strides && q_rope_strides && ckv_strides && k_rope_strides,
              "null pointer");
  int64_t all = ckv_strides[0] | ckv_strides[1] | k_rope_strides[0] | k_rope_strides[1];
  for (int i = 0; i < 3; ++i) all |= q_latent_strides[i] | q_rope_strides[i];
  LCQ_REQUIRE((all & 7) == 0, "row strides must be multiples of 8 elements");
  LCQ_REQUIRE(al16(q_latent) && al16(q_rope) && al16(ckv) && al16(k_rope) && al16(out),
              "16-byte aligned tensors required");
  const DecPlan p = dec_plan(B, Sq * H, nb * page_size);
  LCQ_REQUIRE(B * p.ny * ((nb * page_size + DKT - 1) / DKT) < (int64_t(1) << 30), "cache too long");
  const int64_t need = lcq_mla_decode_workspace_bytes(B, Sq, H, nb * page_size);
  LCQ_REQUIRE(ws_bytes >= need && (need == 0 || (workspace && al16(workspace))),
              "workspace too small (lcq_mla_decode_workspace_bytes)");
  MlaDecArgs a{};
  a.ql = static_cast<const uint16_t*>(q_latent);
  a.qr = static_cast<const uint16_t*>(q_rope);
  a.qlb = q_latent_strides[0]; a.qls = q_latent_strides[1]; a.qlh = q_latent_strides[2];
  a.qrb = q_rope_strides[0]; a.qrs = q_rope_strides[1]; a.qrh = q_rope_strides[2];
  a.ckv = static_cast<const uint16_t*>(ckv);
  a.kr = static_cast<const uint16_t*>(k_rope);
  a.cp = ckv_strides[0]; a.cs = ckv_strides[1];
  a.rp = k_rope_strides[0]; a.rs = k_rope_strides[1];
  a.table = block_table;
  a.lens = kv_lens;
  a.out = static_cast<uint16_t*>(out);
  a.P = pages;
  a.B = (int)B; a.Sq = (int)Sq; a.H = (int)H; a.ps = (int)page_size; a.nb = (int)nb;
  a.nrb = p.nrb; a.ny = p.ny; a.wgs = p.wgs;
  a.part = static_cast<float*>(workspace);
  a.ml = a.part ? a.part + 2 * (int64_t)p.wgs * p.rb * D_PART : nullptr;
  a.sl2 = scale * 1.44269504088896340736f;
  hipStream_t st = as_stream(stream);
  auto go = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    return p.rb == 8   ? launch_dec<DT, 8, 4>(a, st)
           : p.rb == 4 ? launch_dec<DT, 4, 2>(a, st)
           : p.rb == 2 ? launch_dec<DT, 2, 2>(a, st)
                       : launch_dec<DT, 1, 2>(a, st);
  };
  return dtype == LCQ_BF16 ? go(std::integral_constant<int, LCQ_BF16>{})
                           : go(std::integral_constant<int, LCQ_F16>{});
}
