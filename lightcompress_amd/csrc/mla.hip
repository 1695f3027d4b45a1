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

// ---------------------------------------------------------------------------------------
// Expanded form
// ---------------------------------------------------------------------------------------
constexpr int FQT = 128;  // query rows per workgroup (4 waves of 32)
constexpr int FKT = 64;   // keys per tile
constexpr int F_STAGE = FKT * (DN + DR + DV) * 2;  // 40 KB

struct MlaFwdArgs {
  const uint16_t *qn, *qr, *kn, *kr, *v;
  uint16_t* out;            // [B, Sq, H, 128]
  int64_t qnb, qnh, qns, qrb, qrh, qrs, knb, knh, kns, krb, krs, vb, vh, vs;  // elements
  const int32_t* q_start;   // nullable [B]: position of query 0 (default Skv - Sq)
  const int32_t* kv_lens;   // nullable [B]: valid keys (default Skv)
  int Sq, Skv, H, nqt;
  float sl2;                // scale * log2(e)
};

// One 64-key tile of the three images by LDS-DMA: 10 instructions per wave. The base moves with the
// tile (64-bit), so only a tile's own span has to fit 32 bits. Keys past `last` re-read it: what
// lies behind a sequence is never loaded.
__device__ __forceinline__ void fwd_stage(uint32_t st, const uint16_t* kn, const uint16_t* kr,
                                          const uint16_t* v, const MlaFwdArgs& a, int k0, int last,
                                          int w, int lane) {
  const uint16_t *bn = uni(kn + k0 * a.kns), *bv = uni(v + k0 * a.vs), *br = uni(kr + k0 * a.krs);
  const int lim = last - k0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = 4 * (4 * w + j) + (lane >> 4);
    const int ch = (lane & 15) ^ swz16(row);
    const uint32_t key = min(row, lim);
    dma16(st + 1024 * (4 * w + j), bn, key * (uint32_t)a.kns * 2 + ch * 16);
    dma16(st + 16384 + 1024 * (4 * w + j), bv, key * (uint32_t)a.vs * 2 + ch * 16);
  }
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int row = 8 * (2 * w + j) + (lane >> 3);
    const int ch = (lane & 7) ^ ((row >> 1) & 7);
    const uint32_t key = min(row, lim);
    dma16(st + 32768 + 1024 * (2 * w + j), br, key * (uint32_t)a.krs * 2 + ch * 16);
  }
}

template <int DT>
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
  const int hq = (L / a.nqt) % a.H, b = L / (a.nqt * a.H);
  const int q0 = qt * FQT;
  const int klen = a.kv_lens ? min(max(a.kv_lens[b], 0), a.Skv) : a.Skv;
  const int qs = a.q_start ? min(max(a.q_start[b], -(1 << 29)), 1 << 29) : a.Skv - a.Sq;
  const int kend = min(klen, qs + q0 + FQT);
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
  const uint16_t* knp = a.kn + b * a.knb + hq * a.knh;
  const uint16_t* krp = a.kr + b * a.krb;
  const uint16_t* vp = a.v + b * a.vb + hq * a.vh;
  fwd_stage(lds0, knp, krp, vp, a, 0, klen - 1, w, lane);

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
  const int wmin = min(qs + q0 + 32 * w, klen - 1);  // the least of the wave's rows
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

  int it = 0;
  for (int k0 = 0; k0 < kend; k0 += FKT, ++it) {
    const uint32_t cur = lds0 + (it & 1) * F_STAGE;
    // every wave is done with the stage the next tile overwrites
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    if (k0 + FKT < kend) {
      fwd_stage(lds0 + ((it & 1) ^ 1) * F_STAGE, knp, krp, vp, a, k0 + FKT, klen - 1, w, lane);
      asm volatile("s_waitcnt vmcnt(10)" ::: "memory");  // this tile's loads, not the next's
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    __builtin_amdgcn_s_barrier();  // this tile is in LDS for every wave
    // S^T tiles t: register r holds key k0 + 32 t + (r & 3) + 8 (r >> 2) + 4 h of the lane's row
    v16f_t s[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
#pragma unroll
      for (int r = 0; r < 16; ++r) s[t][r] = 0.f;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk)
        s[t] = mfma32<DT>(lds_read16(((cur + ka) ^ (32 * kk)) + 8192 * t), qf[kk], s[t]);
#pragma unroll
      for (int kk = 0; kk < 4; ++kk)
        s[t] = mfma32<DT>(lds_read16(((cur + ra) ^ (32 * kk)) + 4096 * t), qf[8 + kk], s[t]);
    }
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
    const float mn = fmaxf(m, mx);
    const float alpha = (mn == -INFINITY) ? 1.f : __builtin_amdgcn_exp2f(m - mn);
    const float msub = (mn == -INFINITY) ? 0.f : mn;
    float rs = 0.f;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float p = __builtin_amdgcn_exp2f(__fmaf_rn(s[t][r], a.sl2, -msub));
        s[t][r] = p;
        rs += p;
      }
    rs += other_half(rs, h);
    l = l * alpha + rs;
    m = mn;
    if (alpha != 1.f) {
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[dt][r] *= alpha;
    }
    // O^T += V^T P^T; k-step (t, s2): score registers 8 s2 .. 8 s2 + 7 of tile t, V^T fragments by
    // transposed reads of the same keys' rows
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int s2 = 0; s2 < 2; ++s2) {
        v8s_t pf;
        uint32_t* pw = reinterpret_cast<uint32_t*>(&pf);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          pw[j] = pack_dt<DT>(s[t][8 * s2 + 2 * j], s[t][8 * s2 + 2 * j + 1]);
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) {
          const uint32_t at = (cur + va) ^ (64 * dt);
          const v4s_t lo = lds_read_tr(at + 256 * (32 * t + 16 * s2));
          const v4s_t hi = lds_read_tr((at ^ 32) + 256 * (32 * t + 16 * s2 + 8));
          const v8s_t vf = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
          o[dt] = mfma32<DT>(vf, pf, o[dt]);
        }
      }
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

// ---------------------------------------------------------------------------------------
// Absorbed form over a paged latent cache
// ---------------------------------------------------------------------------------------
constexpr int DKT = 32;                          // keys per tile
constexpr int D_STAGE = DKT * (DL + DR) * 2;     // 36 KB: latent rows of 1 KB, rotary rows of 128 B
constexpr int D_TAB = 2048;                      // keys whose page numbers are held in LDS at a time
constexpr int D_ROWS = 16;                       // query rows (token x head) per wave
constexpr int D_PART = D_ROWS * DL;              // floats of one row block's partial output

typedef float v4f_t __attribute__((ext_vector_type(4)));

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
  float* part;              // [splits][B][nrb][D_PART]
  float* ml;                // [splits][B][nrb][16][2]
  int64_t P;
  int B, Sq, H, ps, nb, nrb, chunk, nsplit;
  float sl2;
};

// One wave per 16 query rows, RB waves per workgroup sharing the key tiles. Scores are held
// transposed (mfma(K, Q^T): a lane has 8 keys of one row), so they turn into the B operand of
// O^T += C^T P^T in place; lane (c, q), register j of output block dt = dim 16 dt + 4 q + j of row
// c. Element j of a k-step's operands is key 16 (j >> 2) + 4 q + (j & 3).
template <int DT, int RB, int NST>
__global__ void __launch_bounds__(64 * RB, 2) k_mla_dec(MlaDecArgs a) {
  extern __shared__ __attribute__((aligned(1024))) char mla_lds[];
  int32_t* tab = reinterpret_cast<int32_t*>(mla_lds + NST * D_STAGE);
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane & 15, q = lane >> 4;
  const int sp = blockIdx.x, b = blockIdx.z;
  const int rb = blockIdx.y * RB + w;  // this wave's row block
  const int rows = a.Sq * a.H;
  const int len = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.nb * a.ps);
  const int kbeg = sp * a.chunk, kend = min(len, kbeg + a.chunk);
  const int row = D_ROWS * rb + c;
  const int qi = row / a.H, qh = row - qi * a.H;
  const bool live = row < rows;
  const uint32_t lds0 = lds_addr(mla_lds);

  v8s_t qf[18];  // Q^T as the B operand: Q[row][32 kk + 8 q + j]
#pragma unroll
  for (int kk = 0; kk < 18; ++kk) {
    qf[kk] = (v8s_t){0, 0, 0, 0, 0, 0, 0, 0};
    if (live)
      qf[kk] = *reinterpret_cast<const v8s_t*>(
          kk < 16 ? a.ql + b * a.qlb + qi * a.qls + qh * a.qlh + 32 * kk + 8 * q
                  : a.qr + b * a.qrb + qi * a.qrs + qh * a.qrh + 32 * (kk - 16) + 8 * q);
  }
  const int pos = len - a.Sq + qi;  // last key this lane's row sees
  float m = -INFINITY, l = 0.f;
  const v4f_t zero = {0.f, 0.f, 0.f, 0.f};
  v4f_t o[32];
#pragma unroll
  for (int dt = 0; dt < 32; ++dt) o[dt] = zero;

  // LDS offsets in a stage; a constant XOR walks the swizzled chunks of a row
  const int q4 = c >> 2, pp = c & 3;
  const uint32_t ka = 1024 * c + 16 * (q ^ swz16(c));                      // chunk 4 kk + q
  const uint32_t ra = DKT * 1024 + 128 * c + 16 * (q ^ ((c >> 1) & 7));     // rotary chunk
  const uint32_t va = 1024 * (4 * q + q4) + 16 * ((pp >> 1) ^ (q4 << 2 | q)) + 8 * (pp & 1);

  // Stage the tile of keys kb .. kb + 31; returns the mask of its keys that exist. A key past the
  // end or on a page outside the pool is loaded from the tile's first existing key (or the pool's
  // first row): nothing behind a sequence is read.
  auto stage = [&](uint32_t st, int kb, int p0) -> uint32_t {
    const int key = kb + (lane & 31);
    const int pg = key / a.ps, slot = key - pg * a.ps;
    const int page = key < kend ? tab[pg - p0] : -1;
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
#pragma unroll
    for (int j = 0; j < DKT / RB; ++j) {
      const int r = w * (DKT / RB) + j;
      const uint64_t row = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(cb >> 32), r)
                            << 32) |
                           (uint32_t)__builtin_amdgcn_readlane((uint32_t)cb, r);
      dma16(st + 1024 * r, reinterpret_cast<const void*>(row), (lane ^ swz16(r)) * 16);
    }
    // rotary rows, 8 keys an instruction
    for (int g8 = w; g8 < DKT / 8; g8 += RB) {
      const int r = 8 * g8 + (lane >> 3);
      dma16_at(st + DKT * 1024 + 1024 * g8,
               __shfl(rbs, r) + ((lane & 7) ^ ((r >> 1) & 7)) * 16);
    }
    return mask;
  };

  for (int kt = kbeg; kt < kend; kt += D_TAB) {
    const int ke = min(kend, kt + D_TAB);
    const int p0 = kt / a.ps, p1 = (ke - 1) / a.ps;
    __syncthreads();
    for (int i = tid; i <= p1 - p0; i += 64 * RB) tab[i] = a.table[(int64_t)b * a.nb + p0 + i];
    __syncthreads();
    uint32_t masks[NST];
#pragma unroll
    for (int i = 0; i < NST - 1; ++i)
      masks[i] = kt + DKT * i < ke ? stage(lds0 + i * D_STAGE, kt + DKT * i, p0) : 0;
    for (int k0 = kt; k0 < ke; k0 += DKT) {
      const int t = (k0 - kt) / DKT;
      const uint32_t cur = lds0 + (t % NST) * D_STAGE;
      // this wave's part of the tile has arrived; behind the barrier every wave's has, and every
      // wave is done with the tile before, whose stage is filled next
      asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      const int kn = k0 + DKT * (NST - 1);
      const uint32_t vm = masks[0];
#pragma unroll
      for (int i = 0; i < NST - 2; ++i) masks[i] = masks[i + 1];
      masks[NST - 2] = kn < ke ? stage(lds0 + ((t + NST - 1) % NST) * D_STAGE, kn, p0) : 0;
      if (vm == 0) continue;

      // S^T: register j of tile u = key 16 u + 4 q + j of the lane's row
      v4f_t s[2] = {zero, zero};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
#pragma unroll
        for (int kk = 0; kk < 16; ++kk)
          s[u] = mfma16<DT>(
              lds_read16(((cur + ka) ^ (64 * (kk & 3))) + 256 * (kk >> 2) + 16384 * u), qf[kk],
              s[u]);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
          s[u] = mfma16<DT>(lds_read16(((cur + ra) ^ (64 * kk)) + 2048 * u), qf[16 + kk], s[u]);
      }
      // keys this lane's row sees: bit = key offset in the tile
      const int d = pos - k0;
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
      const float mn = fmaxf(m, mx);
      const float alpha = (mn == -INFINITY) ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      const float msub = (mn == -INFINITY) ? 0.f : mn;
      float rsum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float p = __builtin_amdgcn_exp2f(__fmaf_rn(s[j >> 2][j & 3], a.sl2, -msub));
        s[j >> 2][j & 3] = p;
        rsum += p;
      }
      rsum = row_sum(rsum);
      l = l * alpha + rsum;
      m = mn;
      if (!__all(alpha == 1.f)) {
#pragma unroll
        for (int dt = 0; dt < 32; ++dt) o[dt] *= alpha;
      }
      v8s_t pf;
      uint32_t* pw = reinterpret_cast<uint32_t*>(&pf);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        pw[j] = pack_dt<DT>(s[j >> 1][2 * (j & 1)], s[j >> 1][2 * (j & 1) + 1]);
#pragma unroll
      for (int dt = 0; dt < 32; ++dt) {
        const uint32_t at = ((cur + va) ^ (32 * (dt & 7))) + 256 * (dt >> 3);
        const v4s_t lo = lds_read_tr(at), hi = lds_read_tr(at + 16384);
        const v8s_t vf = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        o[dt] = mfma16<DT>(vf, pf, o[dt]);
      }
    }
  }
  if (rb >= a.nrb) return;
  if (a.nsplit == 1) {
    const float il = l == 0.f ? 0.f : 1.f / l;  // a row without a key: zeros
    if (live) {
      uint16_t* op = a.out + ((int64_t)b * rows + row) * DL;
#pragma unroll
      for (int dt = 0; dt < 32; ++dt) {
        uint2 pk;
        pk.x = pack_dt<DT>(o[dt][0] * il, o[dt][1] * il);
        pk.y = pack_dt<DT>(o[dt][2] * il, o[dt][3] * il);
        *reinterpret_cast<uint2*>(op + 16 * dt + 4 * q) = pk;
      }
    }
    return;
  }
  if (kbeg >= len && sp > 0) return;  // the join reads only the splits a length reaches
  const int64_t at = ((int64_t)sp * a.B + b) * a.nrb + rb;
  if (q == 0) {
    a.ml[(at * D_ROWS + c) * 2] = m;
    a.ml[(at * D_ROWS + c) * 2 + 1] = l;
  }
  v4f_t* pt = reinterpret_cast<v4f_t*>(a.part + at * D_PART);
#pragma unroll
  for (int dt = 0; dt < 32; ++dt) pt[dt * 64 + lane] = o[dt];
}

// Joins the splits of one row block in split order: 8 workgroups of 256 threads per block, a thread
// one float4 (4 dims of a row) of every split.
template <int DT>
__global__ void __launch_bounds__(256) k_mla_join(MlaDecArgs a) {
  const int b = blockIdx.y, rb = blockIdx.x >> 3;
  const int at4 = (blockIdx.x & 7) * 256 + threadIdx.x;  // float4 of the block: dt * 64 + lane
  const int lane = at4 & 63, c = lane & 15, q = lane >> 4, dt = at4 >> 6;
  const int row = D_ROWS * rb + c, rows = a.Sq * a.H;
  if (row >= rows) return;
  const int len = (int)min((int64_t)max(a.lens[b], 0), (int64_t)a.nb * a.ps);
  const int ns = max(1, (len + a.chunk - 1) / a.chunk);
  const int64_t step = (int64_t)a.B * a.nrb, at = (int64_t)b * a.nrb + rb;
  float m = -INFINITY;
  for (int s = 0; s < ns; ++s) m = fmaxf(m, a.ml[((s * step + at) * D_ROWS + c) * 2]);
  float l = 0.f;
  v4f_t acc = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < ns; ++s) {
    const int64_t i = s * step + at;
    const float ms = a.ml[(i * D_ROWS + c) * 2];
    // a NaN partial (fmaxf passes it by) must reach the result
    const float f = ms == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ms - m);
    l += f * a.ml[(i * D_ROWS + c) * 2 + 1];
    acc += f * reinterpret_cast<const v4f_t*>(a.part + i * D_PART)[at4];
  }
  const float il = l == 0.f ? 0.f : 1.f / l;
  uint2 pk;
  pk.x = pack_dt<DT>(acc[0] * il, acc[1] * il);
  pk.y = pack_dt<DT>(acc[2] * il, acc[3] * il);
  *reinterpret_cast<uint2*>(a.out + ((int64_t)b * rows + row) * DL + 16 * dt + 4 * q) = pk;
}

struct DecPlan {
  int rb, nrb, nsplit, chunk;
};
// RB row blocks per workgroup (all heads of a token share its key tiles); the keys split until
// about two workgroups per CU exist, no split below 128 keys
DecPlan dec_plan(int64_t B, int64_t rows, int64_t maxlen) {
  DecPlan p;
  p.nrb = (int)((rows + D_ROWS - 1) / D_ROWS);
  p.rb = p.nrb <= 1 ? 1 : p.nrb <= 2 ? 2 : p.nrb <= 4 ? 4 : 8;
  const int64_t wgs = B * ((p.nrb + p.rb - 1) / p.rb);
  int64_t ns = (512 + wgs - 1) / wgs;
  const int64_t most = (maxlen + 127) / 128;
  if (ns > most) ns = most;
  if (ns < 1) ns = 1;
  p.chunk = (int)(((maxlen + ns - 1) / ns + DKT - 1) / DKT * DKT);
  if (p.chunk < DKT) p.chunk = DKT;
  p.nsplit = (int)((maxlen + p.chunk - 1) / p.chunk);
  if (p.nsplit < 1) p.nsplit = 1;
  return p;
}

template <int DT, int RB, int NST>
int launch_dec(const MlaDecArgs& a, hipStream_t st) {
  constexpr int lds = NST * D_STAGE + (D_TAB + 1) * 4;
  (void)hipFuncSetAttribute((const void*)k_mla_dec<DT, RB, NST>,
                            hipFuncAttributeMaxDynamicSharedMemorySize, lds);
  hipLaunchKernelGGL((k_mla_dec<DT, RB, NST>),
                     dim3((unsigned)a.nsplit, (unsigned)((a.nrb + RB - 1) / RB), (unsigned)a.B),
                     64 * RB, lds, st, a);
  if (int rc = check_launch("lcq_mla_decode")) return rc;
  if (a.nsplit > 1) {
    hipLaunchKernelGGL(k_mla_join<DT>, dim3((unsigned)a.nrb * 8, (unsigned)a.B), 256, 0, st, a);
    return check_launch("lcq_mla_decode");
  }
  return LCQ_OK;
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace lcq

using namespace lcq;

extern "C" int lcq_mla_fwd_causal(const void* q_nope, const int64_t* q_nope_strides,
                                  const void* q_rope, const int64_t* q_rope_strides,
                                  const void* k_nope, const int64_t* k_nope_strides,
                                  const void* k_rope, const int64_t* k_rope_strides,
                                  const void* v, const int64_t* v_strides, int dtype, int64_t B,
                                  int64_t H, int64_t Sq, int64_t Skv, const int32_t* q_start,
                                  const int32_t* kv_lens, float scale, void* out, void* stream) {
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
  LCQ_REQUIRE(B < (1 << 24) && H < (1 << 24) && B * H * nqt < (int64_t(1) << 31),
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
  constexpr int lds = 2 * F_STAGE;
  const dim3 grid((unsigned)(B * H * nqt));
  if (dtype == LCQ_BF16) {
    (void)hipFuncSetAttribute((const void*)k_mla_fwd<LCQ_BF16>,
                              hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    hipLaunchKernelGGL(k_mla_fwd<LCQ_BF16>, grid, 256, lds, as_stream(stream), a);
  } else {
    (void)hipFuncSetAttribute((const void*)k_mla_fwd<LCQ_F16>,
                              hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    hipLaunchKernelGGL(k_mla_fwd<LCQ_F16>, grid, 256, lds, as_stream(stream), a);
  }
  return check_launch("lcq_mla_fwd_causal");
}

extern "C" int64_t lcq_mla_decode_workspace_bytes(int64_t B, int64_t Sq, int64_t H,
                                                  int64_t max_len) {
  if (B <= 0 || Sq <= 0 || H <= 0 || max_len <= 0) return 0;
  const DecPlan p = dec_plan(B, Sq * H, max_len);
  return p.nsplit == 1 ? 0 : (int64_t)p.nsplit * B * p.nrb * (D_PART + 2 * D_ROWS) * 4;
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
  LCQ_REQUIRE(Sq * H <= (1 << 20) && B <= 65535, "too many query rows");
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
  a.nrb = p.nrb; a.chunk = p.chunk; a.nsplit = p.nsplit;
  a.part = static_cast<float*>(workspace);
  a.ml = a.part ? a.part + (int64_t)p.nsplit * B * p.nrb * D_PART : nullptr;
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
