// chunk.cu -- attention of every sequence's new tokens over the paged KV cache
// (bf16 or 8-bit pages, see kv8.cu for the format): causal inside the chunk,
// optional sliding window, GQA, learned sinks.
//
//   s_ij = (q_i . k_j) * sm_scale,   j visible to token i of the chunk iff
//          0 <= j <= pos_i and, with a window W, j > pos_i - W;
//   o_i  = sum_j 2^(s2_ij - m_i) v_j / (l_i + 2^(sink2 - m_i)),
//   l_i  = sum_j 2^(s2_ij - m_i),  lse_i = m_i + log2(l_i),  s2 = s * log2(e);
//   a token that sees nothing gets o = 0 and lse = -inf.
//
// chunk_keys_kernel   up to 48 rows (tokens x heads of a kv head) against a
//                     line of keys: S^T = K Q^T and O^T = V^T P^T on tcgen05
//                     with the keys on the 128-row side
// chunk_rows_kernel   longer chunks: 256 rows against the keys, S = Q K^T and
//                     O = P V with the rows on the 128-row side
//
// The output is rounded once, from fp32; P is rounded to bf16 as the operand
// of P V (its relative error of 2^-9 an element is the size of the output's
// own rounding; chunk_keys_kernel over 8-bit pages splits it into two e4m3
// terms, 2^-8 of itself, in units that follow each row's largest of a key tile,
// see there), the sum l takes the unrounded values.
#include "chunk.cuh"
#include "launch.h"

namespace gptoss {

namespace {

constexpr float kChLog2e = 1.4426950408889634f;

__device__ __forceinline__ uint32_t ch_bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float ch_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// lo -> byte 0, hi -> byte 1; saturates, NaN stays NaN
__device__ __forceinline__ uint32_t ch_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// Two 16-bit floats as e4m3 bytes (nearest, ties to even; saturates) and back (exact).
__device__ __forceinline__ uint32_t ch_e4m3x2_f16(uint32_t f16x2) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f16x2 %0, %1;" : "=h"(r) : "r"(f16x2));
  return r;
}
__device__ __forceinline__ uint32_t ch_f16x2_e4m3(uint32_t e4m3x2) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)e4m3x2));
  return r;
}
__device__ __forceinline__ uint32_t ch_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// a * b + c and a * b of two 16-bit floats
__device__ __forceinline__ uint32_t ch_hfma2(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
  return r;
}
__device__ __forceinline__ uint32_t ch_hmul2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
// x rounded to 4 significant bits (half away from zero), exact in e4m3 for 2^-6 <= |x| <= 448
__device__ __forceinline__ float ch_round4(float x) {
  return __uint_as_float((__float_as_uint(x) + 0x80000u) & 0xFFF00000u);
}
// Four e4m3 bytes as two bf16 pairs (b0, b1), (b2, b3) times `mul`, exactly: a
// byte below eight copies of its sign, moved up by four bits, is a bf16 that
// reads 2^-120 of the value.  ch_code_mul is 2^(e + 120) for the code 127 + e,
// NaN for that of a row that held one; beyond e = 7, which bf16 does not hold,
// it is 2^127 and ch_code_rest the factor that is left.
__device__ __forceinline__ void ch_e4m3_to_bf16(uint32_t w, uint32_t mul, uint32_t& p01, uint32_t& p23) {
  p01 = bf16x2_mul((prmt(w, 0u, 0x9180u) << 4) & 0x87F087F0u, mul);
  p23 = bf16x2_mul((prmt(w, 0u, 0xB3A2u) << 4) & 0x87F087F0u, mul);
}
constexpr uint32_t kCodeOne = 134;  // the largest code that takes one factor
__device__ __forceinline__ uint32_t ch_code_mul(uint32_t code) {
  const uint32_t h = code == 255u ? 0x7FC0u : ((min(code, kCodeOne) + 120u) << 7);
  return h | (h << 16);
}
__device__ __forceinline__ uint32_t ch_code_rest(uint32_t code) {
  const uint32_t h = (min(code, 194u) - kCodeOne + 127u) << 7;
  return h | (h << 16);
}
// Two fp32 at a time.
typedef unsigned long long ch_f2;
__device__ __forceinline__ ch_f2 ch_pair(float a, float b) {
  return ((ch_f2)__float_as_uint(b) << 32) | __float_as_uint(a);
}
__device__ __forceinline__ float ch_lo(ch_f2 v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float ch_hi(ch_f2 v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ ch_f2 ch_fma2(ch_f2 a, ch_f2 b, ch_f2 c) {
  ch_f2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ ch_f2 ch_add2(ch_f2 a, ch_f2 b) {
  ch_f2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ ch_f2 ch_mul2(ch_f2 a, ch_f2 b) {
  ch_f2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// Largest of the warp's values (a NaN counts as the smallest).
__device__ __forceinline__ float ch_warp_max(float v) {
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}
__device__ __forceinline__ void ch_named_sync(int id, int n) {
  asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory");
}
__device__ __forceinline__ bool ch_named_or(int id, int n, bool v) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %1, 0;\n\t"
      "bar.red.or.pred q, %2, %3, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"((uint32_t)v), "r"(id), "r"(n)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void ch_tma_4d(void* dst, const void* tmap, int32_t z, int32_t w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %3, %4}], "
      "[%5];" ::"r"(smem_u32(dst)),
      "l"(tmap), "r"(0), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
// D[tmem] (+)= A[smem] B[smem]: bf16, or e4m3 (kind::f8f6f4).
template <bool F8>
__device__ __forceinline__ void ch_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (!F8) {
    tc_mma_ss(d, a, b, idesc, accumulate);
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}
// Shared-memory matrix descriptor: 8-row groups `group` bytes apart; rows of
// 128 bytes with the 128-byte swizzle, or of 64 with the 64-byte one.
__device__ __forceinline__ uint64_t ch_sdesc(uint32_t addr, uint32_t group, bool sw64) {
  return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(group >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)(sw64 ? 4 : 2) << 61);
}
// 8 or 16 consecutive 32-bit columns of this warp's 32 lanes, no wait.
__device__ __forceinline__ void ch_ld8(uint32_t taddr, uint32_t* r) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void ch_st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}

// One row's value from its sum, maximum and unnormalised output.
__device__ __forceinline__ float ch_norm(const ChunkParams& p, int h, float l, float m) {
  float den = l;
  if (p.sinks) den += exp2f(bf16_bits_to_f32(p.sinks[h]) * kChLog2e - m);
  return l == 0.f ? 0.f : 1.0f / den;
}

// The partial results of a unit, joined in the order of the keys: 16 threads
// per row, 4 dims each, four parts' loads in flight.  `heads` kv heads of
// `rows` rows each per slot.
__device__ __forceinline__ void chunk_join(const ChunkParams& p, const ChunkSeg& sg, int heads, int rows, int tid,
                                           int nthreads) {
  const int c0 = sg.c0, c1 = sg.c1, s0 = 2 * sg.c0 + 1;
  const int64_t rs = (int64_t)heads * rows;
  for (int x = tid; x < heads * sg.nrows * 16; x += nthreads) {
    const int hr = x >> 4, d = (x & 15) * 4;
    const int hb = hr / sg.nrows, r = hr - hb * sg.nrows;
    const int64_t at = (int64_t)hb * rows + r;
    float m = -INFINITY, l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int c = c0; c <= c1; c += 4) {
      float2 ml[4];
      float4 y[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int cc = min(c + k, c1);
        const int64_t row = (cc == c0 ? s0 : 2 * cc) * rs + at;
        ml[k] = __ldcg((const float2*)(p.part_ml + row * 2));
        y[k] = __ldcg((const float4*)(p.part_o + row * kChunkD + d));
      }
      float mn = m;
#pragma unroll
      for (int k = 0; k < 4; ++k) mn = fmaxf(mn, ml[k].x);
      const float me = mn == -INFINITY ? 0.f : mn, f0 = exp2f(m - me);
      l *= f0;
      a.x *= f0;
      a.y *= f0;
      a.z *= f0;
      a.w *= f0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float f = c + k <= c1 ? exp2f(ml[k].x - me) : 0.f;
        if (c + k > c1) break;
        l += ml[k].y * f;
        a.x += y[k].x * f;
        a.y += y[k].y * f;
        a.z += y[k].z * f;
        a.w += y[k].w * f;
      }
      m = mn;
    }
    const int tk = r / p.G, h = (sg.hg * heads + hb) * p.G + r - tk * p.G;
    const int64_t tok = sg.tok0 + tk;
    if (p.lse && d == 0) p.lse[tok * p.Hq + h] = m + log2f(l);
    const float inv = ch_norm(p, h, l, m);
    *(uint2*)(p.o + (tok * p.Hq + h) * kChunkD + d) =
        make_uint2(ch_bf16x2(a.x * inv, a.y * inv), ch_bf16x2(a.z * inv, a.w * inv));
  }
}

// ---------------------------------------------------------- keys on M --
// CTA = two streams of softmax warps (a kv head each), a warp each that loads K
// and V, and one per stream that issues the products.  A tile is 128 keys of
// both heads (up to 16 rows in 8 bits: 256; the chain from one tile's products
// to the next takes about 2000 cycles whatever it holds).  From 32 rows on a
// stream has 8 warps, two for the same keys with half of the rows each: a
// thread's rows are unrolled, and past about 700 instructions a tile the
// instruction cache, not the issue, sets the pace.  One TMA box brings a page's
// keys of both, in groups of 8 rows of 128 bytes (bf16: a head's, 8-bit: both
// heads' side by side), so that a head's 128 keys are one matrix operand with an
// even stride.  Two warps load: the copy engine takes 2 KB in about 97 cycles
// from two issuers, 135 from one.  Per tile and stream, N rows:
//   S^T [128 keys x N] = K Q^T    A = the K tile as it lies, B = Q
//   a thread owns a key: its N scores (or N / 2) are registers, the key's mask,
//     scale and V exponent are its own constants
//   O^T [64 dims x W] += V^T P^T  A = the V tile read dims-major, B = P^T,
//     which the threads wrote to shared memory row by key; W = N, 8-bit 2 N
// With the keys on the 128-row side nothing is padded to 128 queries: 8 rows
// (one token's group of heads) cost N = 16 columns.  (An mma.sync form of this
// kernel, rows on M, ran 32 x 5 tokens over 8191 8-bit keys in 317 us: legacy
// mma.sync reaches 1009 multiply-adds per cycle and SM here, a quarter of
// tcgen05's, and each 8-bit value had to be widened.)
//
// 8-bit pages are operands as they are (kind::f8f6f4).  The other side is then
// e4m3 too, as two terms.  Q is scaled by a power of two per unit and head; hi =
// Q to 4 significant bits and lo = the rest are two products into the same
// columns (2^-18 of the largest).  P's terms have columns of their own, W = 2 N:
// hi = P in e4m3, lo = 28 times what that leaves, 2^-8 of P in all.  The key's
// power of two meets the score in fp32; the value's goes into the exponent, t = s
// + e_v, and the softmax reference follows t:  P = 2^(t - m), l = sum P 2^-e_v.
//
// The reference m of a row moves up when a score exceeds it by 8 (8 bit: 8.75, P
// up to 430), which one barrier of the stream's warps tells; then O^T in TMEM is
// rescaled.  In 8 bits it moves down, too, when no P of the row reaches 1 in a
// tile: the two terms end at 2^-14.8, and thousands of keys that each fall below it
// may weigh as much as the largest.  Each second tile is looked at, which bounds
// what is lost: 2^-18 a key of the row's largest so far, which is 2^3.5 or more in
// units of 2^m; and by the 128 or 256 keys of a tile together 2^-6.8 at most of the
// tile before, whose largest P is 1 or more.  kDepth bounds the way down from the
// row's highest reference, since O^T and l are multiplied on the way: keys that
// far below it weigh nothing beside the one that set it.  (32 sequences of 1 to 5
// tokens on up to 8191 keys: 109 us without the way down, 114 with it, 120 where
// every tile is looked at; units that begin at 2^3: 117, at 2^5: 120.)
//
// Measured, 32 sequences of 8192 keys, 8 kv heads: one token 90 us in bf16 (6.0
// TB/s, the bytes bound it), 71 us in 8 bits (3.9 TB/s: a tile's chain of barrier
// waits, products and softmax, not the bytes, bounds it); five tokens 118 and 144
// us (the softmax: 5 times the exponentials and, in 8 bits, P as two terms).
template <bool F8, int N_>
struct KeysCfg {
  static constexpr int N = N_;                             // rows of a unit
  static constexpr int W = F8 ? 2 * N : N;                 // columns of O^T
  static constexpr bool kSplit = N >= 32;                  // two warps share 32 keys, half of the rows each
  static constexpr int KT = F8 && !kSplit ? 256 : 128;     // keys of a tile
  static constexpr int kWps = kSplit ? 8 : KT / 32;        // softmax warps of a stream
  static constexpr int NR = kSplit ? N / 2 : N;            // rows of a thread
  static constexpr int kSums = KT / 32;                    // warps that hold a part of a row's sum
  static constexpr int kThreads = 2 * kWps * 32 + 128;
  static constexpr int kRowBytes = F8 ? 64 : 128;
  static constexpr int kSide = 2 * KT * kRowBytes;         // K or V of a tile, two heads
  static constexpr int kCodes = F8 ? 2 * 2 * KT : 0;       // [K, V][head][KT]
  static constexpr int kStages = F8 && kSplit ? 4 : 2;
  static constexpr int kQ = N * 128;                       // per stream: N rows of 128 bytes, or 2 N of 64
  static constexpr int kP = KT * 128;                      // per stream
  static constexpr int kColO = 2 * (KT / 128) * N;         // S^T: N columns per stream and 128 keys, then O^T
  static constexpr int kCols = kColO + 2 * W;
  static constexpr int kTmem = kCols <= 64 ? 64 : kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
  static constexpr int kOffP = kStages * 2 * kSide;
  static constexpr int kOffQ = kOffP + 2 * kP;
  static constexpr int kOffCodes = kOffQ + 2 * kQ;
  static constexpr int kOffRed = kOffCodes + kStages * kCodes;  // per stream: [kSums][N] maxima or sums
  static constexpr int kOffRef = kOffRed + 2 * kSums * N * 4;   // per stream: -m, factor, 8 bit: -(highest m); [N] each
  static constexpr int kOffLow = kOffRef + 2 * 3 * N * 4;       // 8 bit, per stream: each warp's rows below 1
  static constexpr int kOffPre = kOffLow + 2 * 8 * 4;
  static constexpr int kOffSeg = kOffPre + (kChunkMaxSeqs + 1 + 15) / 16 * 64;
  static constexpr int kOffBar = kOffSeg + 2 * (int)sizeof(ChunkSeg);
  static constexpr int kAlloc = kOffBar + (4 * kStages + 4 + 10) * 8 + 32 + 1024;
  static_assert(kAlloc <= 227 * 1024 && kCols <= 512, "shared memory, TMEM");
};

template <bool F8, int N_>
__global__ void __launch_bounds__(KeysCfg<F8, N_>::kThreads, 1)
    chunk_keys_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                      const ChunkParams p, const int HB) {
  using C = KeysCfg<F8, N_>;
  constexpr int N = C::N, W = C::W, RB = C::kRowBytes, NS = C::kStages, KT = C::KT, kWps = C::kWps, NR = C::NR,
                kSums = C::kSums, kParts = kWps / 4;
  constexpr int kLoadK = 2 * kWps, kLoadV = kLoadK + 2, kMma0 = kLoadK + 1, kMma1 = kLoadK + 3;  // warps
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  int32_t* pre = (int32_t*)(smem + C::kOffPre);
  ChunkSeg* segs = (ChunkSeg*)(smem + C::kOffSeg);
  uint64_t* kfull = (uint64_t*)(smem + C::kOffBar);
  uint64_t* kempty = kfull + NS;
  uint64_t* vfull = kempty + NS;  // V and the codes
  uint64_t* vempty = vfull + NS;
  uint64_t* seg_full = vempty + NS;
  uint64_t* seg_empty = seg_full + 2;
  uint64_t* qfull = seg_empty + 2;  // per stream from here on
  uint64_t* sfull = qfull + 2;
  uint64_t* sfree = sfull + 2;
  uint64_t* pfull = sfree + 2;
  uint64_t* ofull = pfull + 2;
  volatile uint32_t* flag = (volatile uint32_t*)(ofull + 2);
  volatile uint32_t* tmem_slot = flag + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&kfull[s], 1);
      mbar_init(&kempty[s], HB);
      mbar_init(&vfull[s], F8 ? 33 : 1);  // 8 bit: the loading warp's lanes arrive with their copies of the codes
      mbar_init(&vempty[s], HB);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&seg_full[s], 1);
      mbar_init(&seg_empty[s], 2 * kWps + 1 + HB);
      mbar_init(&qfull[s], kWps);
      mbar_init(&sfull[s], 1);
      mbar_init(&sfree[s], kWps);
      mbar_init(&pfull[s], kWps);
      mbar_init(&ofull[s], 1);
    }
    fence_mbar_init();
  }
  if (warp == kMma0) {
    tmem_alloc((uint32_t*)tmem_slot, C::kTmem);
    tmem_relinquish();
  }
  tc_fence_before();
  chunk_plan(p, pre, C::kThreads);  // with a __syncthreads at its end
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  int it = 0;  // key tiles so far
  bool bad = false;

  // 640 threads start with 96 registers each: 512 * 104 + 128 * 64 of them from here on
  if (kWps == 8 && warp >= kLoadK) asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
  if (warp == kLoadK || warp == kLoadV) {
    // ------------------------------------------------------------- loads
    const bool is_v = warp == kLoadV;  // V and the codes; the other: K, and the parts' descriptions
    ChunkWalk walk;
    if (!is_v) walk.begin(p, pre, gridDim.x, blockIdx.x);
    const uint32_t box = (uint32_t)(HB * kChunkPage * RB);
    const CUtensorMap* tmap = is_v ? &tmap_v : &tmap_k;
    uint64_t* full = is_v ? vfull : kfull;
    uint64_t* empty = is_v ? vempty : kempty;
    for (int sn = 0;; ++sn) {
      const int sb = sn & 1;
      if (!is_v) {
        ChunkSeg sg;
        const bool more = walk.next(p, sg);
        if (!bad) bad = !mbar_wait(&seg_empty[sb], ((uint32_t)(sn >> 1) & 1u) ^ 1u, p.err, kErrTimeoutEmpty);
        if (lane == 0) {
          if (!more) sg.nrows = -1;
          segs[sb] = sg;
          mbar_arrive(&seg_full[sb]);
        }
        __syncwarp();
        if (!more || bad) break;
      } else {
        if (!bad) bad = !mbar_wait(&seg_full[sb], (uint32_t)(sn >> 1) & 1u, p.err, kErrTimeoutFull);
        if (bad || segs[sb].nrows < 0) break;
      }
      const int32_t ntile = segs[sb].ntile, j0 = segs[sb].j0, lo = segs[sb].lo, hi = segs[sb].hi;
      const int32_t head = segs[sb].hg * HB;
      const int32_t* trow = p.table + (int64_t)segs[sb].row * p.tstride;
      for (int i = 0; i < ntile; ++i, ++it) {
        const int st = it % NS;
        // the pages of this tile that hold a key to look at, one a lane (8 or 16)
        constexpr int kPages = KT / kChunkPage;
        const int32_t j = j0 + i * KT + (lane & (kPages - 1)) * kChunkPage;
        const bool on = j < hi && j + kChunkPage > lo;
        int32_t page = -1;
        if (on) page = __ldg(trow + (uint32_t)(j / kChunkPage) % (uint32_t)p.tstride);
        if (page >= p.pool_pages) page = -1;  // a page outside the pool is not read
        const uint32_t bytes = (uint32_t)__popc(__ballot_sync(0xffffffffu, page >= 0 && lane < kPages)) * box;
        if (!bad) bad = !mbar_wait(&empty[st], ((uint32_t)(it / NS) & 1u) ^ 1u, p.err, kErrTimeoutEmpty);
        if (lane == 0) mbar_arrive_expect_tx(&full[st], bytes);
        __syncwarp();
        if (page >= 0 && lane < kPages)
          ch_tma_4d(smem + st * 2 * C::kSide + (is_v ? C::kSide : 0) + lane * box, tmap, F8 && HB == 2 ? head / 2 : head,
                    page * 2, &full[st]);
        if (F8 && is_v) {
          // 16 bytes of codes per page and head, [K, V][head][page]: lane = [head][page], K's and V's
          const int hb = lane / kPages;
          if (page >= 0 && hb < HB) {
            const int64_t src = ((int64_t)page * p.Hkv + head + hb) * kChunkPage;
            uint8_t* dst = smem + C::kOffCodes + st * C::kCodes + lane * kChunkPage;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(p.k_code + src) : "memory");
            asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst + 2 * KT)), "l"(p.v_code + src)
                         : "memory");
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&full[st])) : "memory");
        }
        __syncwarp();
      }
      if (is_v) {
        if (lane == 0) mbar_arrive(&seg_empty[sb]);
        __syncwarp();
      }
    }
  } else if (warp == kMma0 || warp == kMma1) {
    // ---------------------------------------------------------- products
    // one thread per stream: S^T, A = K (K-major, 128 keys), B = Q (K-major, N rows; 8 bit: its two terms one after
    // the other); O^T, A = V^T (dims-major), B = P^T (rows-major)
    const int s = warp == kMma1;
    if (s < HB && elect_one()) {
      const uint32_t fmt = F8 ? (1u << 4) : ((1u << 4) | (1u << 7) | (1u << 10));
      const uint32_t idesc_s = fmt | ((uint32_t)(N >> 3) << 17) | (8u << 24);
      const uint32_t idesc_o = fmt | (1u << 15) | (1u << 16) | ((uint32_t)(W >> 3) << 17) | (4u << 24);
      // bytes between groups of 8 keys, and from one head to the next
      const uint32_t group = (uint32_t)(HB * 8 * RB), to_head = F8 ? 64u : 1024u;
      const bool sw64 = F8 && HB == 1;
      const uint64_t dk = ch_sdesc(smem_u32(smem) + s * to_head, group, sw64);
      const uint64_t dv = ch_sdesc(smem_u32(smem + C::kSide) + s * to_head, group, sw64);
      const uint64_t dq = ch_sdesc(smem_u32(smem + C::kOffQ + s * C::kQ), 8 * RB, F8);
      const uint64_t dp = ch_sdesc(smem_u32(smem + C::kOffP + s * C::kP), 1024, false);
      constexpr int kStep = F8 ? 32 : 16;  // keys of one product of O^T
      const uint32_t v_step = (kStep / 8) * (group >> 4);
      int ks = 0, vs = 0;               // stages of the next S^T and the next O^T
      uint32_t kp = 0, vp = 0, tp = 0;  // their parities, and that of S^T's tile
      uint32_t op = 0;                  // parity of O^T's tile
      auto issue_s = [&]() {
        if (!bad) bad = !mbar_wait(&kfull[ks], kp, p.err, kErrTimeoutFull);
        if (!bad) bad = !mbar_wait(&sfree[s], tp ^ 1u, p.err, kErrTimeoutAccum);  // the tile before has been read
        tc_fence_after();
        const uint64_t a = dk + (uint32_t)ks * (2 * C::kSide >> 4);
#pragma unroll
        for (int h = 0; h < KT / 128; ++h)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            ch_mma_ss<F8>(tmem + (s * (KT / 128) + h) * N, a + h * 16 * (group >> 4) + 2 * (F8 ? kk & 1 : kk),
                          dq + (F8 ? (kk >> 1) * (N * 64 >> 4) + 2 * (kk & 1) : 2 * kk), idesc_s, kk > 0 ? 1u : 0u);
        tc_commit(&sfull[s]);
        tc_commit(&kempty[ks]);
        tp ^= 1u;
        if (++ks == NS) {
          ks = 0;
          kp ^= 1u;
        }
      };
      for (int sn = 0; !bad; ++sn) {
        const int sb = sn & 1;
        bad = !mbar_wait(&seg_full[sb], (uint32_t)(sn >> 1) & 1u, p.err, kErrTimeoutFull);
        if (bad || segs[sb].nrows < 0) break;
        const int nt = segs[sb].ntile;
        bad = !mbar_wait(&qfull[s], (uint32_t)sn & 1u, p.err, kErrTimeoutFull);
        if (nt > 0) issue_s();
        for (int i = 0; i < nt; ++i) {
          if (i + 1 < nt) issue_s();
          if (!bad) bad = !mbar_wait(&vfull[vs], vp, p.err, kErrTimeoutFull);
          if (!bad) bad = !mbar_wait(&pfull[s], op, p.err, kErrTimeoutAccum);
          tc_fence_after();
          const uint64_t a = dv + (uint32_t)vs * (2 * C::kSide >> 4);
#pragma unroll
          for (int kk = 0; kk < KT / kStep; ++kk)
            ch_mma_ss<F8>(tmem + C::kColO + s * W, a + kk * v_step, dp + kk * (kStep / 8) * 64, idesc_o,
                          (i > 0 || kk > 0) ? 1u : 0u);
          tc_commit(&ofull[s]);
          tc_commit(&vempty[vs]);
          op ^= 1u;
          if (++vs == NS) {
            vs = 0;
            vp ^= 1u;
          }
        }
        mbar_arrive(&seg_empty[sb]);
      }
    }
    __syncwarp();
  } else {
    // ----------------------------------------------------------- softmax
    if (kWps == 8) asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    constexpr int kBar = kWps * 32;  // threads of a stream
    // tid: thread of the stream; tid % KT: its key of the tile; part: which half of the rows (kSplit) or keys
    const int s = warp / kWps, wq = warp % kWps, tid = threadIdx.x % kBar, key = tid % KT, part = wq >> 2;
    const int rb = C::kSplit ? part * NR : 0;          // its first row
    const int sum_at = C::kSplit ? wq & 3 : wq;        // its warp's place in `red`
    const bool mine = s < HB;
    const uint32_t tl = tmem + ((uint32_t)((wq & 3) * 32) << 16);
    const uint32_t t_s = tl + (C::kSplit ? s * N + rb : (s * (KT / 128) + part) * N), t_o = tl + C::kColO + s * W;
    float* red = (float*)(smem + C::kOffRed) + s * kSums * N;
    float* nref = (float*)(smem + C::kOffRef) + s * 3 * N;  // -m of a row
    float* fac = nref + N;
    float* ntop = fac + N;  // 8 bit: -m where m was highest
    uint32_t* low = (uint32_t*)(smem + C::kOffLow) + s * 8;
    uint8_t* qs = smem + C::kOffQ + s * C::kQ;
    uint8_t* ps = smem + C::kOffP + s * C::kP;
    constexpr float kUp = F8 ? 8.75f : 8.0f;   // P at most 2^kUp (8 bit: 28 times what e4m3 leaves of 448 is 448)
    constexpr float kBase = F8 ? 3.5f : 0.0f;  // log2 P of the largest when the reference moves
    constexpr float kDepth = 32.0f;            // (a V row of zeros counts up to 2^60 in l: 2^26 of them fit fp32 yet)
    constexpr float kNoRef = 3.402823466e38f;
    for (int sn = 0;; ++sn) {
      const int sb = sn & 1;
      if (!bad) bad = !mbar_wait(&seg_full[sb], (uint32_t)(sn >> 1) & 1u, p.err, kErrTimeoutFull);
      bad = ch_named_or(6, 2 * kBar, bad);  // all softmax warps leave together
      const ChunkSeg& sg = segs[sb];
      const int nrows = sg.nrows;
      if (nrows < 0 || bad) break;
      const int ntile = sg.ntile;
      const int32_t lo = sg.lo, hi = sg.hi, first_pos = sg.first_pos;
      const int head0 = (sg.hg * HB + s) * p.G;
      float q_unit = 1.0f;
      const int mine_rows = max(0, min(NR, nrows - rb));  // this thread's rows in use
      ch_f2 l[NR / 2];
#pragma unroll
      for (int r = 0; r < NR / 2; ++r) l[r] = 0ull;
      if (mine && ntile > 0) {
        // Q into shared memory: 8 threads per row
        constexpr int kQRows = kBar / 8, kQIter = (N + kQRows - 1) / kQRows;
        uint4 x[kQIter];
        uint32_t am = 0;
#pragma unroll
        for (int k = 0; k < kQIter; ++k) {
          const int r = k * kQRows + (tid >> 3);
          x[k] = make_uint4(0, 0, 0, 0);
          if (r < nrows) {
            const int tk = r / p.G;
            x[k] = *(const uint4*)(p.q + (sg.tok0 + tk) * p.q_stride + (int64_t)(head0 + r - tk * p.G) * kChunkD +
                                   (tid & 7) * 8);
          }
          const uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t a = (w[e] << 16) & 0x7FFFFFFFu, b = w[e] & 0x7FFF0000u;
            am = max(am, max(a >= 0x7F800000u ? 0u : a, b >= 0x7F800000u ? 0u : b));
          }
        }
        float up = 1.0f;
        if (F8) {
          // largest magnitude of the unit's finite values into [128, 256)
          am = __reduce_max_sync(0xffffffffu, am);
          if (lane == 0) fac[wq] = __uint_as_float(am);
          ch_named_sync(1 + s, kBar);
#pragma unroll
          for (int w = 0; w < kWps; ++w) am = max(am, __float_as_uint(fac[w]));
          const int ex = max((int)(am >> 23), 14);
          up = __uint_as_float((uint32_t)min(261 - ex, 254) << 23);
          q_unit = 1.0f / up;
        }
#pragma unroll
        for (int k = 0; k < kQIter; ++k) {
          const int r = k * kQRows + (tid >> 3), c = tid & 7;
          if (r >= N) continue;
          if (!F8) {
            *(uint4*)(qs + r * 128 + ((c ^ (r & 7)) << 4)) = x[k];
          } else {
            const uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
            uint32_t h4[2], l4[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float v[4] = {__uint_as_float(w[2 * e] << 16) * up, __uint_as_float(w[2 * e] & 0xFFFF0000u) * up,
                                  __uint_as_float(w[2 * e + 1] << 16) * up,
                                  __uint_as_float(w[2 * e + 1] & 0xFFFF0000u) * up};
              float hh[4];
#pragma unroll
              // what is not finite makes the row NaN
              for (int y = 0; y < 4; ++y) hh[y] = fabsf(v[y]) < 1e30f ? ch_round4(v[y]) : __uint_as_float(0x7FC00000u);
              h4[e] = ch_e4m3x2(hh[0], hh[1]) | (ch_e4m3x2(hh[2], hh[3]) << 16);
              l4[e] = ch_e4m3x2(v[0] - hh[0], v[1] - hh[1]) | (ch_e4m3x2(v[2] - hh[2], v[3] - hh[3]) << 16);
            }
            // rows of 64 bytes; the second term N rows further (a whole number of groups of 8)
            const int at = r * 64 + (((c >> 1) ^ ((r >> 1) & 3)) << 4) + (c & 1) * 8;
            *(uint2*)(qs + at) = make_uint2(h4[0], h4[1]);
            *(uint2*)(qs + N * 64 + at) = make_uint2(l4[0], l4[1]);
          }
        }
        if (tid < N) {
          // no reference yet: one below every finite score (a score of -infinity, which has to weigh nothing, is NaN
          // beside an infinite one); unused rows: P = 0
          nref[tid] = tid < nrows ? kNoRef : -INFINITY;
          ntop[tid] = kNoRef;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        ch_named_sync(1 + s, kBar);
        if (lane == 0) mbar_arrive(&qfull[s]);
      } else if (!mine || ntile == 0) {
        // an idle stream keeps the barriers' count of segments
        if (lane == 0) mbar_arrive(&qfull[s]);
      }
      for (int i = 0; i < ntile; ++i, ++it) {
        const int st = it % NS;
        if (!mine) continue;
        const int32_t j = sg.j0 + i * KT + key;
        // of this thread's rows, [r_lo, r_hi) see its key
        int r_lo = 0, r_hi = mine_rows;
        const int32_t jt = sg.j0 + i * KT;
        const bool whole = jt + KT - 1 <= first_pos && jt >= lo &&
                           (p.window <= 0 || jt > first_pos + sg.ntok - 1 - p.window);
        if (!whole) {
          r_lo = max(0, min(j - first_pos, 1 << 16)) * p.G - rb;
          if (p.window > 0) r_hi = min(r_hi, max(0, min(j + p.window - first_pos, 1 << 16)) * p.G - rb);
        }
        float kf = p.scale2, ev = 0.f, einv = 1.f;
        bool v_nan = false;
        if (F8 || !whole) {
          if (!bad) bad = !mbar_wait(&vfull[st], (uint32_t)(it / NS) & 1u, p.err, kErrTimeoutFull);
        }
        if (F8) {
          const uint8_t* cc = smem + C::kOffCodes + st * C::kCodes + s * KT + key;
          const uint32_t kc = cc[0], vc = cc[2 * KT];
          const float nan = __uint_as_float(0x7FC00000u);
          kf = kc == 255u ? nan : p.scale2 * q_unit * __uint_as_float(kc << 23);
          v_nan = vc == 255u;
          ev = v_nan ? 0.f : (float)((int)vc - 127);
          einv = v_nan ? 1.f : __uint_as_float((254u - min(vc, 253u)) << 23);
        }
        // Rows that do not see a key have P = 0 there, and 0 times its V row must be 0: where some row does not, the V
        // rows of keys nobody sees (whatever their page, or an earlier tile, holds) and those that are not finite
        // become zeros, and the latter's P NaN for the rows that do see them.
        // (Swizzled within the row, but for two heads in one row: 16-byte piece c of head s is 4 s + c.)
        uint8_t* vr = smem + st * 2 * C::kSide + C::kSide +
                      (F8 ? key * (HB * RB) : ((key >> 3) * HB + s) * 8 * RB + (key & 7) * RB);
        auto v_piece = [&](int c) { return (uint4*)(vr + (F8 && HB == 2 ? (4 * s + c) ^ (key & 7) : c) * 16); };
        bool v_zero = false;
        if (!whole) {
          if (j < lo || j >= hi) {
            v_zero = true;
          } else {
            uint32_t most = 0;
#pragma unroll 1
            for (int c = 0; c < RB / 16; ++c) {
              const uint4 y = *v_piece(c);
              const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
              for (int e = 0; e < 4; ++e)
                most = F8 ? most | (((w[e] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u)
                          : max(most, max((w[e] << 16) & 0x7FFFFFFFu, w[e] & 0x7FFF0000u));
            }
            if (F8 ? most != 0u : most >= 0x7F800000u) v_nan = true;
            v_zero = v_nan;
          }
        }
        if (!bad) bad = !mbar_wait(&sfull[s], (uint32_t)it & 1u, p.err, kErrTimeoutAccum);
        tc_fence_after();
        ch_f2 x[NR / 2];
        const ch_f2 kf2 = ch_pair(kf, kf), ev2 = ch_pair(ev, ev);
        // t - m (nm: -m of the rows) of this thread's rows r0 .. + 7 from TMEM; -inf where the key is hidden from one
        auto scores = [&](int r0, ch_f2 (&t)[4], const ch_f2 (&nm)[4]) {
          uint32_t a[8];
          ch_ld8(t_s + r0, a);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const ch_f2 v = ((ch_f2)a[2 * e + 1] << 32) | a[2 * e];
            t[e] = F8 ? ch_add2(ch_fma2(v, kf2, ev2), nm[e]) : ch_fma2(v, kf2, nm[e]);
          }
          if (!whole) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = r0 + 2 * e;
              t[e] = ch_pair(r < r_lo || r >= r_hi ? -INFINITY : ch_lo(t[e]),
                             r + 1 < r_lo || r + 1 >= r_hi ? -INFINITY : ch_hi(t[e]));
            }
          }
        };
        auto refs = [&](int r0, ch_f2 (&nm)[4]) {
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const ulonglong2 y = *(const ulonglong2*)(nref + rb + r0 + 2 * e);
            nm[e] = y.x;
            nm[e + 1] = y.y;
          }
        };
        for (int again = 0;; ++again) {
          float mx = -INFINITY;
#pragma unroll
          for (int r0 = 0; r0 < NR; r0 += 8) {
            if (r0 < mine_rows) {
              ch_f2 t[4], nm[4];
              refs(r0, nm);
              scores(r0, t, nm);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                x[r0 / 2 + e] = t[e];
                mx = fmaxf(mx, fmaxf(ch_lo(t[e]), ch_hi(t[e])));
              }
            }
          }
          const bool check = F8 && (i & 1) && !again;
          if (check) {
            // a bit per row, 1: its t is below m (row mine_rows - 1 in bit 0)
            uint32_t neg = 0;
#pragma unroll
            for (int r0 = 0; r0 < NR; r0 += 8) {
              if (r0 < mine_rows) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  neg = __funnelshift_l((uint32_t)x[r0 / 2 + e], neg, 1);
                  neg = __funnelshift_l((uint32_t)(x[r0 / 2 + e] >> 32), neg, 1);
                }
              }
            }
            neg = __reduce_and_sync(0xffffffffu, neg >> (-mine_rows & 7));
            if (lane == 0) low[wq] = neg;
          }
          bool move = ch_named_or(1 + s, kBar, mx > kUp);
          if (check) {  // (two votes or more lie between one tile's `low` and the next one's)
            const uint4 a = *(const uint4*)low, b = *(const uint4*)(low + 4);
            const uint32_t w0 = a.x & a.y & a.z & a.w, w1 = b.x & b.y & b.z & b.w;
            move |= (C::kSplit ? w0 | w1 : w0 & w1) != 0u;
          }
          // the second time round nothing is left above the reference's reach
          if (!move || again) break;
          const ch_f2 zero[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll 1
          for (int r0 = 0; r0 < mine_rows; r0 += 8) {
            ch_f2 t[4];
            scores(r0, t, zero);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float m0 = ch_warp_max(ch_lo(t[e])), m1 = ch_warp_max(ch_hi(t[e]));
              if (lane == 0) *(float2*)(red + sum_at * N + rb + r0 + 2 * e) = make_float2(m0, m1);
            }
          }
          ch_named_sync(3 + s, kBar);
          if (tid < nrows) {
            float m = red[tid];
#pragma unroll
            for (int w = 1; w < kSums; ++w) m = fmaxf(m, red[w * N + tid]);
            const float m0 = -nref[tid];
            float m1 = m > m0 + kUp ? m - kBase : m0;
            if (F8) {
              const float top = -ntop[tid];
              // down, unless nothing in the tile is seen (or the row has seen a score of infinity)
              if (m < m0 && m > -INFINITY && m0 < INFINITY) m1 = fminf(m0, fmaxf(m - kBase, top - kDepth));
              ntop[tid] = -fmaxf(top, m1);
            }
            fac[tid] = m1 == m0 ? 1.0f : ch_exp2(m0 - m1);
            nref[tid] = -m1;
          }
          ch_named_sync(3 + s, kBar);
#pragma unroll
          for (int r = 0; r < NR; r += 2)
            if (r < mine_rows) l[r / 2] = ch_mul2(l[r / 2], *(const ch_f2*)(fac + rb + r));
          if (i > 0) {
            // O^T of the tiles before, once their products are done
            if (!bad) bad = !mbar_wait(&ofull[s], ((uint32_t)it & 1u) ^ 1u, p.err, kErrTimeoutAccum);
            tc_fence_after();
#pragma unroll 1
            for (int c0 = part * 8; c0 < W; c0 += 8 * kParts) {
              const int r0 = F8 && c0 >= N ? c0 - N : c0;
              if (r0 >= nrows) continue;
              uint32_t o8[8];
              ch_ld8(t_o + c0, o8);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 8; ++e) o8[e] = __float_as_uint(__uint_as_float(o8[e]) * fac[r0 + e]);
              ch_st8(t_o + c0, o8);
            }
            tmem_st_wait();
          }
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sfree[s]);  // S^T is in registers
        if (v_zero && (!C::kSplit || part == 0)) {  // both halves have looked, before the vote
#pragma unroll 1
          for (int c = 0; c < RB / 16; ++c) *v_piece(c) = make_uint4(0, 0, 0, 0);
        }
        // P^T of the tile before has been used
        if (i > 0) {
          if (!bad) bad = !mbar_wait(&ofull[s], ((uint32_t)it & 1u) ^ 1u, p.err, kErrTimeoutAccum);
        }
        uint8_t* pr = ps + key * 128;
        const int sw = (key & 7) << 4;
        const ch_f2 einv2 = ch_pair(einv, einv);
#pragma unroll
        for (int r0 = 0; r0 < NR; r0 += 8) {
          if (r0 >= mine_rows) break;  // columns of rows that are not there: nobody reads their results
          uint32_t w[4], hl[4];  // bf16: 16 bytes; 8 bit: 8 of each term
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const ch_f2 v = x[r0 / 2 + e], pe = ch_pair(ch_exp2(ch_lo(v)), ch_exp2(ch_hi(v)));
            l[r0 / 2 + e] = F8 ? ch_fma2(pe, einv2, l[r0 / 2 + e]) : ch_add2(pe, l[r0 / 2 + e]);
            if (!F8) {
              w[e] = ch_bf16x2(ch_lo(pe), ch_hi(pe));
            } else {
              // hi: P in e4m3; lo: 28 times the rest, which 16 bits hold exactly (P to 2^-11 of itself and 2^-25)
              const uint32_t p16 = ch_f16x2(ch_lo(pe), ch_hi(pe));
              w[e] = ch_e4m3x2_f16(p16);
              hl[e] = ch_e4m3x2_f16(ch_hfma2(p16, 0x4F004F00u, ch_hmul2(ch_f16x2_e4m3(w[e]), 0xCF00CF00u)));
            }
          }
          const int b = (rb + r0) * (F8 ? 1 : 2);  // byte of the row's place
          if (!F8) {
            *(uint4*)(pr + (b ^ sw)) = make_uint4(w[0], w[1], w[2], w[3]);
          } else {
            *(uint2*)(pr + ((b & ~15) ^ sw) + (b & 8)) = make_uint2(w[0] | (w[1] << 16), w[2] | (w[3] << 16));
            const int b2 = N + b;
            *(uint2*)(pr + ((b2 & ~15) ^ sw) + (b2 & 8)) = make_uint2(hl[0] | (hl[1] << 16), hl[2] | (hl[3] << 16));
          }
        }
        if (v_nan) {
#pragma unroll 1
          for (int r = max(0, r_lo); r < r_hi; ++r) {
            const int b = (rb + r) * (F8 ? 1 : 2), at = ((b & ~15) ^ sw) + (b & 15);
            if (F8) pr[at] = 0x7F;
            else *(uint16_t*)(pr + at) = 0x7FC0;
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) mbar_arrive(&pfull[s]);
      }

      // ----------------------------------------------------- end of a part
      const int slot = sg.slot;
      if (mine) {
        if (ntile > 0) {
          if (!bad) bad = !mbar_wait(&ofull[s], ((uint32_t)it & 1u) ^ 1u, p.err, kErrTimeoutAccum);
          tc_fence_after();
        }
        // sums over the keys, 8 rows side by side
#pragma unroll
        for (int r0 = 0; r0 < NR; r0 += 8) {
          if (r0 < mine_rows) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = e & 1 ? ch_hi(l[(r0 + e) / 2]) : ch_lo(l[(r0 + e) / 2]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
#pragma unroll
              for (int e = 0; e < 8; ++e) v[e] += __shfl_xor_sync(0xffffffffu, v[e], o);
            if (lane == 0) {
#pragma unroll
              for (int e = 0; e < 8; e += 4)
                *(float4*)(red + sum_at * N + rb + r0 + e) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
            }
          }
        }
        // O^T from TMEM to rows of 64 floats in P's place: a lane below 16 of warp wq holds dim 16 (wq mod 4) + lane
        float* os = (float*)ps;
        if (ntile > 0) {
#pragma unroll
          for (int r0 = 0; r0 < N; r0 += 8) {
            if (r0 < nrows && (kParts == 1 || (r0 >> 3 & 1) == part)) {
              uint32_t a[8], b[8];
              ch_ld8(t_o + r0, a);
              if (F8) ch_ld8(t_o + N + r0, b);
              tmem_ld_wait();
              if (lane < 16) {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                  os[(r0 + e) * 64 + (wq & 3) * 16 + lane] =
                      F8 ? fmaf(__uint_as_float(b[e]), 0.0357142857f, __uint_as_float(a[e])) : __uint_as_float(a[e]);
              }
            }
          }
        }
        tc_fence_before();
        ch_named_sync(3 + s, kBar);
        for (int x = tid; x < nrows * 16; x += kBar) {
          const int r = x >> 4, d = (x & 15) * 4;
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
          float lr = 0.f, m = -INFINITY;
          if (ntile > 0) {
            y = *(const float4*)(os + r * 64 + d);
            lr = red[r];
#pragma unroll
            for (int w = 1; w < kSums; ++w) lr += red[w * N + r];
            m = -nref[r];
          }
          if (slot >= 0) {
            const int64_t row = ((int64_t)slot * HB + s) * N + r;
            *(float4*)(p.part_o + row * kChunkD + d) = y;
            if (d == 0) *(float2*)(p.part_ml + row * 2) = make_float2(m, lr);
          } else {
            const int tk = r / p.G, h = head0 + r - tk * p.G;
            const int64_t tok = sg.tok0 + tk;
            if (p.lse && d == 0) p.lse[tok * p.Hq + h] = m + log2f(lr);
            const float inv = ch_norm(p, h, lr, m);
            *(uint2*)(p.o + (tok * p.Hq + h) * kChunkD + d) =
                make_uint2(ch_bf16x2(y.x * inv, y.y * inv), ch_bf16x2(y.z * inv, y.w * inv));
          }
        }
        ch_named_sync(3 + s, kBar);  // red, nref and os are free again
      }
      if (slot >= 0) {
        __threadfence();
        ch_named_sync(5, 2 * kBar);
        if (threadIdx.x == 0) {
          const uint32_t old = atomicAdd(&p.counters[sg.c0], 1u);
          const uint32_t last = old == (uint32_t)(sg.c1 - sg.c0);
          if (last) p.counters[sg.c0] = 0u;
          *flag = last;
        }
        ch_named_sync(6, 2 * kBar);
        if (*flag) {
          __threadfence();
          chunk_join(p, sg, HB, N, threadIdx.x, 2 * kBar);
        }
        ch_named_sync(5, 2 * kBar);  // flag is free again
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[sb]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kMma0) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmem);
  }
}

// ---------------------------------------------------------- rows on M --
// CTA = two tiles of 128 rows (128 / G tokens times the G heads of a kv head),
// two softmax warpgroups each (thread = row = TMEM lane, half of a tile's 128
// keys), one warp that loads, one that issues the products: S_t = Q_t K^T (both
// in shared memory), O_t += P_t V (P_t bf16 in TMEM, in the place of S_t).  S has
// three buffers: the scores of three (key tile, tile) steps are ahead of their
// softmax, so a warp that ends a step finds the next one's ready.
//
// Bound by the exponentials and what stands around them: 2 x 128 x 128 a key
// tile at 16 per cycle and SM are 2048 cycles, the products 1024, K and V from
// L2 32 KB; a step of a warp is 405 instructions for its 32 x 64 scores, 64 of
// them exponentials, and every operation that passes the same queue (barriers,
// shared memory, TMEM) waits behind those.  So a step has few: the row's two
// warps agree by one barrier whether a reference has to move (they exchange
// maxima only then), and wait for O_t only then.  Measured, 2048 tokens on a
// sequence of 32768: 1342 us in bf16, 794 TFLOP/s, 3000 cycles a key tile.  One
// softmax warpgroup a tile took 1718, two that exchange every maximum 1504,
// turns between the tiles by a barrier 1480; without the polynomial below 1421.
//
// 8-bit pages: two more warpgroups turn a tile's values into bf16 with their
// power of two (exact) while those before are used: 60 instructions for 32 x 16
// values; the rest of the kernel is the same.  1872 us for the same call: a key
// tile's conversion is a third of the instructions that its softmax is.  (One
// converting warpgroup: 3121.)  Its 28 warps leave 72 registers a thread (88 for
// the softmax): 222 bytes of one are spilled, 12 in bf16.
constexpr int kRowsKT = 128;
// Bits 0 .. n set (none for n < 0).
__device__ __forceinline__ uint32_t ch_bits_to(int32_t n) { return n < 0 ? 0u : n >= 31 ? ~0u : (2u << n) - 1u; }
__device__ __forceinline__ float ch_max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}
__device__ __forceinline__ float ch_max3_nan(float a, float b, float c) {
  float m;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
  return m;
}
// 2^x of two values without the exponential unit: x = n + f with n its floor, 2^f a polynomial of degree 4 with value 1
// at 0 that is nowhere on [0, 1] further than 2^-17 of 2^f (its coefficients solve that minimax problem), n added to the
// exponent.  Below 2^-127 it is 0: f is 0 there.  P has 8 bits.
__device__ __forceinline__ void ch_exp2_poly(ch_f2 x, float& p0, float& p1) {
  const float kMagic = 12582912.0f;  // 1.5 * 2^23: a sum with it has its integer part in the low bits
  x = ch_pair(fmaxf(ch_lo(x), -127.0f), fmaxf(ch_hi(x), -127.0f));
  ch_f2 t;
  asm("add.rm.f32x2 %0, %1, %2;" : "=l"(t) : "l"(x), "l"(ch_pair(kMagic, kMagic)));
  const ch_f2 n = ch_add2(t, ch_pair(-kMagic, -kMagic));
  const ch_f2 f = ch_fma2(n, ch_pair(-1.0f, -1.0f), x);
  ch_f2 q = ch_fma2(f, ch_pair(0.0134266838f, 0.0134266838f), ch_pair(0.0522424765f, 0.0522424765f));
  q = ch_fma2(q, f, ch_pair(0.241280198f, 0.241280198f));
  q = ch_fma2(q, f, ch_pair(0.693044841f, 0.693044841f));
  q = ch_fma2(q, f, ch_pair(1.0f, 1.0f));
  p0 = __uint_as_float((uint32_t)q + ((uint32_t)t << 23));
  p1 = __uint_as_float((uint32_t)(q >> 32) + ((uint32_t)(t >> 32) << 23));
}

template <bool F8>
struct RowsCfg {
  static constexpr int kSoftmax = 16;        // softmax warps; then 4 that load, issue and check
  static constexpr int kConv = F8 ? 8 : 0;   // and those that turn 8-bit tiles into bf16
  static constexpr int kThreads = 32 * (kSoftmax + 4 + kConv);
  // registers: all have the same at first, then the softmax warps get what the others do without
  static constexpr int kRegs = (65536 / kThreads) & ~7;
  static constexpr int kRegAux = F8 ? 40 : 64, kRegConv = 56;
  static constexpr int kRegSoftmax = ((kRegs * kThreads - 128 * kRegAux - 32 * kConv * kRegConv) / (32 * kSoftmax)) & ~7;
  static constexpr int kStages = 4;
  static constexpr int kSide = kRowsKT * 128;            // K or V of a tile, bf16
  static constexpr int kRaw = F8 ? 2 : 0;                // stages of 8-bit tiles
  static constexpr int kRawSide = kRowsKT * 64;
  static constexpr int kOffRaw = 2 * 128 * 128 + kStages * 2 * kSide;
  static constexpr int kOffCodes = kOffRaw + kRaw * 2 * kRawSide;
  static constexpr int kOffNan = kOffCodes + kRaw * 2 * kRowsKT;  // per stage: a bit for each key, V row not finite
  static constexpr int kOffMax = kOffNan + kStages * 16;  // [tile][half][128]: maxima, at the end sums
  static constexpr int kOffPre = kOffMax + 2 * 2 * 128 * 4;
  static constexpr int kOffSeg = kOffPre + (kChunkMaxSeqs + 1 + 15) / 16 * 64;
  static constexpr int kOffBar = kOffSeg + 2 * (int)sizeof(ChunkSeg);
  static constexpr int kAlloc = kOffBar + (3 * kStages + 4 + 4 + 2 + 4 + 4 + 2) * 8 + 16 + 1024;
  static_assert(kAlloc <= 227 * 1024, "shared memory");
};

// 32 consecutive 32-bit columns of this warp's 32 lanes, no wait.
__device__ __forceinline__ void ch_ld32(uint32_t taddr, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void ch_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

template <bool F8>
__global__ void __launch_bounds__(RowsCfg<F8>::kThreads, 1)
    chunk_rows_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                      const __grid_constant__ CUtensorMap tmap_v, const ChunkParams p) {
  using C = RowsCfg<F8>;
  constexpr int NS = C::kStages, RB = F8 ? 64 : 128;
  constexpr int SW = C::kSoftmax, CV = C::kConv, KW = 64, DW = 32;  // a warp's share of a tile's keys, of the dims
  constexpr uint32_t kColO = 384;  // after three buffers of 128 columns for S
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* kv0 = smem + 2 * 128 * 128;
  int32_t* pre = (int32_t*)(smem + C::kOffPre);
  ChunkSeg* segs = (ChunkSeg*)(smem + C::kOffSeg);
  uint64_t* kvfull = (uint64_t*)(smem + C::kOffBar);
  uint64_t* kvempty = kvfull + NS;
  uint64_t* vready = kvempty + NS;  // bf16: V has been looked at
  uint64_t* rawfull = vready + NS;  // [2]
  uint64_t* rawempty = rawfull + 2;  // [2]
  uint64_t* seg_full = rawempty + 2;
  uint64_t* seg_empty = seg_full + 2;
  uint64_t* qfull = seg_empty + 2;
  uint64_t* qempty = qfull + 1;
  uint64_t* sfull = qempty + 1;  // [tile][key tile & 1]
  uint64_t* pfull = sfull + 4;   // [tile][key tile & 1]
  uint64_t* ofull = pfull + 4;   // [tile]
  volatile uint32_t* flag = (volatile uint32_t*)(ofull + 2);
  volatile uint32_t* tmem_slot = flag + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tq1 = p.TQ / 2;  // tokens of a tile

  if (threadIdx.x == 0) {
    for (int s = 0; s < NS; ++s) {
      mbar_init(&kvfull[s], F8 ? CV : 1);
      mbar_init(&kvempty[s], 1);
      mbar_init(&vready[s], 2);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(&rawfull[s], 33);  // the loading warp's lanes arrive with their copies of the codes
      mbar_init(&rawempty[s], CV);
      mbar_init(&seg_full[s], 1);
      mbar_init(&seg_empty[s], SW + 1 + (F8 ? CV : 2));
      mbar_init(&sfull[2 * s], 1);
      mbar_init(&sfull[2 * s + 1], 1);
      mbar_init(&pfull[2 * s], SW / 2);
      mbar_init(&pfull[2 * s + 1], SW / 2);
      mbar_init(&ofull[s], 1);
    }
    mbar_init(qfull, 1);
    mbar_init(qempty, 1);
    fence_mbar_init();
  }
  if (warp == SW + 1) {
    tmem_alloc((uint32_t*)tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  chunk_plan(p, pre, C::kThreads);  // with a __syncthreads at its end
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  int it = 0;  // key tiles so far
  bool bad = false;
  if (warp >= SW + 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegConv));
  if (warp >= SW && warp < SW + 4) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::kRegAux));
  if (warp == SW) {
    // ------------------------------------------------------------- loads
    ChunkWalk walk;
    walk.begin(p, pre, gridDim.x, blockIdx.x);
    for (int sn = 0;; ++sn) {
      const int sb = sn & 1;
      ChunkSeg sg;
      const bool more = walk.next(p, sg);
      if (!bad) bad = !mbar_wait(&seg_empty[sb], ((uint32_t)(sn >> 1) & 1u) ^ 1u, p.err, kErrTimeoutEmpty);
      if (lane == 0) {
        if (!more) sg.nrows = -1;
        segs[sb] = sg;
        mbar_arrive(&seg_full[sb]);
      }
      __syncwarp();
      if (!more || bad) break;
      if (!bad) bad = !mbar_wait(qempty, ((uint32_t)sn & 1u) ^ 1u, p.err, kErrTimeoutEmpty);
      if (lane == 0) {
        // Q: rows (token, head of the group) of both tiles
        const int nq = sg.ntile == 0 ? 0 : sg.ntok > tq1 ? 2 : 1;
        mbar_arrive_expect_tx(qfull, (uint32_t)(nq * tq1 * p.G * 128));
        for (int t = 0; t < nq; ++t)
          tma_load_3d(smem + t * 128 * 128, &tmap_q, 0, sg.hg * p.G, (int32_t)(sg.tok0 + t * tq1), qfull);
      }
      __syncwarp();
      const int32_t* trow = p.table + (int64_t)sg.row * p.tstride;
      for (int i = 0; i < sg.ntile; ++i, ++it) {
        // lanes 0..7: the pages of this tile that hold a key to look at
        const int32_t j = sg.j0 + i * kRowsKT + (lane & 7) * kChunkPage;
        const bool on = j < sg.hi && j + kChunkPage > sg.lo;
        int32_t page = -1;
        if (on) page = __ldg(trow + (uint32_t)(j / kChunkPage) % (uint32_t)p.tstride);
        if (page >= p.pool_pages) page = -1;  // a page outside the pool is not read
        const uint32_t n8 = (uint32_t)__popc(__ballot_sync(0xffffffffu, page >= 0 && lane < 8));
        const int st = F8 ? it % 2 : it % NS;
        uint64_t* full = F8 ? &rawfull[st] : &kvfull[st];
        uint8_t* kd = F8 ? smem + C::kOffRaw + st * 2 * C::kRawSide : kv0 + st * 2 * C::kSide;
        const int side = F8 ? C::kRawSide : C::kSide;
        if (!bad)
          bad = !mbar_wait(F8 ? &rawempty[st] : &kvempty[st], ((uint32_t)(it / (F8 ? 2 : NS)) & 1u) ^ 1u, p.err,
                           kErrTimeoutEmpty);
        if (lane == 0) mbar_arrive_expect_tx(full, n8 * 2 * kChunkPage * RB);
        __syncwarp();
        if (page >= 0 && lane < 8) {
          tma_load_3d(kd + lane * kChunkPage * RB, &tmap_k, 0, sg.hg, page * kChunkPage, full);
          tma_load_3d(kd + side + lane * kChunkPage * RB, &tmap_v, 0, sg.hg, page * kChunkPage, full);
        }
        if (F8) {
          // 16 bytes of codes per page: lanes 0..7 K's, 8..15 V's
          if (page >= 0 && lane < 16) {
            const uint8_t* src = (lane >> 3 ? p.v_code : p.k_code) + ((int64_t)page * p.Hkv + sg.hg) * kChunkPage;
            asm volatile("cp.async.ca.shared.global [%0], [%1], 16;" ::"r"(
                             smem_u32(smem + C::kOffCodes + st * 2 * kRowsKT + lane * kChunkPage)),
                         "l"(src)
                         : "memory");
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(full)) : "memory");
        }
        __syncwarp();
      }
    }
  } else if (warp == SW + 1) {
    // ---------------------------------------------------------- products
    if (elect_one()) {
      const uint32_t idesc_s = make_idesc_bf16(128, kRowsKT);
      const uint32_t idesc_o = make_idesc_bf16(128, 64) | (1u << 16);  // B (V) read dims-major
      const uint64_t dq = make_sdesc_sw128(smem_u32(smem)), dk = make_sdesc_sw128(smem_u32(kv0)),
                     dv = make_sdesc_sw128(smem_u32(kv0 + C::kSide));
      int ks = 0, vs = 0, sbuf = 0, pbuf = 0;
      uint32_t kp = 0, op = 0, sp = 0;  // parity of the stage; P_t and S_t so far, 2 and 1 bits each (a tile may sit out)
      for (int sn = 0; !bad; ++sn) {
        const int sb = sn & 1;
        bad = !mbar_wait(&seg_full[sb], (uint32_t)(sn >> 1) & 1u, p.err, kErrTimeoutFull);
        if (bad || segs[sb].nrows < 0) break;
        const int nt = segs[sb].ntile, tiles = segs[sb].ntok > tq1 ? 2 : 1, total = nt * tiles;
        bad = !mbar_wait(qfull, (uint32_t)sn & 1u, p.err, kErrTimeoutFull);
        // Products in the order (key tile, tile).  The scores go three ahead of P V (two with one tile, so that the
        // wait for a tile's output cannot meet the one two before): the buffer they go to is the one whose P V was
        // issued last, and the tensor core keeps the order.
        auto issue_s = [&](int n) {
          const int t = tiles == 2 ? n & 1 : 0;
          if (t == 0 && !bad) bad = !mbar_wait(&kvfull[ks], kp, p.err, kErrTimeoutFull);
          tc_fence_after();
          const uint64_t a = dq + t * (128 * 128 >> 4), b = dk + (uint32_t)ks * (2 * C::kSide >> 4);
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            tc_mma_ss(tmem + sbuf * 128, a + 2 * kk, b + 2 * kk, idesc_s, kk > 0 ? 1u : 0u);
          tc_commit(&sfull[2 * t + (sp >> t & 1u)]);
          sp ^= 1u << t;
          if (++sbuf == 3) sbuf = 0;
          if (t == tiles - 1 && ++ks == NS) {
            ks = 0;
            kp ^= 1u;
          }
          if (n == total - 1) tc_commit(qempty);
        };
        if (nt == 0) mbar_arrive(qempty);
        const int ahead = min(tiles + 1, total);
        for (int n = 0; n < ahead; ++n) issue_s(n);
        for (int n = 0; n < total; ++n) {
          const int t = tiles == 2 ? n & 1 : 0;
          // t's tiles so far: bit 0 picks the barrier, bit 1 is its parity
          if (!bad) bad = !mbar_wait(&pfull[2 * t + (op >> 2 * t & 1u)], op >> (2 * t + 1) & 1u, p.err, kErrTimeoutAccum);
          op = t ? (op & 3u) | ((op + 4u) & 12u) : (op & 12u) | ((op + 1u) & 3u);
          tc_fence_after();
          const uint64_t b = dv + (uint32_t)vs * (2 * C::kSide >> 4);
#pragma unroll
          for (int kk = 0; kk < 8; ++kk)
            tc_mma_ts(tmem + kColO + 64 * t, tmem + pbuf * 128 + (kk >> 2) * KW + (kk & 3) * 8, b + 128 * kk, idesc_o,
                      (n >= tiles || kk > 0) ? 1u : 0u);
          tc_commit(&ofull[t]);
          if (++pbuf == 3) pbuf = 0;
          if (t == tiles - 1) {
            tc_commit(&kvempty[vs]);
            if (++vs == NS) vs = 0;
          }
          if (n + ahead < total) issue_s(n + ahead);
        }
        mbar_arrive(&seg_empty[sb]);
      }
    }
    __syncwarp();
  } else if (warp >= SW + 4) {
    // ------------------------------------------- 8-bit tiles to bf16 tiles
    if (F8) {
      const int cw = warp - (SW + 4), tid = cw * 32 + lane;
      for (int sn = 0;; ++sn) {
        const int sb = sn & 1;
        if (!bad) bad = !mbar_wait(&seg_full[sb], (uint32_t)(sn >> 1) & 1u, p.err, kErrTimeoutFull);
        if (bad || segs[sb].nrows < 0) break;
        const int nt = segs[sb].ntile;
        const int32_t j0 = segs[sb].j0, lo = segs[sb].lo, hi = segs[sb].hi, first = segs[sb].first_pos;
        const int32_t last = first + segs[sb].ntok - 1;
        for (int i = 0; i < nt; ++i, ++it) {
          const int rs = it & 1, st = it % NS;
          const int32_t jt = j0 + i * kRowsKT;
          const bool edge = jt + kRowsKT - 1 > first || jt < lo || (p.window > 0 && jt <= last - p.window);
          if (!bad) bad = !mbar_wait(&rawfull[rs], (uint32_t)(it >> 1) & 1u, p.err, kErrTimeoutFull);
          if (!bad) bad = !mbar_wait(&kvempty[st], ((uint32_t)(it / NS) & 1u) ^ 1u, p.err, kErrTimeoutEmpty);
          const uint8_t* raw = smem + C::kOffRaw + rs * 2 * C::kRawSide;
          const uint8_t* codes = smem + C::kOffCodes + rs * 2 * kRowsKT;
          uint8_t* dst = kv0 + st * 2 * C::kSide;
          // 4 threads a key, 16 values each
          constexpr int X = 512 / (CV * 32 + !F8);
          uint4 w4[2 * X];
          uint32_t code4[2 * X];
#pragma unroll
          for (int y = 0; y < 2 * X; ++y) {
            w4[y] = *(const uint4*)(raw + (y * CV * 32 + tid) * 16);
            code4[y] = codes[(y * CV * 32 + tid) >> 2];
          }
#pragma unroll
          for (int side = 0; side < 2; ++side)
#pragma unroll
            for (int x = 0; x < X; ++x) {
              const int idx = x * CV * 32 + tid, key = idx >> 2, c = idx & 3;
              const int32_t j = jt + key;
              uint32_t o[8];
              bool on = j >= lo && j < hi;  // a key nobody may see: zeros, whatever its page (or an earlier tile) holds
              const uint4 w = w4[side * X + x];
              const uint32_t code = code4[side * X + x];
              if (side && edge) {
                // V rows that are not finite, where some row does not see them: zeros and a mark, see the softmax
                uint32_t n = 0;
                const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int y = 0; y < 4; ++y) n |= ((ww[y] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
                const uint32_t bad4 = __ballot_sync(0xffffffffu, on && (n != 0u || code == 255u));
                if (bad4 >> (lane & 28) & 15u) on = false;
                if (lane == 0) {
                  uint32_t bits = 0;
#pragma unroll
                  for (int y = 0; y < 8; ++y) bits |= (bad4 >> (4 * y) & 15u) ? 1u << y : 0u;
                  smem[C::kOffNan + st * 16 + x * CV + cw] = (uint8_t)bits;
                }
              }
              if (on) {
                const uint32_t mul = ch_code_mul(code);
                ch_e4m3_to_bf16(w.x, mul, o[0], o[1]);
                ch_e4m3_to_bf16(w.y, mul, o[2], o[3]);
                ch_e4m3_to_bf16(w.z, mul, o[4], o[5]);
                ch_e4m3_to_bf16(w.w, mul, o[6], o[7]);
                if (code > kCodeOne) {
                  const uint32_t rest = ch_code_rest(code);
#pragma unroll
                  for (int y = 0; y < 8; ++y) o[y] = bf16x2_mul(o[y], rest);
                }
              } else {
#pragma unroll
                for (int y = 0; y < 8; ++y) o[y] = 0u;
              }
              uint8_t* row = dst + side * C::kSide + key * 128;
              *(uint4*)(row + (((2 * c) ^ (key & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
              *(uint4*)(row + (((2 * c + 1) ^ (key & 7)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
            }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&kvfull[st]);
            mbar_arrive(&rawempty[rs]);
          }
        }
        if (lane == 0) mbar_arrive(&seg_empty[sb]);
        __syncwarp();
      }
    }
  } else if (warp >= SW + 2) {
    if (!F8) {
      // ---------------------------------------------------- V rows at the edges
      // Rows that do not see a key have P = 0 there, and 0 times its V row must be 0: in tiles where some row does not,
      // the V rows of keys nobody sees and those that are not finite become zeros, the latter with a mark.
      const int half = warp - (SW + 2);
      for (int sn = 0;; ++sn) {
        const int sb = sn & 1;
        if (!bad) bad = !mbar_wait(&seg_full[sb], (uint32_t)(sn >> 1) & 1u, p.err, kErrTimeoutFull);
        if (bad || segs[sb].nrows < 0) break;
        const int nt = segs[sb].ntile;
        const int32_t j0 = segs[sb].j0, lo = segs[sb].lo, hi = segs[sb].hi, first = segs[sb].first_pos;
        const int32_t last = first + segs[sb].ntok - 1;
        for (int i = 0; i < nt; ++i, ++it) {
          const int st = it % NS;
          const int32_t jt = j0 + i * kRowsKT;
          if (!bad) bad = !mbar_wait(&kvfull[st], (uint32_t)(it / NS) & 1u, p.err, kErrTimeoutFull);
          if (jt + kRowsKT - 1 > first || jt < lo || (p.window > 0 && jt <= last - p.window)) {
#pragma unroll 1
            for (int x = 0; x < 2; ++x) {
              const int key = half * 64 + x * 32 + lane;
              uint4* vr = (uint4*)(kv0 + st * 2 * C::kSide + C::kSide + key * 128);
              const bool seen = jt + key >= lo && jt + key < hi;
              uint32_t most = 0;
#pragma unroll
              for (int c = 0; c < 8; ++c) {
                const uint4 y = vr[c];
                const uint32_t w[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) most = max(most, max((w[e] << 16) & 0x7FFFFFFFu, w[e] & 0x7FFF0000u));
              }
              const bool is_nan = seen && most >= 0x7F800000u;
              if (!seen || is_nan) {
#pragma unroll
                for (int c = 0; c < 8; ++c) vr[c] = make_uint4(0, 0, 0, 0);
              }
              const uint32_t bits = __ballot_sync(0xffffffffu, is_nan);
              if (lane == 0) *(uint32_t*)(smem + C::kOffNan + st * 16 + (half * 2 + x) * 4) = bits;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&vready[st]);
        }
        if (lane == 0) mbar_arrive(&seg_empty[sb]);
        __syncwarp();
      }
    }
  } else {
    // ----------------------------------------------------------- softmax
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::kRegSoftmax));
    // tile, half of its keys (and of the output's dims), row = TMEM lane
    const int t = warp / (SW / 2), half = warp >> 2 & 1, row = (warp & 3) * 32 + lane;
    const int pair = 8 + t * 4 + (warp & 3);  // barrier of the two warps that share 32 rows
    float* const own_max = (float*)(smem + C::kOffMax) + t * 256 + half * 128 + row;
    const float* const other_max = (const float*)(smem + C::kOffMax) + t * 256 + (half ^ 1) * 128 + row;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t o_col = tmem + lane_base + kColO + 64 * t + DW * half;
    const int tok_r = row / p.G;  // token of the row within the tile
    uint32_t c = 0;               // key tiles of this tile so far
    int buf0 = 0;                 // buffer of the part's first scores
    for (int sn = 0;; ++sn) {
      const int sb = sn & 1;
      if (!bad) bad = !mbar_wait(&seg_full[sb], (uint32_t)(sn >> 1) & 1u, p.err, kErrTimeoutFull);
      bad = ch_named_or(6, SW * 32, bad);  // all softmax warps leave together
      const ChunkSeg& sg = segs[sb];
      if (sg.nrows < 0 || bad) break;
      const int ntile = sg.ntile, ntok = sg.ntok;
      const int32_t jbase = sg.j0, first = sg.first_pos;
      const int tiles = ntok > tq1 ? 2 : 1;
      const bool tile_on = t < tiles;
      const int tok = t * tq1 + tok_r;
      const bool row_ok = tok_r < tq1 && tok < ntok;
      const bool warp_on = __any_sync(0xffffffffu, row_ok);
      const int32_t lo = sg.lo;
      const int32_t pos = row_ok ? first + tok : -1;
      const int32_t tile_first = first + t * tq1, tile_last = first + min(ntok, (t + 1) * tq1) - 1;
      // a row that is not in use has whatever its place in shared memory held for a query: scale 0, reference 0
      const float scale = row_ok ? p.scale2 : 0.f;
      float m_ref = row_ok ? -INFINITY : 0.f, l = 0.f;
      int buf = (buf0 + (tile_on ? t : 0)) % 3;
      buf0 = (buf0 + ntile * tiles) % 3;
      if (tile_on) {
        for (int i = 0; i < ntile; ++i, ++c) {
          const int32_t j0 = jbase + i * kRowsKT;
          const uint32_t s_col = tmem + lane_base + (uint32_t)(buf * 128 + KW * half);  // P takes the place of S
          buf = (buf + tiles) % 3;
          const int st = (it + i) % NS;
          if (!bad) bad = !mbar_wait(&sfull[2 * t + (c & 1)], c >> 1 & 1u, p.err, kErrTimeoutAccum);
          tc_fence_after();
          if (!warp_on) {  // no row of this warp is in use
            if (!F8 && t == 0 && !bad)
              bad = !mbar_wait(&vready[st], (uint32_t)((it + i) / NS) & 1u, p.err, kErrTimeoutFull);
            tc_fence_before();
            if (lane == 0) mbar_arrive(&pfull[2 * t + (c & 1)]);
            continue;
          }
          const bool whole = j0 + kRowsKT - 1 <= tile_first && j0 >= lo && (p.window <= 0 || j0 > tile_last - p.window);
          uint32_t r[KW];
#pragma unroll
          for (int e = 0; e < KW; e += 32) ch_ld32(s_col + e, r + e);
          tmem_ld_wait();
          if (!whole) {
            // bit e: the row sees key e of the warp's 64
            const int32_t top = pos - (j0 + KW * half), low = p.window > 0 ? top - p.window : -1;
            const uint32_t see[2] = {ch_bits_to(top) & ~ch_bits_to(low), ch_bits_to(top - 32) & ~ch_bits_to(low - 32)};
#pragma unroll
            for (int e = 0; e < KW; ++e)
              if (!(see[e >> 5] >> (e & 31) & 1u)) r[e] = __float_as_uint(-INFINITY);
          }
          // the largest score of the row: both halves'
          float mx0 = __uint_as_float(r[0]), mx1 = __uint_as_float(r[1]);
#pragma unroll
          for (int e = 2; e + 2 < KW; e += 4) {
            mx0 = ch_max3_nan(mx0, __uint_as_float(r[e]), __uint_as_float(r[e + 2]));
            mx1 = ch_max3_nan(mx1, __uint_as_float(r[e + 1]), __uint_as_float(r[e + 3]));
          }
          mx0 = ch_max3_nan(mx0, __uint_as_float(r[KW - 2]), ch_max_nan(mx1, __uint_as_float(r[KW - 1])));
          // The reference moves when the row's first scores come and when it falls 2^8 behind: P is at most 2^8, and a
          // row's output is multiplied rarely.  The two warps of a row agree by one barrier whether any has to, and
          // exchange their maxima only then.
          float pend = 1.0f;
          const bool over = row_ok && !(mx0 * scale <= m_ref + 8.0f);
          const bool move = ch_named_or(pair, 64, over);
          if (move) {
            *own_max = mx0;
            ch_named_sync(pair, 64);
            mx0 = ch_max_nan(mx0, *other_max) * scale;
            ch_named_sync(pair, 64);  // read before it is written again
            if (row_ok && !(mx0 <= m_ref + 8.0f)) {
              // NaN and infinity make the row NaN
              if (mx0 == INFINITY) mx0 = __int_as_float(0x7FC00000);
              pend = ch_exp2(m_ref - mx0);  // 0 for the first scores
              l *= pend;
              m_ref = mx0;
            }
          }
          {
            const float m_eff = m_ref == -INFINITY ? 0.f : m_ref;  // nothing seen so far: every P is 0
            const ch_f2 sc2 = ch_pair(scale, scale), nm2 = ch_pair(-m_eff, -m_eff);
            ch_f2 sum2 = 0ull;
#pragma unroll
            for (int e0 = 0; e0 < KW; e0 += 32) {
              uint32_t pk[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const ch_f2 x = ch_fma2(((ch_f2)r[e0 + 2 * e + 1] << 32) | r[e0 + 2 * e], sc2, nm2);
                float p0, p1;
                if (!F8 && (e & 7) == 7) {  // an eighth; 8 bit: the converters need those instructions
                  ch_exp2_poly(x, p0, p1);
                } else {
                  p0 = ch_exp2(ch_lo(x));
                  p1 = ch_exp2(ch_hi(x));
                }
                sum2 = ch_add2(sum2, ch_pair(p0, p1));
                pk[e] = ch_bf16x2(p0, p1);
              }
              ch_st16(s_col + e0 / 2, pk);
            }
            l += ch_lo(sum2) + ch_hi(sum2);
          }
          if (j0 + kRowsKT - 1 > first || j0 < lo || (p.window > 0 && j0 <= first + ntok - 1 - p.window)) {
            // P of the rows that see a key whose V row is not finite; the sum keeps its own
            if (!F8 && !bad) bad = !mbar_wait(&vready[st], (uint32_t)((it + i) / NS) & 1u, p.err, kErrTimeoutFull);
            const uint2 nans = *(const uint2*)(smem + C::kOffNan + st * 16 + 8 * half);
            if ((nans.x | nans.y) != 0u) {
              tmem_st_wait();
#pragma unroll 1
              for (int e = 0; e < KW; ++e) {
                if (!((e < 32 ? nans.x : nans.y) >> (e & 31) & 1u)) continue;
                const int32_t kj = j0 + KW * half + e;
                uint32_t w;
                asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(w) : "r"(s_col + e / 2) : "memory");
                tmem_ld_wait();
                if (kj <= pos && (p.window <= 0 || kj > pos - p.window))
                  w = e & 1 ? (w & 0xFFFFu) | 0x7FC00000u : (w & 0xFFFF0000u) | 0x7FC0u;
                asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(s_col + e / 2), "r"(w) : "memory");
                tmem_st_wait();
              }
            }
          }
          if (move && i > 0) {
            // O_t has the tiles before.  (The wait cannot meet the product two before: this tile's scores were issued
            // after it.)
            if (!bad) bad = !mbar_wait(&ofull[t], (c & 1) ^ 1u, p.err, kErrTimeoutAccum);
            tc_fence_after();
            uint32_t ov[DW];
            tmem_ld_x32(o_col, ov);
            tmem_ld_wait();
#pragma unroll
            for (int d = 0; d < DW; ++d) ov[d] = __float_as_uint(__uint_as_float(ov[d]) * pend);
            tmem_st_x32(o_col, ov);
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&pfull[2 * t + (c & 1)]);
        }
      }
      it += ntile;
      // ------------------------------------------------- end of a part
      const int slot = sg.slot;
      uint32_t ov[DW];
      if (tile_on) {  // the row's sum: the two halves' in their order
        *own_max = l;
        ch_named_sync(pair, 64);
        l = half ? *other_max + l : l + *other_max;
        ch_named_sync(pair, 64);
      }
      if (tile_on && ntile > 0) {
        if (!bad) bad = !mbar_wait(&ofull[t], (c & 1) ^ 1u, p.err, kErrTimeoutAccum);
        tc_fence_after();
        ch_ld32(o_col, ov);
        tmem_ld_wait();
        tc_fence_before();
      } else {
#pragma unroll
        for (int d = 0; d < DW; ++d) ov[d] = 0u;
      }
      if (row_ok) {
        const int hh = row - tok_r * p.G;
        if (slot >= 0) {
          const int64_t prow = (int64_t)slot * 256 + tok * p.G + hh;
          if (half == 0) *(float2*)(p.part_ml + prow * 2) = make_float2(m_ref, l);
#pragma unroll
          for (int d = 0; d < DW / 4; ++d)
            *(uint4*)(p.part_o + prow * kChunkD + DW * half + 4 * d) = make_uint4(ov[4 * d], ov[4 * d + 1], ov[4 * d + 2], ov[4 * d + 3]);
        } else {
          const int h = sg.hg * p.G + hh;
          const int64_t tg = sg.tok0 + tok;
          if (p.lse && half == 0) p.lse[tg * p.Hq + h] = m_ref + log2f(l);
          const float inv = ch_norm(p, h, l, m_ref);
          uint4* orow = (uint4*)(p.o + (tg * p.Hq + h) * kChunkD + DW * half);
#pragma unroll
          for (int d = 0; d < DW / 8; ++d) {
            uint32_t w[4];
#pragma unroll
            for (int y = 0; y < 4; ++y)
              w[y] = ch_bf16x2(__uint_as_float(ov[8 * d + 2 * y]) * inv, __uint_as_float(ov[8 * d + 2 * y + 1]) * inv);
            orow[d] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      if (slot >= 0) {
        __threadfence();
        ch_named_sync(5, SW * 32);
        if (threadIdx.x == 0) {
          const uint32_t old = atomicAdd(&p.counters[sg.c0], 1u);
          const uint32_t last = old == (uint32_t)(sg.c1 - sg.c0);
          if (last) p.counters[sg.c0] = 0u;
          *flag = last;
        }
        ch_named_sync(6, SW * 32);
        if (*flag) {
          __threadfence();
          chunk_join(p, sg, 1, 256, threadIdx.x, SW * 32);
        }
        ch_named_sync(5, SW * 32);  // flag is free again
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&seg_empty[sb]);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == SW + 1) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace

// --------------------------------------------------------------- launch --
namespace {

constexpr int kChunkSlotRows = 256;  // the most rows of a partial result

// The line of key tiles is counted in 31 bits.
bool chunk_fits(const ChunkParams& p, int kt) {
  const int64_t span = p.window > 0 ? (int64_t)p.window + p.TQ : (int64_t)p.tstride * kChunkPage;
  return (p.T / p.TQ + p.N) * p.HG * (span / kt + 2 + p.ov) < (1ll << 31);
}

template <bool F8, int N_>
int launch_keys(const void* k, const void* v, ChunkParams p, cudaStream_t s) {
  using C = KeysCfg<F8, N_>;
  static FuncSmemAttr attr;
  ensure_dyn_smem(attr, (const void*)chunk_keys_kernel<F8, N_>, C::kAlloc);
  const int grid = device_sm_count();
  const int HB = p.Hkv % 2 ? 1 : 2;  // with an odd number of kv heads one stream idles
  p.TQ = N_ / p.G;
  p.HG = p.Hkv / HB;
  p.lg_kt = C::KT == 256 ? 8 : 7;
  p.ov = C::KT == 256 ? 2 : 3;
  if (!chunk_fits(p, C::KT)) return -12;
  p.part_ml = p.part_o + (int64_t)2 * grid * HB * N_ * kChunkD;
  CUtensorMap tk, tv;
  const uint64_t rb = C::kRowBytes, tok = (uint64_t)p.Hkv * rb;
  const CUtensorMapDataType dt = F8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  // [values of a row, 8 rows, rows of a token, half pages]: a box is a page's 16 tokens in groups of 8; a row is a
  // head's values, or in 8 bits a pair of heads'
  const bool pair = F8 && HB == 2;
  const uint64_t width = pair ? 128 : 64;
  const uint64_t dims[4] = {width, 8, (uint64_t)(pair ? p.Hkv / 2 : p.Hkv), (uint64_t)p.pool_pages * 2};
  const uint64_t strides[3] = {tok, pair ? 128 : rb, tok * 8};
  const uint32_t box[4] = {(uint32_t)width, 8, (uint32_t)(pair ? 1 : HB), 2};
  const CUtensorMapSwizzle sw = F8 && !pair ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  if (make_tmap_4d(&tk, k, dt, dims, strides, box, sw) || make_tmap_4d(&tv, v, dt, dims, strides, box, sw)) return -2;
  chunk_keys_kernel<F8, N_><<<(unsigned)grid, C::kThreads, C::kAlloc, s>>>(tk, tv, p, HB);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

template <bool F8>
int launch_rows(const void* k, const void* v, ChunkParams p, cudaStream_t s) {
  using C = RowsCfg<F8>;
  static FuncSmemAttr attr;
  ensure_dyn_smem(attr, (const void*)chunk_rows_kernel<F8>, C::kAlloc);
  const int grid = device_sm_count();
  const int tq1 = 128 / p.G;
  p.TQ = 2 * tq1;
  p.HG = p.Hkv;
  p.lg_kt = 7;
  // A unit's ends cost about 3 key tiles (4 prompts of 1024: 104 us; with 2 112, with 5 114).  Where a window leaves it
  // no more than that many tiles and every SM has several, a cut through one costs more than it evens out: 8 makes cuts
  // fall between units (2048 tokens, window 128: 41 us, 52 with 3; but 32 x 5 tokens, under two an SM: 22.5, 21.4).
  const bool small = p.window > 0 && p.window + p.TQ <= 3 * kRowsKT;
  p.ov = small && (p.T / p.TQ + p.N) * p.HG > 3 * grid ? 8 : 3;
  if (!chunk_fits(p, kRowsKT)) return -12;
  p.part_ml = p.part_o + (int64_t)2 * grid * 256 * kChunkD;
  CUtensorMap tq, tk, tv;
  const uint64_t rb = F8 ? 64 : 128, tok = (uint64_t)p.Hkv * rb;
  const uint64_t dq[3] = {64, (uint64_t)p.Hq, (uint64_t)p.T}, sq[2] = {128, (uint64_t)p.q_stride * 2};
  const uint32_t bq[3] = {64, (uint32_t)p.G, (uint32_t)tq1};
  const uint64_t dk[3] = {64, (uint64_t)p.Hkv, (uint64_t)p.pool_pages * kChunkPage}, sk[2] = {rb, tok};
  const uint32_t bk[3] = {64, 1, kChunkPage};
  const CUtensorMapDataType dt = F8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMapSwizzle sw = F8 ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B;
  if (make_tmap_3d(&tq, p.q, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, dq, sq, bq, CU_TENSOR_MAP_SWIZZLE_128B) ||
      make_tmap_3d(&tk, k, dt, dk, sk, bk, sw) || make_tmap_3d(&tv, v, dt, dk, sk, bk, sw))
    return -2;
  chunk_rows_kernel<F8><<<(unsigned)grid, C::kThreads, C::kAlloc, s>>>(tq, tk, tv, p);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace

// Workspace: 256 bytes (word 0: the error flags), a counter per CTA (so far it has
// to be zero before its first use), then two partial results per CTA (rows of 64
// values, a maximum and a sum).
int64_t chunk_parts_at() { return 256 + ((int64_t)device_sm_count() * 4 + 255) / 256 * 256; }
int64_t chunk_workspace_bytes() {
  return chunk_parts_at() + (int64_t)device_sm_count() * 2 * kChunkSlotRows * (kChunkD + 2) * 4;
}

int launch_attn_chunk(ChunkParams p, const void* k, const void* v, int32_t f8, int32_t max_q, void* workspace,
                      cudaStream_t s) {
  if (p.N <= 0 || p.T <= 0) return 0;
  p.err = (uint32_t*)workspace;
  p.counters = (uint32_t*)((uint8_t*)workspace + 256);
  p.part_o = (float*)((uint8_t*)workspace + chunk_parts_at());
  const int64_t rows = (int64_t)max_q * p.G;
  // Rows of the longest chunk: up to 48 on the short side of the keys kernel, the smallest tile that holds them (32
  // sequences of 8192 8-bit keys, one token: 71 us with 16 rows, 84 with 32, 90 with 48; four tokens: 118 with 32, 131
  // with 48).  The rows kernel pads them to 128 but takes a key tile in less time and has cheaper ends, so it is ahead
  // from 64 rows on, and with few (sequence, kv head) units, whose tiles are few per SM.  Keys / rows kernel in us, 8 kv
  // heads, sequences x tokens on keys:
  //   bf16  64 rows     64x8 on 512 67 / 43, on 8192 296 / 298;  16x8 on 8192 98 / 87;  1x8 on 8192 67 / 30
  //   bf16  17..48      4x4 on 2048 23 / 18, on 8192 34 / 32;  1x6 on 8192 58 / 29;  but 16x4 on 8192 61 / 82
  //   bf16  9..16       1x2 on 512 15 / 13, on 8192 37 / 21;  but 4x2 on 8192 29 / 31
  //   8 bit 64 rows     16x8 on 8192 157 / 122;  1x8 on 8192 74 / 33;  64x8 on 2048 182 / 133, on 8192 498 / 445
  //   8 bit 33..48      1x6 on 8192 59 / 33;  4x6 on 2048 29 / 24, on 8192 44 / 43;  but 5x6 on 8192 46 / 49, 32x6 154 / 228
  //   8 bit 17..32      1x4 on 512 17 / 16, on 8192 42 / 25;  2x4 on 8192 30 / 29;  but 3x4 on 8192 32 / 34
  //   8 bit 9..16       1x2 on 512 15 / 16, on 8192 24 / 25;  4x2 on 8192 23 / 39
  // and with up to 8 rows the keys kernel, 4x1 on 8192: 24 / 30, 8 bit 21 / 39; 1x1 on 512: 11.8 / 12.1, 8 bit 13 / 15, on
  // 32768 31 / 34, 28 / 42 (but on 8192 23 / 21, 22 / 24).  The keys a token can reach count the same way (`span`, from the
  // window and the table): bf16 33..48 rows, 64x6 on 512 53 / 42, on 2048 89 / 91; 16x6 on 2048 40 / 35.
  const int64_t units = (int64_t)p.N * p.Hkv, sms = device_sm_count();
  const int64_t pages = (int64_t)p.tstride * kChunkPage, span = p.window > 0 ? min64((int64_t)p.window + max_q, pages) : pages;
  const bool few = rows <= 8    ? false
                   : rows <= 16 ? !f8 && 16 * units <= sms
                   : rows <= 48 ? (f8 && rows <= 32 ? 8 : 4) * units <= sms || (!f8 && rows > 32 && span <= 2048)
                                : true;
  if (!few) {
    if (rows <= 16 && p.G <= 16) return f8 ? launch_keys<true, 16>(k, v, p, s) : launch_keys<false, 16>(k, v, p, s);
    if (rows <= 32 && p.G <= 32) return f8 ? launch_keys<true, 32>(k, v, p, s) : launch_keys<false, 32>(k, v, p, s);
    if (rows <= 48 && p.G <= 48) return f8 ? launch_keys<true, 48>(k, v, p, s) : launch_keys<false, 48>(k, v, p, s);
  }
  return f8 ? launch_rows<true>(k, v, p, s) : launch_rows<false>(k, v, p, s);
}

}  // namespace gptoss
