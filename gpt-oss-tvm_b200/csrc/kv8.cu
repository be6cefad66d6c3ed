// kv8.cu -- the 8-bit KV cache: keys and values quantised as they are written
// to the pages, and read back.
//
//   qkv_rope_append_f8_kernel  split of the fused QKV projection, YaRN RoPE on
//                        q and k, k and v quantised into their pool rows
//   kv_pages_f8_kernel   contiguous bf16 rows <-> 8-bit pages (both directions)
//
// Format.  A pool holds e4m3 values [rows, Hkv, 64] (16 rows = one page) and
// one E8M0 code per row and head, [rows / 16, Hkv, 16] -- the 16 codes of a
// page and head are one 16-byte piece.  For a head row x with largest
// magnitude a:
//   e    = the smallest integer in [-60, 60] with a <= 448 * 2^e
//   code = e + 127,  value = e4m3(x * 2^-e)  (nearest, ties to even, +-448 at most)
// A power of two loses nothing against a finer scale: e4m3 is a floating
// format, its relative precision does not depend on where a lies in the
// binade, and value * 2^e is then exact in bf16.  A row that holds a NaN gets
// code 255 and values 0 and reads back as NaN; magnitudes above 448 * 2^60 (infinities too)
// saturate.
#include "common.cuh"
#include "launch.h"

namespace gptoss {

constexpr int kKv8D = 64;
constexpr int kKv8MinExp = -60, kKv8MaxExp = 60;

// Largest magnitude of a row as fp32 bits (NaN patterns sort above infinity) -> code.
__device__ __forceinline__ uint32_t kv8_code(uint32_t amax_bits) {
  if (amax_bits > 0x7F800000u) return 255u;
  const int ex = (int)(amax_bits >> 23) - 127;
  // 448 = 1.75 * 2^8
  int e = ex - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  e = max(kKv8MinExp, min(kKv8MaxExp, e));
  return (uint32_t)(e + 127);
}
// 2^-(code - 127)
__device__ __forceinline__ float kv8_inv_scale(uint32_t code) { return __uint_as_float((254u - min(code, 253u)) << 23); }

// lo -> byte 0, hi -> byte 1
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t bf16x2_of(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

// Four e4m3 bytes of w as two bf16 pairs (b0, b1), (b2, b3) times `mul`, exactly
// (subnormals included): a byte below eight copies of its sign, moved up by four
// bits, is a bf16 that reads 2^-120 of the value.
__device__ __forceinline__ void e4m3x4_to_bf16(uint32_t w, uint32_t mul, uint32_t& p01, uint32_t& p23) {
  p01 = bf16x2_mul((prmt(w, 0u, 0x9180u) << 4) & 0x87F087F0u, mul);
  p23 = bf16x2_mul((prmt(w, 0u, 0xB3A2u) << 4) & 0x87F087F0u, mul);
}
// Its factor: 2^(code - 127 + 120), NaN for code 255.  bf16 ends at 2^127, code 134; what is left above is kv8_rest.
constexpr uint32_t kKv8One = 134;
__device__ __forceinline__ uint32_t kv8_mul(uint32_t code) {
  const uint32_t h = code == 255u ? 0x7FC0u : ((min(code, kKv8One) + 120u) << 7);
  return h | (h << 16);
}
__device__ __forceinline__ uint32_t kv8_rest(uint32_t code) {
  const uint32_t h = (min(code, 194u) - kKv8One + 127u) << 7;
  return h | (h << 16);
}

constexpr int kKv8Tokens = 16, kKv8Blocks = 4;  // the most tokens of a block; blocks an SM holds

struct Kv8Rope {
  float inv_freq[kKv8D / 2];
};

// One block takes `tok_per_block` tokens: their rotation factors go to shared
// memory once (sincosf of pos * inv_freq), then each group of 4 lanes rotates
// one head: a lane holds dims 8 l .. 8 l + 7 and their partners 32 above, two
// 16-byte loads, and the row's largest magnitude takes two shuffles.  The
// rotation rounds as qkv_rope_kernel's does (the same q bits; k is rounded to
// bf16 before it is quantised, so the cache holds e4m3 of the bf16 cache's k).
// Measured, 64 + 2 x 8 heads: 8192 tokens in 34 us, 4.7 TB/s, 160 tokens in 4.0:
// the rotation and a row's exponent stand between a token's loads and its stores.
// Four blocks an SM with the next loads under way are ahead of five (36 us) and
// six (42), one wave of them of twelve an SM (35) and of blocks of 4 tokens without
// the early loads (38).
__global__ void __launch_bounds__(256, kKv8Blocks)
    qkv_rope_append_f8_kernel(const uint16_t* __restrict__ qkv, const int32_t* __restrict__ pos,
                              const int32_t* __restrict__ slot, int64_t S, int64_t pool_rows, int32_t Hq, int32_t Hkv,
                              const Kv8Rope tab, float conc, int32_t tok_per_block, uint16_t* __restrict__ q_out,
                              uint8_t* __restrict__ kp, uint8_t* __restrict__ vp, uint8_t* __restrict__ kcode,
                              uint8_t* __restrict__ vcode) {
  __shared__ __align__(16) float cos_s[kKv8Tokens * 32];
  __shared__ __align__(16) float sin_s[kKv8Tokens * 32];
  __shared__ int32_t slot_s[kKv8Tokens];
  const int64_t s0 = (int64_t)blockIdx.x * tok_per_block;
  const int nt = (int)min64(tok_per_block, S - s0);
  const int32_t Ht = Hq + 2 * Hkv;
  const int total = nt * Ht * 4;
  // a lane's 32 bytes; those of the next round are on their way while one is worked on
  uint4 na = make_uint4(0, 0, 0, 0), nb = na;
  auto fetch = [&](int i) {
    if (i < total) {
      const uint16_t* xr = qkv + (s0 * Ht + (i >> 2)) * kKv8D + 8 * (i & 3);
      na = ldg_nc_v4(xr);
      nb = ldg_nc_v4(xr + 32);
    }
  };
  fetch((int)threadIdx.x);
  if ((int)threadIdx.x < nt && slot) slot_s[threadIdx.x] = slot[s0 + threadIdx.x];
  for (int i = threadIdx.x; i < nt * 32; i += blockDim.x) {
    const float ang = __fmul_rn((float)pos[s0 + (i >> 5)], tab.inv_freq[i & 31]);
    float sn, cs;
    sincosf(ang, &sn, &cs);
    cos_s[i] = __fmul_rn(cs, conc);
    sin_s[i] = __fmul_rn(sn, conc);
  }
  __syncthreads();
  // whole groups of 4 lanes run or skip together; every lane of a warp stays in the loop for the shuffles
  for (int base = 0; base < total; base += blockDim.x) {
    const int i = base + threadIdx.x;
    const bool on = i < total;
    const int l = i & 3, h = on ? (i >> 2) % Ht : 0, tk = on ? (i >> 2) / Ht : 0;
    const int64_t s = s0 + tk;
    const uint4 xa = na, xb = nb;
    fetch(i + (int)blockDim.x);
    const uint32_t wa[4] = {xa.x, xa.y, xa.z, xa.w}, wb[4] = {xb.x, xb.y, xb.z, xb.w};
    float a[8], b[8];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      a[2 * k] = __uint_as_float(wa[k] << 16);
      a[2 * k + 1] = __uint_as_float(wa[k] & 0xFFFF0000u);
      b[2 * k] = __uint_as_float(wb[k] << 16);
      b[2 * k + 1] = __uint_as_float(wb[k] & 0xFFFF0000u);
    }
    if (h < Hq + Hkv) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float c = cos_s[tk * 32 + 8 * l + k], sv = sin_s[tk * 32 + 8 * l + k];
        const float lo = __fsub_rn(__fmul_rn(a[k], c), __fmul_rn(b[k], sv));
        const float hi = __fadd_rn(__fmul_rn(a[k], sv), __fmul_rn(b[k], c));
        a[k] = lo;
        b[k] = hi;
      }
    }
    // one rounding to bf16 (NaN stays NaN); v's values are bf16 already
    uint32_t ra[4], rb[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      ra[k] = bf16x2_of(a[2 * k], a[2 * k + 1]);
      rb[k] = bf16x2_of(b[2 * k], b[2 * k + 1]);
      a[2 * k] = __uint_as_float(ra[k] << 16);
      a[2 * k + 1] = __uint_as_float(ra[k] & 0xFFFF0000u);
      b[2 * k] = __uint_as_float(rb[k] << 16);
      b[2 * k + 1] = __uint_as_float(rb[k] & 0xFFFF0000u);
    }
    if (h < Hq) {
      if (on) {
        uint4* qd = (uint4*)(q_out + (s * Hq + h) * kKv8D + 8 * l);
        qd[0] = make_uint4(ra[0], ra[1], ra[2], ra[3]);
        qd[4] = make_uint4(rb[0], rb[1], rb[2], rb[3]);
      }
    }
    if (!__any_sync(0xffffffffu, on && h >= Hq)) continue;
    uint32_t am = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) am = max(am, max(abs_bits(a[k]), abs_bits(b[k])));
    am = max(am, __shfl_xor_sync(0xffffffffu, am, 1));
    am = max(am, __shfl_xor_sync(0xffffffffu, am, 2));
    if (on && h >= Hq) {
      const int hk = h < Hq + Hkv ? h - Hq : h - Hq - Hkv;
      const int64_t row = slot ? (int64_t)slot_s[tk] : s;
      if (row >= 0 && row < pool_rows) {
        const uint32_t code = kv8_code(am);
        const float inv = kv8_inv_scale(code);
        uint32_t r[4];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          r[k] = e4m3x2(a[4 * k] * inv, a[4 * k + 1] * inv) | (e4m3x2(a[4 * k + 2] * inv, a[4 * k + 3] * inv) << 16);
          r[2 + k] = e4m3x2(b[4 * k] * inv, b[4 * k + 1] * inv) | (e4m3x2(b[4 * k + 2] * inv, b[4 * k + 3] * inv) << 16);
        }
        if (code == 255u) r[0] = r[1] = r[2] = r[3] = 0u;
        uint8_t* p = (h < Hq + Hkv ? kp : vp) + (row * Hkv + hk) * kKv8D + 8 * l;
        *(uint2*)p = make_uint2(r[0], r[1]);
        *(uint2*)(p + 32) = make_uint2(r[2], r[3]);
        if (l == 0) (h < Hq + Hkv ? kcode : vcode)[((row >> 4) * Hkv + hk) * 16 + (row & 15)] = (uint8_t)code;
      }
    }
  }
}

// Rows pos0 .. pos0 + n - 1 of one sequence: 4 lanes per (row, head), K and V
// by the same lanes (two loads in flight); 16 values per lane, 16 bytes on the
// 8-bit side and 32 on the bf16 side.  Bound by the bytes: 131072 rows of 8 heads
// read back in 70 us, 5.8 TB/s, written in 71 (8192 rows in 5.9, from L2; one row
// and 1000 rows in 2.7 and 2.9, a launch).
template <bool kToPages>
__global__ void __launch_bounds__(256)
    kv_pages_f8_kernel(uint8_t* __restrict__ kp, uint8_t* __restrict__ vp, uint8_t* __restrict__ kcode,
                       uint8_t* __restrict__ vcode, int64_t pool_rows, const int32_t* __restrict__ table,
                       int32_t tstride, int64_t pos0, int64_t n, int32_t Hkv, uint16_t* __restrict__ kb,
                       uint16_t* __restrict__ vb) {
  const int64_t total = n * Hkv * 4;
  const int64_t step = (int64_t)gridDim.x * blockDim.x;
  // row and head advance by the step's own: no division in the loop (64-bit ones took as long as the copy)
  const int l = threadIdx.x & 3;
  const uint32_t first = (blockIdx.x * blockDim.x + threadIdx.x) >> 2, ahead = (gridDim.x * blockDim.x) >> 2;
  int64_t r = first / (uint32_t)Hkv;
  int h = (int)(first % (uint32_t)Hkv);
  const int r_step = (int)(ahead / (uint32_t)Hkv), h_step = (int)(ahead % (uint32_t)Hkv);
  auto advance = [&]() {
    r += r_step;
    h += h_step;
    if (h >= Hkv) {
      h -= Hkv;
      ++r;
    }
  };
  for (int64_t base = (int64_t)blockIdx.x * blockDim.x; base < total; base += step, advance()) {
    const int64_t i = base + threadIdx.x;
    const int64_t rh = i >> 2;
    bool on = i < total;
    int64_t row = 0;
    if (on) {
      const int64_t j = pos0 + r;
      row = (int64_t)__ldg(table + (uint32_t)(j >> 4) % (uint32_t)tstride) * 16 + (j & 15);
      on = row >= 0 && row < pool_rows;
    }
    const int64_t at = (row * Hkv + h) * kKv8D + 16 * l;
    const int64_t ca = ((row >> 4) * Hkv + h) * 16 + (row & 15);
    uint4* dk = (uint4*)(kb + rh * kKv8D + 16 * l);
    uint4* dv = (uint4*)(vb + rh * kKv8D + 16 * l);
    if (!kToPages) {
      if (!on) continue;
      const uint4 wk = *(const uint4*)(kp + at), wv = *(const uint4*)(vp + at);
      const uint32_t cc[2] = {kcode[ca], vcode[ca]};
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        const uint4 w = side ? wv : wk;
        const uint32_t mul = kv8_mul(cc[side]);
        uint32_t o[8];
        e4m3x4_to_bf16(w.x, mul, o[0], o[1]);
        e4m3x4_to_bf16(w.y, mul, o[2], o[3]);
        e4m3x4_to_bf16(w.z, mul, o[4], o[5]);
        e4m3x4_to_bf16(w.w, mul, o[6], o[7]);
        if (cc[side] > kKv8One) {
#pragma unroll
          for (int y = 0; y < 8; ++y) o[y] = bf16x2_mul(o[y], kv8_rest(cc[side]));
        }
        uint4* dst = side ? dv : dk;
        dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
        dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
      }
    } else {
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        const uint4* src = side ? dv : dk;
        uint4 x0 = make_uint4(0, 0, 0, 0), x1 = x0;
        if (on) {
          x0 = src[0];
          x1 = src[1];
        }
        const uint32_t w[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
        uint32_t am = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) am = max(am, max((w[k] << 16) & 0x7FFFFFFFu, w[k] & 0x7FFF0000u));
        am = max(am, __shfl_xor_sync(0xffffffffu, am, 1));
        am = max(am, __shfl_xor_sync(0xffffffffu, am, 2));
        const uint32_t code = kv8_code(am);
        const float inv = kv8_inv_scale(code);
        uint32_t o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t u = w[2 * k], t = w[2 * k + 1];
          o[k] = e4m3x2(__uint_as_float(u << 16) * inv, __uint_as_float(u & 0xFFFF0000u) * inv) |
                 (e4m3x2(__uint_as_float(t << 16) * inv, __uint_as_float(t & 0xFFFF0000u) * inv) << 16);
        }
        if (code == 255u) o[0] = o[1] = o[2] = o[3] = 0u;
        if (on) {
          *(uint4*)((side ? vp : kp) + at) = make_uint4(o[0], o[1], o[2], o[3]);
          if (l == 0) (side ? vcode : kcode)[ca] = (uint8_t)code;
        }
      }
    }
  }
}

// --------------------------------------------------------------- launch --
int launch_qkv_rope_append_f8(const uint16_t* qkv, const int32_t* pos, const int32_t* slot, int64_t S,
                              int64_t pool_rows, int32_t Hq, int32_t Hkv, const float* inv_freq, float conc,
                              uint16_t* q_out, uint8_t* kp, uint8_t* vp, uint8_t* kcode, uint8_t* vcode,
                              cudaStream_t s) {
  if (S <= 0) return 0;
  Kv8Rope tab;
  for (int i = 0; i < kKv8D / 2; ++i) tab.inv_freq[i] = inv_freq[i];
  // one wave of blocks: their tokens' loads, sincosf and stores overlap better than a second wave's start
  const int64_t wave = (int64_t)device_sm_count() * kKv8Blocks;
  const int tpb = (int)min64((S + wave - 1) / wave, kKv8Tokens);
  qkv_rope_append_f8_kernel<<<(unsigned)((S + tpb - 1) / tpb), 256, 0, s>>>(qkv, pos, slot, S, pool_rows, Hq, Hkv, tab,
                                                                            conc, tpb, q_out, kp, vp, kcode, vcode);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

int launch_kv_pages_f8(uint8_t* kp, uint8_t* vp, uint8_t* kcode, uint8_t* vcode, int64_t pool_rows,
                       const int32_t* table, int32_t tstride, int64_t pos0, int64_t n, int32_t Hkv, uint16_t* kb,
                       uint16_t* vb, int32_t to_pages, cudaStream_t s) {
  if (n <= 0) return 0;
  const int64_t blocks = min64((n * Hkv * 4 + 255) / 256, (int64_t)device_sm_count() * 32);
  if (to_pages)
    kv_pages_f8_kernel<true><<<(unsigned)blocks, 256, 0, s>>>(kp, vp, kcode, vcode, pool_rows, table, tstride, pos0, n,
                                                              Hkv, kb, vb);
  else
    kv_pages_f8_kernel<false><<<(unsigned)blocks, 256, 0, s>>>(kp, vp, kcode, vcode, pool_rows, table, tstride, pos0,
                                                               n, Hkv, kb, vb);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace gptoss
