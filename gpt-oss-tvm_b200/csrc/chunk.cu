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
// chunk_rows_kernel   up to 64 rows (tokens x heads of a kv head): one pass
//                     over the keys, bound by their bytes
//
// The output is rounded once, from fp32; P is rounded to bf16 as the operand
// of P V (its relative error of 2^-9 an element is the size of the output's
// own rounding), the sum l takes the unrounded values.
#include "chunk.cuh"
#include "launch.h"

namespace gptoss {

namespace {

constexpr float kChLog2e = 1.4426950408889634f;

__device__ __forceinline__ void ch_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ch_ldsm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ch_ldsm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
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
// 128-byte rows, 16-byte piece c of row r (the 128-byte TMA swizzle)
__device__ __forceinline__ uint32_t ch_swz128(int r, int c) { return (uint32_t)(r * 128 + ((c ^ (r & 7)) << 4)); }
// 64-byte rows (the 64-byte TMA swizzle)
__device__ __forceinline__ uint32_t ch_swz64(int r, int c) { return (uint32_t)(r * 64 + ((c ^ ((r >> 1) & 3)) << 4)); }
// bytes (b0, b2) and (b1, b3) of w, e4m3, as bf16 pairs that read 2^-120 of their value
__device__ __forceinline__ uint32_t ch_e4m3_even(uint32_t w) { return ((w << 4) & 0x07F007F0u) | ((w << 8) & 0x80008000u); }
__device__ __forceinline__ uint32_t ch_e4m3_odd(uint32_t w) { return ((w >> 4) & 0x07F007F0u) | (w & 0x80008000u); }
// 2^(code - 127 + bias) as fp32, NaN for code 255 (a row that held a NaN)
__device__ __forceinline__ float ch_code_scale(uint32_t code, int bias) {
  return code == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float((uint32_t)((int)code + bias) << 23);
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
// Untiled 16-byte-granular copy, completion as tx bytes.
__device__ __forceinline__ void ch_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// ------------------------------------------------------------- few rows --
// CTA = 4 compute warps and one that loads.  Key tiles of 64 keys (4 pages) go
// through a ring of stages by TMA, one box of 16 keys x 64 values per page.
// Per tile, warp w takes keys 16 w .. 16 w + 15 of Q K^T for all rows, and after
// P went through shared memory, dims 16 w .. 16 w + 15 of P V over all 64 keys:
// no fragment of K or V is loaded (or, in 8 bits, unpacked) twice.  The softmax
// reference of a row moves only when a score exceeds it by 8 (P <= 2^8), which
// one barrier that also carries the vote tells all warps.
//
// 8-bit pages: e4m3 bits shifted into a bf16 read 2^-120 of the value, so no
// conversion is needed beyond two masks per pair; Q carries a factor 2^60, the
// key's power of two and the remaining 2^60 meet the score in fp32, and V's go
// to the column of P before it is rounded.  A key's code is one byte, applied
// exactly.
constexpr int kRowsKT = 64;
constexpr int kRowsWarps = 4;
constexpr int kRowsThreads = kRowsWarps * 32 + 32;

template <bool F8, int RT>
struct RowsCfg {
  static constexpr int kRows = 16 * RT;
  static constexpr int kStages = F8 ? 4 : 4;
  static constexpr int kRowBytes = F8 ? 64 : 128;
  static constexpr int kTile = kRowsKT * kRowBytes;           // K or V of one stage
  static constexpr int kCodes = F8 ? 2 * kRowsKT : 0;         // K and V codes of one stage
  static constexpr int kStageBytes = 2 * kTile;
  static constexpr int kOffCodes = kStages * kStageBytes;
  static constexpr int kOffP = kOffCodes + kStages * kCodes;  // P [rows][64] bf16
  static constexpr int kOffRed = kOffP + kRows * 128;         // [4][rows] floats
  static constexpr int kOffPre = kOffRed + kRowsWarps * kRows * 4;
  static constexpr int kOffBar = kOffPre + (kChunkMaxSeqs + 1 + 7) / 8 * 64;
  static constexpr int kAlloc = kOffBar + 2 * kStages * 8 + 16 + 1024;
};

template <bool F8, int RT>
__global__ void __launch_bounds__(kRowsThreads, RT == 1 ? 4 : RT == 2 ? 3 : 2)
    chunk_rows_kernel(const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                      const ChunkParams p) {
  using C = RowsCfg<F8, RT>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  float* red = (float*)(smem + C::kOffRed);
  int64_t* pre = (int64_t*)(smem + C::kOffPre);
  uint64_t* full = (uint64_t*)(smem + C::kOffBar);
  uint64_t* empty = full + C::kStages;
  volatile uint32_t* flag = (volatile uint32_t*)(empty + C::kStages);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], kRowsWarps);
    }
    fence_mbar_init();
  }
  ChunkWalk<kRowsKT>::plan(p, pre, kRowsThreads);  // ends with a __syncthreads
  ChunkWalk<kRowsKT> walk;
  walk.begin(p, pre, gridDim.x, blockIdx.x);
  ChunkSeg sg;
  int it = 0;  // key tiles through the ring so far
  bool bad = false;

  if (warp == kRowsWarps) {
    // ------------------------------------------------------------- loads
    while (walk.next(p, sg)) {
      if (sg.n == 0) continue;
      const int32_t* trow = p.table + (int64_t)sg.s.row * p.tstride;
      for (int i = sg.i0; i < sg.i1; ++i, ++it) {
        const int st = it % C::kStages;
        const uint32_t ph = (uint32_t)(it / C::kStages) & 1u;
        // lanes 0..3: the pages of this tile that hold a key to look at
        const int32_t j0 = sg.k0 + i * kRowsKT + lane * kChunkPage;
        const bool on = lane < kRowsKT / kChunkPage && j0 < sg.hi && j0 + kChunkPage > sg.lo;
        int32_t page = 0;
        if (on) page = __ldg(trow + (j0 / kChunkPage) % p.tstride);
        const bool in = on && page >= 0 && page < p.pool_pages;  // a page outside the pool is not read
        const int np = __popc(__ballot_sync(0xffffffffu, in));
        if (!bad) bad = !mbar_wait(&empty[st], ph ^ 1u, p.err, kErrTimeoutEmpty);
        if (lane == 0) mbar_arrive_expect_tx(&full[st], (uint32_t)(np * (2 * kChunkPage * C::kRowBytes + (F8 ? 32 : 0))));
        __syncwarp();
        if (in) {
          uint8_t* kd = smem + st * C::kStageBytes + lane * kChunkPage * C::kRowBytes;
          tma_load_3d(kd, &tmap_k, 0, sg.hk, page * kChunkPage, &full[st]);
          tma_load_3d(kd + C::kTile, &tmap_v, 0, sg.hk, page * kChunkPage, &full[st]);
          if (F8) {
            uint8_t* cd = smem + C::kOffCodes + st * C::kCodes + lane * kChunkPage;
            const int64_t ca = ((int64_t)page * p.Hkv + sg.hk) * kChunkPage;
            ch_bulk(cd, p.k_code + ca, kChunkPage, &full[st]);
            ch_bulk(cd + kRowsKT, p.v_code + ca, kChunkPage, &full[st]);
          }
        }
        __syncwarp();
      }
    }
    return;
  }

  // ------------------------------------------------------------- compute
  const int g = lane >> 2, t4 = lane & 3;
  const uint32_t sp = smem_u32(smem + C::kOffP);
  while (walk.next(p, sg)) {
    const int32_t tok0 = sg.t * p.TQ, ntok = min(p.TQ, sg.s.ql - tok0);
    const int nrows = ntok * p.G;
    // Q fragments, straight from global memory (the row index is token * G + head of the group)
    uint32_t qf[RT][4][4];
    int32_t pos_r[RT][2];  // position of the row's token, or -1 beyond the rows
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int r = rt * 16 + hf * 8 + g;
        const bool ok = r < nrows;
        const int tk = ok ? r / p.G : 0, hh = ok ? r % p.G : 0;
        pos_r[rt][hf] = ok ? sg.s.off + tok0 + tk : -1;
        const uint16_t* qr = p.q + (sg.s.q0 + tok0 + tk) * p.q_stride + (int64_t)(sg.hk * p.G + hh) * kChunkD;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          uint32_t a_lo = 0, a_hi = 0;
          if (ok) {
            if (F8) {
              // k-slots (2 t4, 2 t4 + 1, 2 t4 + 8, 2 t4 + 9) are dims 4 t4 + (0, 2, 1, 3): the order in which
              // the bytes of a key unpack
              const uint2 x = *(const uint2*)(qr + kk * 16 + 4 * t4);
              a_lo = bf16x2_mul(prmt(x.x, x.y, 0x5410u), 0x5D805D80u);  // times 2^60
              a_hi = bf16x2_mul(prmt(x.x, x.y, 0x7632u), 0x5D805D80u);
            } else {
              a_lo = *(const uint32_t*)(qr + kk * 16 + 2 * t4);
              a_hi = *(const uint32_t*)(qr + kk * 16 + 2 * t4 + 8);
            }
          }
          qf[rt][kk][hf] = a_lo;
          qf[rt][kk][2 + hf] = a_hi;
        }
      }
    }
    float m_ref[RT][2], l_r[RT][2], acc[RT][2][4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      m_ref[rt][0] = m_ref[rt][1] = -INFINITY;
      l_r[rt][0] = l_r[rt][1] = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[rt][0][e] = acc[rt][1][e] = 0.f;
    }
    const int ntile = sg.n == 0 ? 0 : sg.i1 - sg.i0;
    for (int ii = 0; ii < ntile; ++ii, ++it) {
      const int st = it % C::kStages;
      const int32_t j0 = sg.k0 + (sg.i0 + ii) * kRowsKT;
      const uint32_t sk = smem_u32(smem + st * C::kStageBytes), sv = sk + C::kTile;
      const uint8_t* ck = smem + C::kOffCodes + st * C::kCodes;
      if (!bad) bad = !mbar_wait(&full[st], (uint32_t)(it / C::kStages) & 1u, p.err, kErrTimeoutFull);
      // scores of keys 16 warp .. + 15
      float sc[RT][2][4];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[rt][0][e] = sc[rt][1][e] = 0.f;
      if (F8) {
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          uint32_t w[4];
          ch_ldsm(w, sk + ch_swz64(warp * 16 + nt * 8 + (lane & 7), lane >> 3));
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) {
            const uint32_t b0 = ch_e4m3_even(w[kk]), b1 = ch_e4m3_odd(w[kk]);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) ch_mma(sc[rt][nt], qf[rt][kk], b0, b1);
          }
        }
      } else {
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          uint32_t w[4];
          ch_ldsm(w, sk + ch_swz128(warp * 16 + (lane & 7) + ((lane >> 4) << 3), 2 * kk + ((lane >> 3) & 1)));
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            ch_mma(sc[rt][0], qf[rt][kk], w[0], w[1]);
            ch_mma(sc[rt][1], qf[rt][kk], w[2], w[3]);
          }
        }
      }
      const int32_t first_pos = sg.s.off + tok0;
      const bool whole = j0 + kRowsKT - 1 <= first_pos && j0 >= sg.lo &&
                         (p.window <= 0 || j0 > first_pos + ntok - 1 - p.window);
      float vscale[2][2];  // per key of this thread: 2^(e_v + 60)
      float mx[RT][2];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) mx[rt][0] = mx[rt][1] = -INFINITY;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        float ks[2] = {p.scale2, p.scale2};
        if (F8) {
          const int key = warp * 16 + nt * 8 + 2 * t4;
          const uint32_t kc = *(const uint16_t*)(ck + key), vc = *(const uint16_t*)(ck + kRowsKT + key);
          ks[0] = p.scale2 * ch_code_scale(kc & 0xFFu, 60);
          ks[1] = p.scale2 * ch_code_scale(kc >> 8, 60);
          vscale[nt][0] = ch_code_scale(vc & 0xFFu, 60);
          vscale[nt][1] = ch_code_scale(vc >> 8, 60);
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v = sc[rt][nt][e] * ks[e & 1];
            if (!whole) {
              const int32_t kj = j0 + warp * 16 + nt * 8 + 2 * t4 + (e & 1), ps = pos_r[rt][e >> 1];
              if (kj > ps || (p.window > 0 && kj <= ps - p.window)) v = -INFINITY;
            }
            sc[rt][nt][e] = v;
            mx[rt][e >> 1] = fmaxf(mx[rt][e >> 1], v);
          }
      }
      bool need = false;
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          mx[rt][hf] = fmaxf(mx[rt][hf], __shfl_xor_sync(0xffffffffu, mx[rt][hf], 1));
          mx[rt][hf] = fmaxf(mx[rt][hf], __shfl_xor_sync(0xffffffffu, mx[rt][hf], 2));
          need |= mx[rt][hf] > m_ref[rt][hf] + 8.0f;
        }
      if (!F8 && !whole) {
        // V rows of keys nobody may see: 0 times what the page holds there must be 0
        for (int c = threadIdx.x; c < kRowsKT * 8; c += kRowsWarps * 32) {
          const int32_t kj = j0 + (c >> 3);
          if (kj < sg.lo || kj >= sg.hi)
            *(uint4*)(smem + st * C::kStageBytes + C::kTile + c * 16) = make_uint4(0, 0, 0, 0);
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      }
      if (ch_named_or(1, kRowsWarps * 32, need)) {
        if (t4 == 0) {
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) red[warp * C::kRows + rt * 16 + hf * 8 + g] = mx[rt][hf];
        }
        ch_named_sync(2, kRowsWarps * 32);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            float m = m_ref[rt][hf];
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) m = fmaxf(m, red[w * C::kRows + rt * 16 + hf * 8 + g]);
            const float c = m == m_ref[rt][hf] ? 1.0f : ch_exp2(m_ref[rt][hf] - m);
            m_ref[rt][hf] = m;
            l_r[rt][hf] *= c;
#pragma unroll
            for (int dt = 0; dt < 2; ++dt) {
              acc[rt][dt][2 * hf] *= c;
              acc[rt][dt][2 * hf + 1] *= c;
            }
          }
      }
      // P, and its bf16 form for P V
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const float m = m_ref[rt][hf] == -INFINITY ? 0.f : m_ref[rt][hf];
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            float p0 = ch_exp2(sc[rt][nt][2 * hf] - m), p1 = ch_exp2(sc[rt][nt][2 * hf + 1] - m);
            l_r[rt][hf] += p0 + p1;
            if (F8) {
              p0 = p0 == 0.f ? 0.f : p0 * vscale[nt][0];
              p1 = p1 == 0.f ? 0.f : p1 * vscale[nt][1];
            }
            const int r = rt * 16 + hf * 8 + g;
            *(uint32_t*)(smem + C::kOffP + ch_swz128(r, 2 * warp + nt) + 4 * t4) = ch_bf16x2(p0, p1);
          }
        }
      ch_named_sync(3, kRowsWarps * 32);
      // O += P V, dims 16 warp .. + 15
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
        uint32_t w8[4];
        if (F8) ch_ldsm_t(w8, sv + ch_swz64(k2 * 32 + lane, warp));
#pragma unroll
        for (int kh = 0; kh < 2; ++kh) {
          const int kk = 2 * k2 + kh;
          uint32_t b[4];
          if (F8) {
            b[0] = ch_e4m3_even(w8[2 * kh]);
            b[1] = ch_e4m3_even(w8[2 * kh + 1]);
            b[2] = ch_e4m3_odd(w8[2 * kh]);
            b[3] = ch_e4m3_odd(w8[2 * kh + 1]);
          } else {
            ch_ldsm_t(b, sv + ch_swz128(kk * 16 + (lane & 7) + (((lane >> 3) & 1) << 3), 2 * warp + (lane >> 4)));
          }
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            uint32_t a[4];
            ch_ldsm(a, sp + ch_swz128(rt * 16 + (lane & 15), 2 * kk + (lane >> 4)));
            ch_mma(acc[rt][0], a, b[0], b[1]);
            ch_mma(acc[rt][1], a, b[2], b[3]);
          }
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }

    // ------------------------------------------------------- end of a part
    // this thread's dims of rows g, g + 8: [0..1] and [2..3] below are consecutive pairs
    //   bf16: dims 16 warp + 2 t4, + 1 (tile 0) and 16 warp + 8 + 2 t4, + 1 (tile 1)
    //   8 bit: dims 16 warp + 4 t4 + (0, 2) (tile 0) and + (1, 3) (tile 1)
    ch_named_sync(1, kRowsWarps * 32);  // red is free
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        float l = l_r[rt][hf];
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        if (t4 == 0) red[warp * C::kRows + rt * 16 + hf * 8 + g] = l;
      }
    ch_named_sync(2, kRowsWarps * 32);
    const float unit = F8 ? 1152921504606846976.0f : 1.0f;  // 2^60: what P and V left out
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const int r = rt * 16 + hf * 8 + g;
        float l = 0.f;
#pragma unroll
        for (int w = 0; w < kRowsWarps; ++w) l += red[w * C::kRows + r];
        const float m = m_ref[rt][hf];
        const int d0 = F8 ? warp * 16 + 4 * t4 : warp * 16 + 2 * t4, d1 = F8 ? d0 + 2 : d0 + 8;
        float x0 = acc[rt][0][2 * hf] * unit, x1 = acc[rt][0][2 * hf + 1] * unit;
        float x2 = acc[rt][1][2 * hf] * unit, x3 = acc[rt][1][2 * hf + 1] * unit;
        if (F8) {  // dims (0, 2), (1, 3) -> (0, 1), (2, 3)
          const float s = x1;
          x1 = x2;
          x2 = s;
        }
        if (sg.slot >= 0) {
          float* po = p.part_o + ((int64_t)sg.slot * C::kRows + r) * kChunkD;
          *(float2*)(po + d0) = make_float2(x0, x1);
          *(float2*)(po + d1) = make_float2(x2, x3);
          if (warp == 0 && t4 == 0)
            *(float2*)(p.part_ml + ((int64_t)sg.slot * C::kRows + r) * 2) = make_float2(m, l);
        } else if (r < nrows) {
          const int h = sg.hk * p.G + r % p.G;
          const int64_t tok = sg.s.q0 + tok0 + r / p.G;
          if (p.lse && warp == 0 && t4 == 0) p.lse[tok * p.Hq + h] = m + log2f(l);
          float den = l;
          if (p.sinks) den += exp2f(bf16_bits_to_f32(p.sinks[h]) * kChLog2e - m);
          const float inv = l == 0.f ? 0.f : 1.0f / den;
          uint16_t* orow = p.o + (tok * p.Hq + h) * kChunkD;
          *(uint32_t*)(orow + d0) = ch_bf16x2(x0 * inv, x1 * inv);
          *(uint32_t*)(orow + d1) = ch_bf16x2(x2 * inv, x3 * inv);
        }
      }
    if (sg.slot >= 0) {
      __threadfence();
      ch_named_sync(3, kRowsWarps * 32);
      if (threadIdx.x == 0) {
        const uint32_t old = atomicAdd(&p.counters[sg.c0], 1u);
        const uint32_t mine = old == (uint32_t)(sg.c1 - sg.c0);
        if (mine) p.counters[sg.c0] = 0u;
        *flag = mine;
      }
      ch_named_sync(1, kRowsWarps * 32);
      if (*flag) {
        __threadfence();
        // join the parts in the order of the keys: 16 lanes per row, 4 dims each
        for (int x = threadIdx.x; x < nrows * 16; x += kRowsWarps * 32) {
          const int r = x >> 4, d = (x & 15) * 4;
          float m = -INFINITY;
          for (int c = sg.c0; c <= sg.c1; ++c) {
            const int64_t sl = c == sg.c0 ? sg.first_slot : 2 * c;
            m = fmaxf(m, __ldcg(p.part_ml + (sl * C::kRows + r) * 2));
          }
          const float me = m == -INFINITY ? 0.f : m;
          float l = 0.f;
          float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
          for (int c = sg.c0; c <= sg.c1; ++c) {
            const int64_t sl = c == sg.c0 ? sg.first_slot : 2 * c;
            const float2 ml = __ldcg((const float2*)(p.part_ml + (sl * C::kRows + r) * 2));
            const float4 y = __ldcg((const float4*)(p.part_o + (sl * C::kRows + r) * kChunkD + d));
            const float f = exp2f(ml.x - me);
            l += ml.y * f;
            a.x += y.x * f;
            a.y += y.y * f;
            a.z += y.z * f;
            a.w += y.w * f;
          }
          const int h = sg.hk * p.G + r % p.G;
          const int64_t tok = sg.s.q0 + tok0 + r / p.G;
          if (p.lse && d == 0) p.lse[tok * p.Hq + h] = m + log2f(l);
          float den = l;
          if (p.sinks) den += exp2f(bf16_bits_to_f32(p.sinks[h]) * kChLog2e - m);
          const float inv = l == 0.f ? 0.f : 1.0f / den;
          uint2 w;
          w.x = ch_bf16x2(a.x * inv, a.y * inv);
          w.y = ch_bf16x2(a.z * inv, a.w * inv);
          *(uint2*)(p.o + (tok * p.Hq + h) * kChunkD + d) = w;
        }
      }
    }
    ch_named_sync(2, kRowsWarps * 32);  // red, flag are free again
  }
}

}  // namespace

// --------------------------------------------------------------- launch --
namespace {

constexpr int kChunkMaxCtasPerSm = 8;

struct Occupancy {
  std::atomic<int> per_dev[kMaxAttrDevices] = {};
};
// Resident CTAs per SM of a kernel, asked once per device.
int ctas_per_sm(Occupancy& c, const void* f, int threads, int smem) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxAttrDevices) dev = 0;
  int n = c.per_dev[dev].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, f, threads, (size_t)smem) != cudaSuccess || n < 1) {
      (void)cudaGetLastError();
      n = 1;
    }
    n = n > kChunkMaxCtasPerSm ? kChunkMaxCtasPerSm : n;
    c.per_dev[dev].store(n, std::memory_order_relaxed);
  }
  return n;
}

template <bool F8, int RT>
int launch_rows(const CUtensorMap& tk, const CUtensorMap& tv, ChunkParams p, float* parts, int64_t max_slots,
                cudaStream_t s) {
  using C = RowsCfg<F8, RT>;
  static FuncSmemAttr attr;
  static Occupancy occ;
  const void* f = (const void*)chunk_rows_kernel<F8, RT>;
  ensure_dyn_smem(attr, f, C::kAlloc);
  const int64_t most = min64((int64_t)device_sm_count() * ctas_per_sm(occ, f, kRowsThreads, C::kAlloc), max_slots);
  p.TQ = C::kRows / p.G;
  p.min_tiles = 2;
  p.part_o = parts;
  p.part_ml = parts + 2 * most * C::kRows * kChunkD;
  chunk_rows_kernel<F8, RT><<<(unsigned)most, kRowsThreads, C::kAlloc, s>>>(tk, tv, p);
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
}

}  // namespace

// Workspace: 256 bytes (word 0: the error flags), a counter per CTA, then two
// partial results (rows x 66 floats) per CTA.
static int64_t chunk_max_ctas() { return (int64_t)device_sm_count() * kChunkMaxCtasPerSm; }
int64_t chunk_workspace_bytes() {
  return 256 + (chunk_max_ctas() * 4 + 255) / 256 * 256 + chunk_max_ctas() * 2 * 64 * (kChunkD + 2) * 4;
}

int launch_attn_chunk(ChunkParams p, const void* k, const void* v, int32_t f8, int32_t max_q, void* workspace,
                      cudaStream_t s) {
  if (p.N <= 0 || p.T <= 0) return 0;
  p.err = (uint32_t*)workspace;
  p.counters = (uint32_t*)((uint8_t*)workspace + 256);
  float* parts = (float*)((uint8_t*)workspace + 256 + (chunk_max_ctas() * 4 + 255) / 256 * 256);
  CUtensorMap tk, tv;
  const uint64_t rb = f8 ? 64 : 128;
  const uint64_t dk[3] = {64, (uint64_t)p.Hkv, (uint64_t)p.pool_pages * kChunkPage};
  const uint64_t sk[2] = {rb, (uint64_t)p.Hkv * rb};
  const uint32_t box[3] = {64, 1, kChunkPage};
  const CUtensorMapDataType dt = f8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const CUtensorMapSwizzle sw = f8 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
  if (make_tmap_3d(&tk, k, dt, dk, sk, box, sw) || make_tmap_3d(&tv, v, dt, dk, sk, box, sw)) return -2;
  const int64_t rows = (int64_t)max_q * p.G;
  const int64_t m = chunk_max_ctas();
  // the smallest tile that holds the longest chunk's rows; longer chunks go in groups of tokens
  if (rows <= 16 && p.G <= 16)
    return f8 ? launch_rows<true, 1>(tk, tv, p, parts, m, s) : launch_rows<false, 1>(tk, tv, p, parts, m, s);
  if (rows <= 32 && p.G <= 32)
    return f8 ? launch_rows<true, 2>(tk, tv, p, parts, m, s) : launch_rows<false, 2>(tk, tv, p, parts, m, s);
  return f8 ? launch_rows<true, 4>(tk, tv, p, parts, m, s) : launch_rows<false, 4>(tk, tv, p, parts, m, s);
}

}  // namespace gptoss
