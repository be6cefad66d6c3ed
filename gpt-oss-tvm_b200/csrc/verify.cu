// verify.cu -- speculative decoding's acceptance test and the token after it,
// from the target's logits and given random numbers.
//
// Rows row_start[b] .. row_start[b + 1] - 1 of sequence b: row r holds the
// target's logits z for the token that follows tokens[r]; the draft to check
// against it is tokens[r + 1] (the last row has none).  With
//   e_i = exp((z_i - max z) / temperature)    (1 where z_i = max z)
//   w_i = floor(e_i * 2^40),  Z = sum w_i,  p_i = e_i / (Z * 2^-40)
// the draft x of row r is accepted when accept[r] * q(x) < p(x); q is the
// draft's own distribution (1 for a draft that was looked up, not drawn).
// At the first rejected row the next token is drawn from max(p - q, 0)
// (without q: from p without x), after the last accepted draft from p of the
// last row: the weights are again whole multiples of 2^-40, and the token is
// the first whose running sum exceeds floor(u * S).
//
// Sums of whole numbers do not depend on their order, so the split of a row
// over threads and CTAs cannot change a token: the kernels and any other
// evaluation of the formulas above agree bit for bit.
//
// verify_rows_kernel    one cluster of CTAs per row: a CTA's slice stays in
//                       shared memory between the maximum and the sums, so the
//                       logits are read once; the sums of pieces of 256 values
//                       go to the scratch buffer
//                       Bound by issue and latency: 30 instructions a value
//                       (the maximum, expf, floor and two sums), and a CTA's
//                       load, exchange and sums follow one another; four
//                       CTAs an SM cover part of it.  168 rows of 201088 fp32
//                       logits: 60 us, 2.2 TB/s (79 with cluster barriers)
// verify_next_kernel    one CTA per sequence: the first rejected row, the piece
//                       that holds the draw from the stored sums, and the
//                       token in it.  Only with draft distributions the
//                       residual needs the whole row again: then a cluster per
//                       sequence sums its pieces first (48 sequences: 37 us,
//                       51 instructions a value, an IEEE division among them;
//                       49 us where four CTAs fit an SM instead of five, for
//                       which 56 bytes of a thread go to local memory)
#include "common.cuh"
#include "launch.h"

namespace gptoss {

constexpr int kVerThreads = 256;
constexpr int kVerWarps = kVerThreads / 32;
constexpr int kVerPiece = 256;            // values per piece of the running sum: 8 a lane
constexpr int kVerCluster = 16;           // CTAs of a row (the most a cluster takes)
constexpr int kVerNextCluster = 16;
constexpr int64_t kVerMaxVocab = 1 << 22;  // 2^22 weights of at most 2^40 stay below 2^63
constexpr int kVerStash = 110 * 1024;      // the most bytes of a slice kept on chip

struct VerifyParams {
  const void* logits;
  int64_t ld;
  const int32_t* tokens;
  const int32_t* row_start;
  int64_t T;
  int32_t N, V, pieces;
  float inv_temp;
  int greedy;
  const float* accept_u;
  const float* next_u;
  const float* draft;  // [T, V] rows of stride ld_draft, or NULL
  int64_t ld_draft;
  // per row: sums of the pieces and of all weights, max, lowest index of the max, accepted
  long long* piece_sum;
  long long* row_sum;
  float* row_max;
  int32_t* row_top;
  int32_t* row_ok;
  int32_t* accepted;
  int32_t* next;
};

template <typename T>
__device__ __forceinline__ float ver_value(T x);
template <>
__device__ __forceinline__ float ver_value<float>(float x) {
  return fmaxf(x, -INFINITY);  // a NaN logit counts as -inf
}
template <>
__device__ __forceinline__ float ver_value<uint16_t>(uint16_t x) {
  return fmaxf(bf16_bits_to_f32(x), -INFINITY);
}
// e of a value; a maximum that is infinite needs the comparison (inf - inf is no number), for any other it says the
// same without: exp(0) is 1
__device__ __forceinline__ float ver_exp(float z, float m, float inv_temp) {
  return isinf(m) && z == m ? 1.0f : expf(__fmul_rn(__fsub_rn(z, m), inv_temp));
}
__device__ __forceinline__ float ver_total(long long z) { return __ll2float_rn(z) * (1.0f / 1099511627776.0f); }

__device__ __forceinline__ long long ver_join(uint32_t hi, uint32_t lo) { return ((long long)hi << 20) + lo; }
// floor(w * 2^40) of 0 <= w <= 1 as hi * 2^20 + lo, both below 2^21, each plus
// kVerBias: an addition of 2^23 that rounds towards zero leaves the whole part
// in the low bits (a conversion to 64 bits runs at a quarter of the rate).
constexpr uint32_t kVerBias = 0x4B000000u;
__device__ __forceinline__ void ver_fix_biased(float w, uint32_t& hi, uint32_t& lo) {
  const float a = w * 1048576.0f;
  const float t = __fadd_rz(a, 8388608.0f);
  hi = __float_as_uint(t);
  lo = __float_as_uint(__fmaf_rz(__fsub_rn(a, __fsub_rn(t, 8388608.0f)), 1048576.0f, 8388608.0f));
}
__device__ __forceinline__ void ver_fix(float w, uint32_t& hi, uint32_t& lo) {
  ver_fix_biased(w, hi, lo);
  hi -= kVerBias;
  lo -= kVerBias;
}
// Sum of a whole piece's weights over the warp, 8 values a lane.
template <typename F>
__device__ __forceinline__ long long ver_piece(const float (&z)[8], F weight) {
  uint32_t h = 0u - 8u * kVerBias, l = h;
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    uint32_t h1, l1;
    ver_fix_biased(weight(z[k], k), h1, l1);
    h += h1;
    l += l1;
  }
  return ver_join(__reduce_add_sync(0xffffffffu, h), __reduce_add_sync(0xffffffffu, l));
}
// The same for the weights exp((z - m) / T) of a finite m, two values an
// instruction where the roundings are each value's own.
__device__ __forceinline__ unsigned long long ver_pair(float a, float b) {
  return ((unsigned long long)__float_as_uint(b) << 32) | __float_as_uint(a);
}
__device__ __forceinline__ long long ver_piece_exp(const float (&z)[8], float m, float inv_temp) {
  using f2 = unsigned long long;
  const f2 nm2 = ver_pair(-m, -m), it2 = ver_pair(inv_temp, inv_temp), one2 = ver_pair(-1.0f, -1.0f);
  const f2 s20 = ver_pair(1048576.0f, 1048576.0f), p23 = ver_pair(8388608.0f, 8388608.0f);
  const f2 n23 = ver_pair(-8388608.0f, -8388608.0f);
  uint32_t h = 0u - 8u * kVerBias, l = h;
#pragma unroll
  for (int k = 0; k < 8; k += 2) {
    f2 x = ver_pair(z[k], z[k + 1]), t, d;
    asm("add.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(nm2));
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(it2));
    x = ver_pair(expf(__uint_as_float((uint32_t)x)), expf(__uint_as_float((uint32_t)(x >> 32))));
    asm("mul.rn.f32x2 %0, %0, %1;" : "+l"(x) : "l"(s20));
    asm("add.rz.f32x2 %0, %1, %2;" : "=l"(t) : "l"(x), "l"(p23));
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(t), "l"(n23));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(d), "l"(one2), "l"(x));
    asm("fma.rz.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(d), "l"(s20), "l"(p23));
    h += (uint32_t)t + (uint32_t)(t >> 32);
    l += (uint32_t)d + (uint32_t)(d >> 32);
  }
  return ver_join(__reduce_add_sync(0xffffffffu, h), __reduce_add_sync(0xffffffffu, l));
}
// Eight values of a lane: 4 lane .. 4 lane + 3 and 128 more of a piece at q
// (`wide`: 16-byte aligned, or 8 for bf16), -inf from index n on.
template <typename T>
__device__ __forceinline__ void ver_load8(const T* q, int n, bool wide, float (&z)[8]) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = 128 * h + 4 * lane;
    T e[4];
    if (wide && n >= 256) {
      if (sizeof(T) == 4) *(uint4*)e = *(const uint4*)(q + i);
      else *(uint2*)e = *(const uint2*)(q + i);
#pragma unroll
      for (int k = 0; k < 4; ++k) z[4 * h + k] = ver_value<T>(e[k]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) z[4 * h + k] = i + k < n ? ver_value<T>(q[i + k]) : -INFINITY;
    }
  }
}
__device__ __forceinline__ long long warp_sum64(long long v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ long long warp_scan64(long long v) {
  for (int o = 1; o < 32; o <<= 1) {
    const long long t = __shfl_up_sync(0xffffffffu, v, o);
    if ((int)(threadIdx.x & 31) >= o) v += t;
  }
  return v;
}
// Exchange in a cluster without its barriers (whose release waits for every store
// of every warp, about 1600 cycles each): a value is written into another CTA's
// shared memory together with the bytes that the mbarrier there counts.
__device__ __forceinline__ void ver_push(void* slot, uint64_t* bar, uint32_t rank, long long v) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(
                   mapa_shared(smem_u32(slot), rank)),
               "l"(v), "r"(mapa_shared(smem_u32(bar), rank))
               : "memory");
}
// One thread: `bar` for `bytes` bytes.  Then all: ver_cluster_arrive, and ver_cluster_wait before the first push (every
// CTA runs and has its barriers by then; nothing else is ordered, so the arrival may be relaxed).
__device__ __forceinline__ void ver_expect(uint64_t* bar, uint32_t bytes) {
  mbar_init(bar, 1);
  fence_mbar_init();
  mbar_arrive_expect_tx(bar, bytes);
}
__device__ __forceinline__ void ver_cluster_arrive() { asm volatile("barrier.cluster.arrive.relaxed;" ::: "memory"); }
__device__ __forceinline__ void ver_cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
__device__ __forceinline__ bool ver_wait(uint64_t* bar) {
  for (uint32_t i = 0; i < kWaitPolls; ++i)
    if (mbar_try_wait(bar, 0u)) return true;
  return false;
}

// The pieces [lo, hi) of a row that CTA `rank` of `n` takes.
__device__ __forceinline__ void ver_slice(int pieces, uint32_t rank, uint32_t n, int& lo, int& hi) {
  const int per = (pieces + (int)n - 1) / (int)n;
  lo = min(pieces, (int)rank * per);
  hi = min(pieces, lo + per);
}

// Largest value of row[lo, hi) over the calling threads (each its own), the
// values copied to `keep` (from index `pad` on, so that both sides are aligned
// alike) when it is given: 16-byte loads over the aligned middle, eight in
// flight.
template <typename T>
__device__ __forceinline__ float ver_max(const T* __restrict__ row, int lo, int hi, T* keep, int& pad) {
  constexpr int kVec = 16 / (int)sizeof(T);
  const int mis = (int)((kVec - (((uintptr_t)(row + lo) / sizeof(T)) & (kVec - 1))) & (kVec - 1));
  pad = (kVec - mis) & (kVec - 1);
  const int a0 = min(hi, lo + mis);
  const int nv = (hi - a0) / kVec;
  const int tail = a0 + nv * kVec;
  float m = -INFINITY;
  auto one = [&](int i) {
    const T x = row[i];
    if (keep) keep[i - lo + pad] = x;
    m = fmaxf(m, ver_value<T>(x));
  };
  if (threadIdx.x < (unsigned)(a0 - lo)) one(lo + (int)threadIdx.x);
  for (int v0 = threadIdx.x; v0 < nv; v0 += 8 * kVerThreads) {
    uint4 x[8];
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (v0 + k * kVerThreads < nv) x[k] = ldg_nc_v4(row + a0 + (v0 + k * kVerThreads) * kVec);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int v = v0 + k * kVerThreads;
      if (v < nv) {
        if (keep) *(uint4*)(keep + (a0 - lo + pad) + v * kVec) = x[k];
        const uint32_t w[4] = {x[k].x, x[k].y, x[k].z, x[k].w};
#pragma unroll
        for (int y = 0; y < 4; ++y) {  // fmaxf drops a NaN
          if (sizeof(T) == 4) m = fmaxf(m, __uint_as_float(w[y]));
          else m = fmaxf(m, fmaxf(__uint_as_float(w[y] << 16), __uint_as_float(w[y] & 0xFFFF0000u)));
        }
      }
    }
  }
  if (threadIdx.x < (unsigned)(hi - tail)) one(tail + (int)threadIdx.x);
  return m;
}

// One cluster of `C` CTAs per row.
template <typename T>
__global__ void __launch_bounds__(kVerThreads) verify_rows_kernel(const VerifyParams p, int C, int stash) {
  extern __shared__ __align__(16) uint8_t ver_smem[];
  T* keep = (T*)ver_smem;  // this CTA's slice, when `stash`
  __shared__ float wm[kVerWarps];
  __shared__ long long ws[kVerWarps];
  __shared__ long long maxima[kVerCluster], sums[kVerCluster];  // of the cluster's CTAs; the sums in the first one only
  __shared__ uint64_t max_bar, sum_bar;
  cudaTriggerProgrammaticLaunchCompletion();  // the next kernel may take its place and wait
  const uint32_t rank = cluster_ctarank();
  if (threadIdx.x == 0) {
    ver_expect(&max_bar, (uint32_t)C * 8);
    ver_expect(&sum_bar, (uint32_t)C * 8);
  }
  __syncwarp();
  ver_cluster_arrive();
  const int64_t r = blockIdx.x / (unsigned)C;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* row = (const T*)p.logits + r * p.ld;
  int plo, phi;
  ver_slice(p.pieces, rank, (uint32_t)C, plo, phi);
  const int lo = plo * kVerPiece, hi = min(p.V, phi * kVerPiece);
  // pass 1: the maximum
  int pad = 0;
  float m = lo < hi ? ver_max<T>(row, lo, hi, stash ? keep : (T*)nullptr, pad) : -INFINITY;
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (lane == 0) wm[warp] = m;
  __syncthreads();
  ver_cluster_wait();
  if (warp == 0) {
    m = lane < kVerWarps ? wm[lane] : -INFINITY;
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane < C) ver_push(&maxima[rank], &max_bar, (uint32_t)lane, (long long)__float_as_uint(m));
  }
  const bool came = ver_wait(&max_bar);
  m = lane < C ? __uint_as_float((uint32_t)maxima[lane]) : -INFINITY;
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  // pass 2: the sums of the pieces' weights, or the lowest index of the maximum
  const T* src = stash ? keep + pad : row + lo;
  if (!p.greedy) {
    const bool wide = ((uintptr_t)src & (4 * sizeof(T) - 1)) == 0;
    long long sum = 0;
    for (int c = plo + warp; c < phi; c += kVerWarps) {
      float z[8];
      ver_load8<T>(src + (c * kVerPiece - lo), hi - c * kVerPiece, wide, z);
      // beyond the row's end z is -inf: e = 0, but for a row of nothing else
      const int left = hi - c * kVerPiece;
      const long long s =
          isinf(m) ? ver_piece(z, [&](float v, int k) {
            return 128 * (k >> 2) + 4 * lane + (k & 3) < left ? ver_exp(v, m, p.inv_temp) : 0.f;
          })
                   : ver_piece_exp(z, m, p.inv_temp);
      if (lane == 0) p.piece_sum[r * p.pieces + c] = s;
      sum += s;
    }
    if (lane == 0) ws[warp] = sum;
  } else {
    int mi = 0x7FFFFFFF;
    for (int i = lo + (int)threadIdx.x; i < hi; i += kVerThreads)
      if (ver_value<T>(src[i - lo]) == m) {
        mi = i;
        break;
      }
    ws[warp] = 0;
    mi = __reduce_min_sync(0xffffffffu, mi);
    if (lane == 0) ws[warp] = mi;
  }
  __syncthreads();
  // nothing comes here any more but to the first CTA, the others are done
  if (warp != 0) return;
  {
    long long part = p.greedy ? __reduce_min_sync(0xffffffffu, lane < kVerWarps ? (int)ws[lane] : 0x7FFFFFFF)
                              : warp_sum64(lane < kVerWarps ? ws[lane] : 0);
    if (!came) part = -1;  // a bounded wait that ran out
    if (lane == 0) ver_push(&sums[rank], &sum_bar, 0u, part);
  }
  if (rank == 0) {
    const bool all = ver_wait(&sum_bar);
    const long long part = lane < C ? sums[lane] : p.greedy ? 0x7FFFFFFF : 0;
    const bool good = __all_sync(0xffffffffu, all && part >= 0);
    const long long z = p.greedy ? 0 : warp_sum64(part);
    const int mi = p.greedy ? __reduce_min_sync(0xffffffffu, (int)part) : -1;
    if (lane == 0) {
      int ok = 0;
      if (r + 1 < p.T) {  // the draft of this row, if the row is not its sequence's last (then nobody looks)
        const int x = p.tokens[r + 1];
        if (x >= 0 && x < p.V) {
          if (p.greedy) {
            ok = x == mi;
          } else {
            const float px = __fdiv_rn(ver_exp(ver_value<T>(row[x]), m, p.inv_temp), ver_total(z));
            const float qx = p.draft ? p.draft[r * p.ld_draft + x] : 1.0f;
            ok = __fmul_rn(p.accept_u[r], qx) < px;
          }
        }
      }
      p.row_max[r] = m;
      p.row_sum[r] = z;
      p.row_top[r] = good ? mi : -2;
      p.row_ok[r] = good && ok;
    }
  }
}

// One CTA per sequence, or with kDraft a cluster of kVerNextCluster.
template <typename T, bool kDraft>
__global__ void __launch_bounds__(kVerThreads, 5) verify_next_kernel(const VerifyParams p) {
  extern __shared__ __align__(16) uint8_t ver_smem[];
  long long* mine = (long long*)ver_smem;  // kDraft: sums of this CTA's pieces
  __shared__ long long ws[kVerWarps];
  __shared__ long long sums[kVerNextCluster], found_run;
  __shared__ uint64_t sum_bar;
  __shared__ int found;
  const uint32_t rank = kDraft ? cluster_ctarank() : 0u;
  const int b = blockIdx.x / (kDraft ? kVerNextCluster : 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  cudaGridDependencySynchronize();  // the rows' results
  const int64_t r0 = max64(0, min64(p.T, p.row_start[b])), r1 = max64(r0, min64(p.T, p.row_start[b + 1]));
  if (r1 <= r0) {  // no rows: nothing to answer
    if (rank == 0 && threadIdx.x == 0) {
      p.accepted[b] = 0;
      p.next[b] = -1;
    }
    return;
  }
  int64_t at = r0;
  for (; at < r1 - 1; at += 32) {
    const unsigned bad = __ballot_sync(0xffffffffu, at + lane < r1 - 1 && !p.row_ok[at + lane]);
    if (bad) {
      at += __ffs(bad) - 1;
      break;
    }
  }
  at = min64(at, r1 - 1);
  const bool last = at == r1 - 1;
  const bool lost = p.row_top[at] == -2;  // its cluster's exchange did not come to its end
  if (rank == 0 && threadIdx.x == 0) {
    p.accepted[b] = (int32_t)(at - r0);
    if (p.greedy || lost) p.next[b] = max(p.row_top[at], -1);
  }
  if (p.greedy || lost) return;
  const T* row = (const T*)p.logits + at * p.ld;
  const float* qrow = kDraft ? p.draft + at * p.ld_draft : nullptr;
  const float m = p.row_max[at];
  const long long z = p.row_sum[at];
  const float total = ver_total(z);
  const int x = last ? -1 : p.tokens[at + 1];
  const long long* stored = p.piece_sum + at * p.pieces;
  auto own = [&](int i) -> long long {
    uint32_t h, l;
    ver_fix(ver_exp(ver_value<T>(row[i]), m, p.inv_temp), h, l);
    return ver_join(h, l);
  };
  // the first of pieces [lo, hi) whose running sum from `before` on exceeds u, then the first value in it; whole CTA
  auto search = [&](int lo, int hi, long long before, long long u, auto sum_of, auto weight) {
    if (threadIdx.x == 0) found = hi - 1;
    __syncthreads();
    long long run = before;
    for (int c0 = lo; c0 < hi; c0 += kVerThreads) {
      const int c = c0 + (int)threadIdx.x;
      const long long v = c < hi ? sum_of(c) : 0;
      const long long inc = warp_scan64(v);
      if (lane == 31) ws[warp] = inc;
      __syncthreads();
      long long below = run, all = 0;
      for (int w = 0; w < kVerWarps; ++w) {
        if (w < warp) below += ws[w];
        all += ws[w];
      }
      if (c < hi && below + inc > u && below + inc - v <= u) {  // one thread at most
        found = c;
        found_run = below + inc - v;
      }
      run += all;
      __syncthreads();
      if (run > u) break;
    }
    const int c = found;
    if (threadIdx.x < kVerPiece) {
      const int i = c * kVerPiece + (int)threadIdx.x;
      const long long v = i < p.V ? weight(i) : 0;
      const long long inc = warp_scan64(v);
      if (lane == 31) ws[warp] = inc;
      asm volatile("bar.sync 1, %0;" ::"n"(kVerPiece) : "memory");
      long long below = found_run;
      for (int w = 0; w < warp; ++w) below += ws[w];
      if (below + inc > u && below + inc - v <= u) p.next[b] = i;
    }
  };
  // u in [0, S): the token is the first whose running sum is above it
  auto draw = [&](long long s) {
    const long long u = __double2ll_rd(__dmul_rn((double)p.next_u[b], __ll2double_rn(s)));
    return max(0ll, min(u, s - 1));
  };
  if (kDraft && !last) {
    auto left = [&](int i) -> long long {
      const float e = ver_exp(ver_value<T>(row[i]), m, p.inv_temp);
      uint32_t h, l;
      ver_fix(fminf(fmaxf(__fsub_rn(__fdiv_rn(e, total), fmaxf(qrow[i], -INFINITY)), 0.0f), 1.0f), h, l);  // as in the sums
      return ver_join(h, l);
    };
    if (threadIdx.x == 0) ver_expect(&sum_bar, kVerNextCluster * 8);
    __syncwarp();
    ver_cluster_arrive();
    const bool wide = ((uintptr_t)row & (4 * sizeof(T) - 1)) == 0, wide_q = ((uintptr_t)qrow & 15) == 0;
    int plo, phi;
    ver_slice(p.pieces, rank, kVerNextCluster, plo, phi);
    long long sum = 0;
    float zn[8], qn[8];  // the next piece's values are on their way while one is summed
    auto fetch = [&](int c) {
      if (c < phi) {
        ver_load8<T>(row + c * kVerPiece, p.V - c * kVerPiece, wide, zn);
        ver_load8<float>(qrow + c * kVerPiece, p.V - c * kVerPiece, wide_q, qn);
      }
    };
    fetch(plo + warp);
    for (int c = plo + warp; c < phi; c += kVerWarps) {
      float z8[8], q8[8];
      const int left_n = p.V - c * kVerPiece;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        z8[k] = zn[k];
        q8[k] = qn[k];
      }
      fetch(c + kVerWarps);
      const long long s = ver_piece(z8, [&](float v, int k) {
        const float d = fminf(fmaxf(__fsub_rn(__fdiv_rn(ver_exp(v, m, p.inv_temp), total), q8[k]), 0.0f), 1.0f);
        return 128 * (k >> 2) + 4 * lane + (k & 3) < left_n ? d : 0.f;
      });
      if (lane == 0) mine[c - plo] = s;
      sum += s;
    }
    if (lane == 0) ws[warp] = sum;
    __syncthreads();
    ver_cluster_wait();
    if (warp == 0) {
      sum = warp_sum64(lane < kVerWarps ? ws[lane] : 0);
      if (lane < kVerNextCluster) ver_push(&sums[rank], &sum_bar, (uint32_t)lane, sum);
    }
    if (!__syncthreads_and(ver_wait(&sum_bar))) {  // a bounded wait that ran out
      if (rank == 0 && threadIdx.x == 0) p.next[b] = -1;
      return;
    }
    long long before = 0, all = 0, here = 0;
    for (uint32_t c = 0; c < kVerNextCluster; ++c) {
      const long long v = sums[c];
      if (c < rank) before += v;
      if (c == rank) here = v;
      all += v;
    }
    if (all > 0) {
      const long long u = draw(all);
      if (u >= before && u < before + here)
        search(plo, phi, before, u, [&](int c) { return mine[c - plo]; }, left);
      return;
    }
  }
  if (kDraft && rank != 0) return;
  // the row's own weights, without the draft when it was looked up and rejected (unless nothing else is left)
  const bool drop = !kDraft && x >= 0 && x < p.V && own(x) < z;
  const long long wx = drop ? own(x) : 0;
  search(0, p.pieces, 0, draw(z - wx), [&](int c) { return stored[c] - (drop && x / kVerPiece == c ? wx : 0); },
         [&](int i) { return drop && i == x ? 0ll : own(i); });
}

// --------------------------------------------------------------- launch --
static int64_t ver_pieces(int64_t V) { return (V + kVerPiece - 1) / kVerPiece; }
int64_t verify_scratch_bytes(int64_t T, int64_t V) { return T * (8 * ver_pieces(V) + 8 + 4 + 4 + 4) + 64; }

// Clusters of 16 have to be asked for, once per kernel and device.
struct VerWide {
  std::atomic<bool> asked[kMaxAttrDevices] = {};
};
static bool ver_wide_clusters(const void* f, VerWide& w) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxAttrDevices) dev = 0;
  if (w.asked[dev].load(std::memory_order_acquire)) return true;
  if (cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return false;
  w.asked[dev].store(true, std::memory_order_release);
  return true;
}

template <typename T>
static int launch_verify_t(const VerifyParams& p, cudaStream_t s) {
  static VerWide wide_rows, wide_next;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  cfg.blockDim = dim3(kVerThreads);
  cfg.stream = s;
  cfg.attrs = at;
  if (p.T > 0) {
    static FuncSmemAttr attr;
    ensure_dyn_smem(attr, (const void*)verify_rows_kernel<T>, kVerStash + 16);
    const int C = kVerCluster;
    if (!ver_wide_clusters((const void*)verify_rows_kernel<T>, wide_rows)) return -3;
    int keep = (p.pieces + C - 1) / C * kVerPiece * (int)sizeof(T) + 16;
    const int stash = keep <= kVerStash;
    if (!stash) keep = 0;
    cfg.gridDim = dim3((unsigned)(p.T * C));
    cfg.dynamicSmemBytes = (size_t)keep;
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned)C;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, verify_rows_kernel<T>, p, C, stash) != cudaSuccess) return -3;
  }
  // starts while the rows' kernel ends, and waits for its results
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  if (p.draft) {
    if (!ver_wide_clusters((const void*)verify_next_kernel<T, true>, wide_next)) return -3;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = kVerNextCluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cfg.numAttrs = 2;
    cfg.gridDim = dim3((unsigned)(p.N * kVerNextCluster));
    cfg.dynamicSmemBytes = (size_t)((p.pieces + kVerNextCluster - 1) / kVerNextCluster) * 8;
    return cudaLaunchKernelEx(&cfg, verify_next_kernel<T, true>, p) == cudaSuccess ? 0 : -3;
  }
  cfg.gridDim = dim3((unsigned)p.N);
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, verify_next_kernel<T, false>, p) == cudaSuccess ? 0 : -3;
}

int launch_verify(const void* logits, int32_t bf16, int64_t ld, const int32_t* tokens, const int32_t* row_start,
                  int64_t T, int32_t N, int32_t V, double temperature, const float* accept_u, const float* next_u,
                  const float* draft, int64_t ld_draft, void* scratch, int32_t* accepted, int32_t* next,
                  cudaStream_t s) {
  if (N <= 0) return 0;
  if (V > kVerMaxVocab) return -12;
  VerifyParams p;
  p.logits = logits;
  p.ld = ld;
  p.tokens = tokens;
  p.row_start = row_start;
  p.T = T;
  p.N = N;
  p.V = V;
  p.pieces = (int32_t)ver_pieces(V);
  p.greedy = temperature < 1e-6;
  // 2^-126 at least: a zero would make a logit of -infinity no number (every finite one weighs 1 there, as it should)
  p.inv_temp = p.greedy ? 1.0f : fmaxf((float)(1.0 / temperature), 1.17549435e-38f);
  p.accept_u = accept_u;
  p.next_u = next_u;
  p.draft = p.greedy ? nullptr : draft;
  p.ld_draft = ld_draft;
  p.piece_sum = (long long*)(((uintptr_t)scratch + 7) & ~(uintptr_t)7);
  p.row_sum = p.piece_sum + T * p.pieces;
  p.row_max = (float*)(p.row_sum + T);
  p.row_top = (int32_t*)(p.row_max + T);
  p.row_ok = p.row_top + T;
  p.accepted = accepted;
  p.next = next;
  return bf16 ? launch_verify_t<uint16_t>(p, s) : launch_verify_t<float>(p, s);
}

}  // namespace gptoss
