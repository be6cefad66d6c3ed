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
// verify_rows_kernel    one cluster of 8 CTAs per row: its slice of the row
//                       stays in shared memory between the maximum and the
//                       sum, so the logits are read once
// verify_next_kernel    one cluster per sequence: the first rejected row, the
//                       sum of its weights by 1024-value pieces, then the one
//                       piece that holds the draw
#include "common.cuh"
#include "launch.h"

namespace gptoss {

constexpr int kVerCluster = 8;
constexpr int kVerThreads = 512;
constexpr int kVerPiece = 1024;          // values per piece of the running sum
constexpr float kVerFix = 1099511627776.0f;  // 2^40
constexpr int64_t kVerMaxVocab = 1 << 22;    // 2^22 weights of at most 2^40 stay below 2^63

struct VerifyParams {
  const void* logits;
  int64_t ld;
  const int32_t* tokens;
  const int32_t* row_start;
  int64_t T;
  int32_t N, V;
  float inv_temp;
  int greedy;
  const float* accept_u;
  const float* next_u;
  const float* draft;  // [T, V] rows of stride ld_draft, or NULL
  int64_t ld_draft;
  // per row: max, sum of the weights, lowest index of the max, accepted
  float* row_max;
  long long* row_sum;
  int32_t* row_top;
  int32_t* row_ok;
  int32_t* accepted;
  int32_t* next;
};

template <typename T>
__device__ __forceinline__ float ver_value(T x);
template <>
__device__ __forceinline__ float ver_value<float>(float x) {
  return x != x ? -INFINITY : x;  // a NaN logit counts as -inf
}
template <>
__device__ __forceinline__ float ver_value<uint16_t>(uint16_t x) {
  const float f = bf16_bits_to_f32(x);
  return f != f ? -INFINITY : f;
}
__device__ __forceinline__ float ver_exp(float z, float m, float inv_temp) {
  return z == m ? 1.0f : expf(__fmul_rn(__fsub_rn(z, m), inv_temp));
}
__device__ __forceinline__ long long ver_fix(float w) { return __float2ll_rz(w * kVerFix); }
__device__ __forceinline__ float ver_total(long long z) { return __ll2float_rn(z) * (1.0f / kVerFix); }

__device__ __forceinline__ long long warp_sum64(long long v) {
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ void better(float& m, int& i, float m2, int i2) {
  if (m2 > m || (m2 == m && i2 < i)) {
    m = m2;
    i = i2;
  }
}
// Value of a shared variable in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t ld_cluster_u32(const void* p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}
__device__ __forceinline__ long long ld_cluster_s64(const void* p, uint32_t rank) {
  long long v;
  asm volatile("ld.shared::cluster.s64 %0, [%1];" : "=l"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}

// The slice [lo, hi) of a row that CTA `rank` takes: whole pieces.
__device__ __forceinline__ void ver_slice(int V, uint32_t rank, int& lo, int& hi) {
  const int pieces = (V + kVerPiece - 1) / kVerPiece;
  const int per = (pieces + kVerCluster - 1) / kVerCluster;
  lo = min(V, (int)rank * per * kVerPiece);
  hi = min(V, lo + per * kVerPiece);
}

// Calls f(index, value) for this thread's values of [lo, hi); 16-byte loads
// over the aligned middle (a row of an odd vocabulary starts anywhere).
template <typename T, typename F>
__device__ __forceinline__ void ver_each(const T* __restrict__ row, int lo, int hi, F f) {
  constexpr int kVec = 16 / (int)sizeof(T);
  const int mis = (int)((kVec - (((uintptr_t)(row + lo) / sizeof(T)) & (kVec - 1))) & (kVec - 1));
  const int a0 = min(hi, lo + mis);
  const int nv = (hi - a0) / kVec;
  const int tail = a0 + nv * kVec;
  if (threadIdx.x < (unsigned)(a0 - lo)) f(lo + (int)threadIdx.x, row[lo + threadIdx.x]);
#pragma unroll 4
  for (int v = threadIdx.x; v < nv; v += kVerThreads) {
    const uint4 x = ldg_nc_v4(row + a0 + v * kVec);
    const T* e = (const T*)&x;
#pragma unroll
    for (int k = 0; k < kVec; ++k) f(a0 + v * kVec + k, e[k]);
  }
  if (threadIdx.x < (unsigned)(hi - tail)) f(tail + (int)threadIdx.x, row[tail + threadIdx.x]);
}

template <typename T>
__global__ void __cluster_dims__(kVerCluster, 1, 1) __launch_bounds__(kVerThreads)
    verify_rows_kernel(const VerifyParams p, int stash) {
  extern __shared__ __align__(16) uint8_t ver_smem[];
  T* keep = (T*)ver_smem;  // this CTA's slice, when `stash`
  __shared__ float wm[kVerThreads / 32];
  __shared__ int wi[kVerThreads / 32];
  __shared__ long long ws[kVerThreads / 32];
  __shared__ float cta_m;
  __shared__ int cta_i;
  __shared__ long long cta_s;
  const uint32_t rank = cluster_ctarank();
  const int64_t r = blockIdx.x / kVerCluster;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const T* row = (const T*)p.logits + r * p.ld;
  int lo, hi;
  ver_slice(p.V, rank, lo, hi);
  // pass 1: maximum and its lowest index
  float m = -INFINITY;
  int mi = 0x7FFFFFFF;
  ver_each<T>(row, lo, hi, [&](int i, T x) {
    if (stash) keep[i - lo] = x;
    const float z = ver_value<T>(x);
    if (z > m || mi == 0x7FFFFFFF) {  // a thread's indices rise, but for its head and tail values
      m = z;
      mi = i;
    } else if (z == m && i < mi) {
      mi = i;
    }
  });
  for (int o = 16; o > 0; o >>= 1)
    better(m, mi, __shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, mi, o));
  if (lane == 0) {
    wm[warp] = m;
    wi[warp] = mi;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kVerThreads / 32; ++w) better(m, mi, wm[w], wi[w]);
    cta_m = m;
    cta_i = mi;
  }
  cluster_sync_all();
  m = -INFINITY;
  mi = 0x7FFFFFFF;
  for (uint32_t c = 0; c < kVerCluster; ++c)
    better(m, mi, __uint_as_float(ld_cluster_u32(&cta_m, c)), (int)ld_cluster_u32(&cta_i, c));
  // pass 2: the sum of the weights
  long long sum = 0;
  if (!p.greedy) {
    if (stash) {
      for (int i = threadIdx.x; i < hi - lo; i += kVerThreads)
        sum += ver_fix(ver_exp(ver_value<T>(keep[i]), m, p.inv_temp));
    } else {
      ver_each<T>(row, lo, hi, [&](int i, T x) { sum += ver_fix(ver_exp(ver_value<T>(x), m, p.inv_temp)); });
    }
    sum = warp_sum64(sum);
    if (lane == 0) ws[warp] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
      sum = 0;
      for (int w = 0; w < kVerThreads / 32; ++w) sum += ws[w];
      cta_s = sum;
    }
  }
  cluster_sync_all();
  if (rank == 0 && threadIdx.x == 0) {
    long long z = 0;
    if (!p.greedy)
      for (uint32_t c = 0; c < kVerCluster; ++c) z += ld_cluster_s64(&cta_s, c);
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
    p.row_top[r] = mi;
    p.row_ok[r] = ok;
  }
  cluster_sync_all();  // nobody leaves while its shared memory may be read
}

// One cluster per sequence.
template <typename T>
__global__ void __cluster_dims__(kVerCluster, 1, 1) __launch_bounds__(kVerThreads)
    verify_next_kernel(const VerifyParams p) {
  extern __shared__ __align__(16) uint8_t ver_smem[];
  long long* piece = (long long*)ver_smem;  // sums of this CTA's pieces
  __shared__ long long cta_s;
  const uint32_t rank = cluster_ctarank();
  const int b = blockIdx.x / kVerCluster;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
  if (rank == 0 && threadIdx.x == 0) {
    p.accepted[b] = (int32_t)(at - r0);
    if (p.greedy) p.next[b] = p.row_top[at];
  }
  if (p.greedy) return;
  const T* row = (const T*)p.logits + at * p.ld;
  const float* qrow = p.draft ? p.draft + at * p.ld_draft : nullptr;
  const float m = p.row_max[at], total = ver_total(p.row_sum[at]);
  const int x = last ? -1 : p.tokens[at + 1];
  int lo, hi;
  ver_slice(p.V, rank, lo, hi);
  const int np = (hi - lo + kVerPiece - 1) / kVerPiece;
  // mode 0: the residual (or the last row's weights); mode 1, when nothing is left of it: the row's own weights
  for (int mode = 0; mode < 2; ++mode) {
    auto weight = [&](int i) -> long long {
      const float e = ver_exp(ver_value<T>(row[i]), m, p.inv_temp);
      if (last || mode == 1) return ver_fix(e);
      if (qrow) return ver_fix(fmaxf(__fsub_rn(__fdiv_rn(e, total), qrow[i]), 0.0f));
      return i == x ? 0 : ver_fix(e);
    };
    for (int c = warp; c < np; c += kVerThreads / 32) {
      const int p0 = lo + c * kVerPiece, p1 = min(hi, p0 + kVerPiece);
      long long s = 0;
#pragma unroll 8
      for (int i = p0 + lane; i < p1; i += 32) s += weight(i);
      s = warp_sum64(s);
      if (lane == 0) piece[c] = s;
    }
    __syncthreads();
    if (warp == 0) {
      long long s = 0;
      for (int c = lane; c < np; c += 32) s += piece[c];
      s = warp_sum64(s);
      if (lane == 0) cta_s = s;
    }
    cluster_sync_all();
    long long before = 0, all = 0, mine = 0;
    for (uint32_t c = 0; c < kVerCluster; ++c) {
      const long long s = ld_cluster_s64(&cta_s, c);
      if (c < rank) before += s;
      if (c == rank) mine = s;
      all += s;
    }
    cluster_sync_all();
    if (all == 0 && mode == 0) continue;
    // u in [0, S): the token is the first whose running sum is above it
    const double sd = __ll2double_rn(all);
    long long u = __double2ll_rd(__dmul_rn((double)p.next_u[b], sd));
    u = max(0ll, min(u, all - 1));
    if (warp == 0 && u >= before && u < before + mine) {
      long long run = before;
      int c = 0;
      while (c < np - 1 && run + piece[c] <= u) run += piece[c++];
      const int p0 = lo + c * kVerPiece, p1 = min(hi, p0 + kVerPiece);
      for (int i0 = p0; i0 < p1; i0 += 32) {
        const int i = i0 + lane;
        long long s = i < p1 ? weight(i) : 0;
        for (int o = 1; o < 32; o <<= 1) {
          const long long t = __shfl_up_sync(0xffffffffu, s, o);
          if (lane >= o) s += t;
        }
        const unsigned hit = __ballot_sync(0xffffffffu, run + s > u);
        if (hit) {
          if (lane == 0) p.next[b] = i0 + __ffs(hit) - 1;
          break;
        }
        run += __shfl_sync(0xffffffffu, s, 31);
      }
    }
    break;
  }
}

// --------------------------------------------------------------- launch --
int64_t verify_scratch_bytes(int64_t T) { return T * (8 + 4 + 4 + 4) + 64; }

template <typename T>
static int launch_verify_t(const VerifyParams& p, cudaStream_t s) {
  const int pieces = (p.V + kVerPiece - 1) / kVerPiece;
  const int per = (pieces + kVerCluster - 1) / kVerCluster;
  // the slice stays in shared memory while two CTAs fit on an SM
  int keep = per * kVerPiece * (int)sizeof(T);
  const int stash = keep <= 110 * 1024;
  if (!stash) keep = 0;
  static FuncSmemAttr attr_rows, attr_next;
  if (keep > 40 * 1024) ensure_dyn_smem(attr_rows, (const void*)verify_rows_kernel<T>, 110 * 1024);
  verify_rows_kernel<T><<<(unsigned)(p.T * kVerCluster), kVerThreads, keep, s>>>(p, stash);
  if (cudaGetLastError() != cudaSuccess) return -3;
  verify_next_kernel<T><<<(unsigned)(p.N * kVerCluster), kVerThreads, per * 8, s>>>(p);
  (void)attr_next;
  return cudaGetLastError() == cudaSuccess ? 0 : -3;
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
  p.greedy = temperature < 1e-6;
  p.inv_temp = p.greedy ? 1.0f : (float)(1.0 / temperature);
  p.accept_u = accept_u;
  p.next_u = next_u;
  p.draft = draft;
  p.ld_draft = ld_draft;
  p.row_sum = (long long*)(((uintptr_t)scratch + 7) & ~(uintptr_t)7);
  p.row_max = (float*)(p.row_sum + T);
  p.row_top = (int32_t*)(p.row_max + T);
  p.row_ok = p.row_top + T;
  p.accepted = accepted;
  p.next = next;
  return bf16 ? launch_verify_t<uint16_t>(p, s) : launch_verify_t<float>(p, s);
}

}  // namespace gptoss
