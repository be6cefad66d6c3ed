// chunk.cuh -- what the chunk attention kernels share: their parameters and
// the division of a ragged batch over the CTAs.
//
// A unit is (sequence, group of its new tokens, kv head): the G = Hq / Hkv
// query heads of the kv head times the tokens of the group are the rows of one
// tile, so a key is read once for all of them.  A unit's work is its number of
// key tiles; all units of the batch, one after another, form a line of key
// tiles that is cut into equal parts, one per CTA, wherever the cut falls (the
// lengths are only known on the device, and one long context beside many short
// ones must not leave CTAs idle).  A unit cut between CTAs leaves partial
// results (unnormalised output, maximum, sum) in the workspace; whichever CTA
// finishes last joins them in the order of the keys, so the result does not
// depend on which one that was.  A CTA has at most two partial results (its
// first and its last unit), and nobody waits for another CTA.
#pragma once
#include "common.cuh"

namespace gptoss {

constexpr int kChunkD = 64;
constexpr int kChunkPage = 16;
constexpr int kChunkMaxSeqs = 1024;

struct ChunkParams {
  const uint16_t* q;
  int64_t q_stride;  // elements between tokens
  const uint8_t* k_code;
  const uint8_t* v_code;
  int64_t pool_pages;
  const int32_t* table;
  int32_t table_rows, tstride;
  const int32_t* seq_rows;
  const int32_t* q_start;
  const int32_t* kv_len;
  int32_t N, Hq, Hkv, G, TQ, window;  // TQ: tokens of a unit
  int64_t T;
  float scale2;  // sm_scale * log2(e)
  const uint16_t* sinks;
  uint16_t* o;
  float* lse;
  uint32_t* err;
  uint32_t* counters;  // [grid], zero between launches
  float* part_o;       // [2 * grid][rows][64]
  float* part_ml;      // [2 * grid][rows][2]
  int32_t min_tiles;   // key tiles below which a part is not worth a CTA
};

struct ChunkSeq {
  int64_t q0;   // first token
  int32_t ql;   // new tokens
  int32_t off;  // position of the first one (negative: the first tokens see nothing)
  int32_t row;  // page-table row
};

__device__ __forceinline__ ChunkSeq chunk_seq(const ChunkParams& p, int b) {
  ChunkSeq s;
  const int64_t a = max64(0, min64(p.T, p.q_start[b]));
  const int64_t e = max64(a, min64(p.T, p.q_start[b + 1]));
  s.q0 = a;
  s.ql = (int32_t)(e - a);
  s.row = p.seq_rows[b];
  int32_t kl = max(0, p.kv_len[b]);
  if (s.row < 0 || s.row >= p.table_rows) {
    kl = 0;  // no such sequence: nothing to see
    s.row = 0;
  }
  s.off = kl - s.ql;
  return s;
}

// Keys [lo, hi) that some token of group t may see, and the key tiles over them.
template <int KT>
__device__ __forceinline__ int chunk_tiles(const ChunkParams& p, const ChunkSeq& s, int t, int32_t& lo, int32_t& hi) {
  const int32_t t0 = t * p.TQ, t1 = min(s.ql, t0 + p.TQ);
  hi = max(0, s.off + t1);
  lo = p.window > 0 ? min(hi, max(0, s.off + t0 - p.window + 1)) : 0;
  return hi > lo ? (hi + KT - 1) / KT - lo / KT : 0;
}

// A part of a unit for one CTA.
struct ChunkSeg {
  ChunkSeq s;
  int32_t t, hk;
  int32_t lo, hi;    // keys
  int32_t k0;        // first key of tile 0 (lo rounded down)
  int32_t n;         // key tiles of the unit (0: nothing to see, one empty step)
  int32_t i0, i1;    // this CTA's key tiles
  int32_t slot;      // -1: the whole unit; else where the partial result goes
  int32_t c0, c1;    // CTAs that share the unit
  int32_t first_slot;  // slot of CTA c0's part (the others': 2 c)
};

// The walk of one CTA over its part of the line.  `pre` is shared memory for
// kChunkMaxSeqs + 1 prefix sums; init() is called by all threads of the block
// (a multiple of 32) with a __syncthreads inside; next() by any thread, each
// with its own walk.
template <int KT>
struct ChunkWalk {
  int64_t pos, end, total, ubase;
  int32_t b, t, hk, g, cta;
  ChunkSeq s;
  int32_t lo, hi, n;

  __device__ __forceinline__ static void plan(const ChunkParams& p, int64_t* pre, int nthreads) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = nthreads >> 5;
    for (int b = warp; b < p.N; b += nw) {
      const ChunkSeq s = chunk_seq(p, b);
      const int nt = (s.ql + p.TQ - 1) / p.TQ;
      int64_t w = 0;
      for (int t = lane; t < nt; t += 32) {
        int32_t lo, hi;
        w += max(1, chunk_tiles<KT>(p, s, t, lo, hi));
      }
      for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
      if (lane == 0) pre[b + 1] = w * p.Hkv;
    }
    __syncthreads();
    if (warp == 0) {
      int64_t run = 0;
      for (int b0 = 0; b0 < p.N; b0 += 32) {
        int64_t v = b0 + lane < p.N ? pre[b0 + lane + 1] : 0;
        for (int o = 1; o < 32; o <<= 1) {
          const int64_t u = __shfl_up_sync(0xffffffffu, v, o);
          if (lane >= o) v += u;
        }
        if (b0 + lane < p.N) pre[b0 + lane + 1] = run + v;
        run += __shfl_sync(0xffffffffu, v, 31);
      }
      if (lane == 0) pre[0] = 0;
    }
    __syncthreads();
  }

  __device__ __forceinline__ int64_t cut(int c) const { return total * c / g; }
  __device__ __forceinline__ int owner(int64_t x) const { return (int)(((x + 1) * g - 1) / total); }

  __device__ __forceinline__ void begin(const ChunkParams& p, const int64_t* pre, int grid, int cta_) {
    cta = cta_;
    total = pre[p.N];
    g = (int)max64(1, min64(grid, (total + p.min_tiles - 1) / p.min_tiles));
    pos = end = 0;
    if (total == 0 || cta >= g) return;
    pos = cut(cta);
    end = cut(cta + 1);
    int a = 0, z = p.N - 1;  // the last b with pre[b] <= pos and pre[b + 1] > pos
    while (a < z) {
      const int mid = (a + z + 1) >> 1;
      if (pre[mid] <= pos) a = mid;
      else z = mid - 1;
    }
    b = a;
    while (pre[b + 1] <= pos) ++b;
    s = chunk_seq(p, b);
    ubase = pre[b];
    t = 0;
    for (;; ++t) {
      n = chunk_tiles<KT>(p, s, t, lo, hi);
      const int64_t w = (int64_t)max(1, n) * p.Hkv;
      if (ubase + w > pos) break;
      ubase += w;
    }
    hk = (int)((pos - ubase) / max(1, n));
    ubase += (int64_t)hk * max(1, n);
  }

  // The next segment; false at the end of the part.
  __device__ __forceinline__ bool next(const ChunkParams& p, ChunkSeg& x) {
    if (pos >= end) return false;
    const int32_t c = max(1, n);
    const int64_t uend = ubase + c;
    x.s = s;
    x.t = t;
    x.hk = hk;
    x.lo = lo;
    x.hi = hi;
    x.k0 = lo / KT * KT;
    x.n = n;
    x.i0 = (int32_t)(pos - ubase);
    x.i1 = (int32_t)min64(c, end - ubase);
    x.slot = -1;
    if (x.i0 > 0 || x.i1 < c) {
      const bool first = pos == cut(cta);
      x.slot = 2 * cta + (first ? 0 : 1);
      x.c0 = owner(ubase);
      x.c1 = owner(uend - 1);
      x.first_slot = cut(x.c0) == ubase ? 2 * x.c0 : 2 * x.c0 + 1;
    }
    pos = min64(end, uend);
    if (pos >= end) return true;
    // on to the next unit
    ubase = uend;
    if (++hk == p.Hkv) {
      hk = 0;
      if (++t * p.TQ >= s.ql) {
        t = 0;
        do {
          ++b;
          s = chunk_seq(p, b);
        } while (s.ql == 0);
      }
      n = chunk_tiles<KT>(p, s, t, lo, hi);
    }
    return true;
  }
};

}  // namespace gptoss
