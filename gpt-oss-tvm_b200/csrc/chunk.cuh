// chunk.cuh -- what the chunk attention kernels share: their parameters and
// the division of a ragged batch over the CTAs.
//
// A unit is (sequence, group of its new tokens, kv head): the G = Hq / Hkv
// query heads of the kv head times the tokens of the group are the rows of one
// tile, so a key is read once for all of them.  A unit's work is its number of
// key tiles, plus `ov` for its beginning and end (in key tiles, measured); all
// units of the batch, one after another, form a line that is cut into equal
// parts, one per CTA, wherever the cut falls (the lengths are only known on the
// device, and one long context beside many short ones must not leave CTAs
// idle).  A unit cut between CTAs leaves partial
// results (unnormalised output, maximum, sum) in the workspace; whichever CTA
// finishes last joins them in the order of the keys, so the result does not
// depend on which one that was.  A CTA has at most two partial results (slot
// 2 c: of a unit that others began; 2 c + 1: of one that it began and others go
// on with), and nobody waits for another CTA.
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
  int32_t HG;          // groups of kv heads: units per group of tokens
  int32_t lg_kt;       // log2 of the keys of a tile
  int32_t ov;          // a unit's beginning and end, in key tiles
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
  // a full-causal sequence has no keys beyond its table row's pages (a window's ring may have gone round)
  if (p.window <= 0) kl = (int32_t)min64(kl, (int64_t)p.tstride * kChunkPage);
  s.off = kl - s.ql;
  return s;
}

// Keys [lo, hi) that some token of group t may see, and the key tiles over them.
__device__ __forceinline__ int chunk_tiles(const ChunkParams& p, const ChunkSeq& s, int t, int32_t& lo, int32_t& hi) {
  const int32_t t0 = t * p.TQ, t1 = min(s.ql, t0 + p.TQ);
  hi = max(0, s.off + t1);
  lo = p.window > 0 ? min(hi, max(0, s.off + t0 - p.window + 1)) : 0;
  return hi > lo ? ((hi - 1) >> p.lg_kt) + 1 - (lo >> p.lg_kt) : 0;
}

// A part of a unit for one CTA, as the loading warp hands it to the others.
struct ChunkSeg {
  int64_t tok0;        // first token (row of q)
  int32_t nrows;       // rows in use: tokens * G; -1: no more parts
  int32_t first_pos;   // position of the first token
  int32_t ntok;
  int32_t hg;          // group of kv heads
  int32_t lo, hi;      // keys some row may see
  int32_t j0;          // first key of the part's first tile
  int32_t ntile;       // key tiles of the part (0: a unit that sees nothing)
  int32_t slot;        // -1: the whole unit; else where the partial result goes
  int32_t c0, c1;      // CTAs that share the unit
  int32_t row;         // page-table row
};

// Prefix sums of the sequences' key tiles (times head groups) in `pre`
// [kChunkMaxSeqs + 1], shared memory; all `nthreads` threads of the block.
// The host has made sure that the total fits 31 bits.
__device__ __forceinline__ void chunk_plan(const ChunkParams& p, int32_t* pre, int nthreads) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, nw = nthreads >> 5;
  // a warp per sequence while there are enough, its lanes over the groups of tokens; else a thread per sequence
  const bool wide = p.N <= nw;
  const int step = wide ? 32 : 1, first = wide ? lane : 0;
  for (int b = wide ? warp : (int)threadIdx.x; b < p.N; b += wide ? nw : nthreads) {
    const ChunkSeq s = chunk_seq(p, b);
    const int nt = (s.ql + p.TQ - 1) / p.TQ;
    int32_t w = 0;
    for (int t = first; t < nt; t += step) {
      int32_t lo, hi;
      w += max(1, chunk_tiles(p, s, t, lo, hi)) + p.ov;
    }
    if (wide)
      for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    if (!wide || lane == 0) pre[b + 1] = w * p.HG;
  }
  __syncthreads();
  if (warp == 0) {
    int32_t run = 0;
    for (int b0 = 0; b0 < p.N; b0 += 32) {
      int32_t v = b0 + lane < p.N ? pre[b0 + lane + 1] : 0;
      for (int o = 1; o < 32; o <<= 1) {
        const int32_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
      }
      if (b0 + lane < p.N) pre[b0 + lane + 1] = run + v;
      run += __shfl_sync(0xffffffffu, v, 31);
    }
    if (lane == 0) pre[0] = 0;
  }
  __syncthreads();
}

// The walk of one CTA over its part of the line (one warp, all lanes alike).
struct ChunkWalk {
  int32_t pos, end, total, ubase;
  int32_t b, t, hg, g, cta, per, rem;
  ChunkSeq s;
  int32_t lo, hi, n;

  // CTA c takes tiles cut(c) .. cut(c + 1) - 1: `per` of them, the first `rem` CTAs one more
  __device__ __forceinline__ int32_t cut(int c) const { return c * per + min(c, rem); }
  __device__ __forceinline__ int owner(int32_t x) const {
    const int32_t big = rem * (per + 1);
    return x < big ? (int)((uint32_t)x / (uint32_t)(per + 1)) : rem + (int)((uint32_t)(x - big) / (uint32_t)per);
  }

  __device__ __forceinline__ void begin(const ChunkParams& p, const int32_t* pre, int grid, int cta_) {
    const int lane = threadIdx.x & 31;
    cta = cta_;
    total = pre[p.N];
    g = max(1, min(grid, total));
    per = (int32_t)((uint32_t)total / (uint32_t)g);
    rem = total - per * g;
    pos = end = 0;
    if (total == 0 || cta >= g) return;
    pos = cut(cta);
    end = cut(cta + 1);
    int a = 0, z = p.N - 1;  // the last b with pre[b] <= pos: it has tiles, since pre[b + 1] > pos
    while (a < z) {
      const int mid = (a + z + 1) >> 1;
      if (pre[mid] <= pos) a = mid;
      else z = mid - 1;
    }
    b = a;
    s = chunk_seq(p, b);
    // the group of tokens that holds pos: 32 groups at a time
    ubase = pre[b];
    for (t = 0;; t += 32) {
      int32_t l_, h_;
      const int nt = (s.ql + p.TQ - 1) / p.TQ;
      int32_t w = t + lane < nt ? (max(1, chunk_tiles(p, s, t + lane, l_, h_)) + p.ov) * p.HG : 0;
      for (int o = 1; o < 32; o <<= 1) {
        const int32_t u = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += u;
      }
      const unsigned past = __ballot_sync(0xffffffffu, ubase + w > pos);
      if (past) {
        const int k = __ffs(past) - 1;
        if (k > 0) ubase += __shfl_sync(0xffffffffu, w, k - 1);
        t += k;
        break;
      }
      ubase += __shfl_sync(0xffffffffu, w, 31);
      if (t + 32 >= nt) break;  // not reached: pos lies in this sequence
    }
    n = chunk_tiles(p, s, t, lo, hi);
    const int32_t c = max(1, n) + p.ov;
    hg = (int)((uint32_t)(pos - ubase) / (uint32_t)c);
    ubase += hg * c;
  }

  // The next part with a key tile (or the one empty step of a unit that sees nothing); false at the end.
  __device__ __forceinline__ bool next(const ChunkParams& p, ChunkSeg& x) {
    while (pos < end) {
      const int32_t c = max(1, n), ub = ubase + p.ov, uend = ub + c;  // the unit's tiles are [ub, uend)
      const int32_t i0 = max(0, pos - ub), i1 = min(c, end - ub);
      x.tok0 = s.q0 + (int64_t)t * p.TQ;
      x.ntok = min(p.TQ, s.ql - t * p.TQ);
      x.nrows = x.ntok * p.G;
      x.first_pos = s.off + t * p.TQ;
      x.hg = hg;
      x.lo = lo;
      x.hi = hi;
      x.j0 = ((lo >> p.lg_kt) + i0) << p.lg_kt;
      x.ntile = n == 0 ? 0 : i1 - i0;
      x.row = s.row;
      x.slot = -1;
      x.c0 = x.c1 = 0;
      if (i0 > 0 || i1 < c) {
        x.slot = 2 * cta + (i0 > 0 ? 0 : 1);
        x.c0 = owner(ub);
        x.c1 = owner(uend - 1);
      }
      pos = min(end, uend);
      if (pos < end) {
        // on to the next unit
        ubase = uend;
        if (++hg == p.HG) {
          hg = 0;
          if (++t * p.TQ >= s.ql) {
            t = 0;
            do {
              ++b;
              s = chunk_seq(p, b);
            } while (s.ql == 0);
          }
          n = chunk_tiles(p, s, t, lo, hi);
        }
      }
      if (i1 > i0) return true;
    }
    return false;
  }
};

}  // namespace gptoss
