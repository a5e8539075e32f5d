// Pieces shared by the differential-attention kernels (diff_attention.cu,
// diff_attention_tc.cu): which sequence and query block a CTA has.
#pragma once
#include "elem.cuh"
#include "kernels.h"

namespace le {
namespace dif {

// Query blocks of BQ rows are numbered so that sequence s begins at number
// offsets[s] / BQ + s: that grows by at least ceil(length / BQ) per sequence,
// so T / BQ + nseq numbers cover every block (a few are empty) without a list
// or the lengths on the host.
__host__ __device__ inline int block_count(int T, int nseq, int bq) { return T / bq + nseq; }

struct Where {
  int t0, len, q0;  // first row and length of the sequence, first query of the block
};

// Sequence s; false when it is empty or not within [0, T] (reported).
__device__ __forceinline__ bool sequence(const DiffParams& p, int s, Where& w) {
  const int t0 = p.offsets[s], t1 = p.offsets[s + 1];
  if (t0 < 0 || t1 < t0 || t1 > p.T) {
    if ((threadIdx.x & 31) == 0) report(p.status, DE_BOUNDS, 80, s);
    return false;
  }
  w.t0 = t0;
  w.len = t1 - t0;
  w.q0 = 0;
  return t1 > t0;
}

// The sequence of block number `tile` in `offsets` (p.offsets or a copy), found
// by the calling warp (32 probes a step).  False when the block is empty or the
// offsets do not describe sequences within [0, T] (reported).
__device__ __forceinline__ bool find_block(const DiffParams& p, const int32_t* offsets, int tile, int bq, Where& w) {
  const int lane = threadIdx.x & 31;
  int lo = 0, hi = p.nseq;  // the answer is in [lo, hi)
  int t0 = 0, t1 = 0;
  while (true) {
    const int step = (hi - lo + 31) / 32;
    const int i = lo + lane * step;
    const int at = i <= p.nseq ? offsets[i] : 0;
    const bool le = i < hi && (long)at / bq + i <= tile;
    const int n = __popc(__ballot_sync(0xffffffffu, le));
    if (n == 0) return false;
    lo += (n - 1) * step;
    hi = min(hi, lo + step);
    if (hi - lo <= 1) {  // its offsets: with steps of one, lanes n - 1 and n have them
      t0 = __shfl_sync(0xffffffffu, at, n - 1);
      t1 = __shfl_sync(0xffffffffu, at, n & 31);
      if (step > 1 || n > 31) t1 = offsets[lo + 1];
      break;
    }
  }
  if (t0 < 0 || t1 < t0 || t1 > p.T) {
    if (lane == 0) report(p.status, DE_BOUNDS, 80, lo);
    return false;
  }
  w.t0 = t0;
  w.len = t1 - t0;
  const long q0 = ((long)tile - (t0 / bq + lo)) * bq;
  if (q0 < 0 || q0 >= w.len) return false;
  w.q0 = (int)q0;
  return true;
}

// Reports offsets that descend or leave [0, T] (one warp of a launch runs it).
__device__ __forceinline__ void check_offsets(const DiffParams& p) {
  for (int s = threadIdx.x & 31; s < p.nseq; s += 32) {
    const int a = p.offsets[s], b = p.offsets[s + 1];
    if (a < 0 || b < a || b > p.T) report(p.status, DE_BOUNDS, 81, s);
  }
}

__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace dif
}  // namespace le
