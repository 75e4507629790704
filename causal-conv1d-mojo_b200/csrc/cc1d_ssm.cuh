// What the state space scan kernels share: their arguments, and how a
// launch's items (pieces of sequences) are found.
//
// A sequence is cut into segments of seg_len tokens when there are too few
// (sequence, head) rows to fill the GPU.  The recurrence is linear in the
// state, so a segment's effect on it is S -> decay * S + part, with part the
// state that the segment reaches from zero: one launch computes (part,
// decay) of every segment but each sequence's last, the next one runs every
// segment from the state that the earlier ones combine to.
#pragma once

#include "cc1d_common.cuh"
#include "cc1d_internal.h"

namespace cc1d {

constexpr float kLog2e = 1.4426950408889634f;

struct ScanArgs {
  const void* x; i64 xs_b, xs_t, xs_h, xs_p;
  const void* dt; i64 ds_b, ds_t, ds_h;
  const void* B; i64 bs_b, bs_t, bs_g, bs_n;
  const void* C; i64 cs_b, cs_t, cs_g, cs_n;
  const float* A;
  const float* D;
  const float* dt_bias;
  const int* cu;       // packed sequences, or null
  const void* init; i64 is_s, is_h;
  void* y; i64 ys_b, ys_t, ys_h;
  float* fin; i64 fs_s, fs_h;
  float* part;         // [segments][heads][P][N]: a segment's state from zero
  float* decay;        // [segments][heads]: log of its decay (natural in the walk, base 2 on the tensor cores)
  i64 L;               // tokens of a row
  int H, P, N, G, R;   // R = H / G heads per group
  int nseq;
  i64 seg_len;         // tokens per segment
  int segs;            // segments per sequence (without cu)
  i64 items;           // upper bound of the number of segments
  i64 whole;           // tensor cores, without cu: (sequence, heads) rows that are not cut
  int softplus, dt_f32, init_f32;
};

struct ScanItem {
  int seq;             // sequence
  int seg, nsegs;      // its segment of how many
  i64 batch;           // row of x
  i64 t0, t1;          // tokens [t0, t1) of that row
  i64 first;           // item number of the sequence's segment 0
};

// The segment that item number `item` stands for; false for the numbers
// past the last one.  Called by full warps, with the same item.  Packed
// sequences are counted 32 at a time: every sequence has at least one
// segment (an empty one still has a final state).  Ranges are clamped to the
// row, so a bad table cannot make a kernel leave its buffers.
__device__ __forceinline__ bool scan_locate(const ScanArgs& a, i64 item, ScanItem* it) {
  if (a.cu == nullptr) {
    it->seq = (int)(item / a.segs);
    it->seg = (int)(item - (i64)it->seq * a.segs);
    it->nsegs = a.segs;
    it->batch = it->seq;
    it->t0 = it->seg * a.seg_len;
    it->t1 = min(a.L, it->t0 + a.seg_len);
    it->first = item - it->seg;
    return it->seq < a.nseq;
  }
  const int lane = threadIdx.x & 31;
  i64 before = 0;
  for (int base = 0; base < a.nseq; base += 32) {
    const int s = base + lane;
    i64 b = 0, e = 0, n = 0;
    if (s < a.nseq) {
      b = min(max((i64)a.cu[s], (i64)0), a.L);
      e = min(max((i64)a.cu[s + 1], b), a.L);
      n = max((e - b + a.seg_len - 1) / a.seg_len, (i64)1);
    }
    i64 incl = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const i64 v = __shfl_up_sync(kFull, incl, o);
      if (lane >= o) incl += v;
    }
    const unsigned hit = __ballot_sync(kFull, before + incl > item);
    if (hit) {
      const int src = __ffs(hit) - 1;
      const i64 first = before + __shfl_sync(kFull, incl - n, src);
      b = __shfl_sync(kFull, b, src);
      e = __shfl_sync(kFull, e, src);
      it->seq = base + src;
      it->nsegs = (int)__shfl_sync(kFull, n, src);
      it->seg = (int)(item - first);
      it->batch = 0;
      it->t0 = b + it->seg * a.seg_len;
      it->t1 = min(e, it->t0 + a.seg_len);
      it->first = first;
      return true;
    }
    before += __shfl_sync(kFull, incl, 31);
  }
  return false;
}

// log(1 + exp(v)), v itself where the two agree in fp32.
__device__ __forceinline__ float softplus_f(float v) { return v > 20.f ? v : log1pf(expf(v)); }

// A token's dt as it is stored, and the step length: dt + bias, through
// softplus on request.
template <typename T>
__device__ __forceinline__ float scan_raw_step(const ScanArgs& a, i64 off) {
  return a.dt_f32 ? static_cast<const float*>(a.dt)[off] : Cvt<T>::f(static_cast<const T*>(a.dt)[off]);
}
template <typename T>
__device__ __forceinline__ float scan_step(const ScanArgs& a, i64 off, float bias) {
  const float v = scan_raw_step<T>(a, off) + bias;
  return a.softplus ? softplus_f(v) : v;
}

// Tensor-core scan (cc1d_ssm_tc.cu): what it takes, the CTAs it runs per
// segment, its tokens per block and its launch (the partial states first when
// `part` is set).
constexpr int kScanBlock = 128;
i64 scan_tc_parts(const ScanArgs& a);  // partial states of a split launch
bool scan_tc_eligible(int dtype, const ScanArgs& a, i64 batch);
int scan_tc_pairs(const ScanArgs& a);
cudaError_t launch_scan_tc(int dtype, const ScanArgs& a, i64 batch, cudaStream_t stream);

}  // namespace cc1d
